"""The SwiGLU fold of the experts' products where the exponential leaves the
range of fp32, with up values of every size.

Bounds, on h = g / (1 + exp(-g)) u of exact g and u.  Where exp(-g) is below
2^128: the exponential is off by two roundings, its correction, the sum, the
quotient's two and the products by one each, 8 in all, relative to h; a
sigmoid below the smallest normal is off by 2^-150, so h by |g u| 2^-150 more,
and a g sigmoid or an h below it by half the smallest step, 2^-150 |u| and
2^-150.  Past 2^128 the formula in fp32 has g / infinity = 0, so anything from
h to 0 is right.  bf16: the exponent's argument is rounded once more, |g| 2^-24
relative to h, and the result to bf16."""
import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, torch
from test_gpu_mx import Encoded, run_experts

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu

K = 32
GATES = [0.0, 0.5, -1.0, 20.0, -20.0, 80.0, -80.0, 87.25, -87.25, 87.5, -87.5, 88.0, -88.0, -88.25, -88.5, -88.75,
         -89.0, -90.0, -92.0, 96.0, -104.0, -120.0, -128.0, 128.0, -144.0, 150.0, -150.0, -176.0, 1536.0, -1536.0, -2.0 ** 20, 2.0 ** 40,
         -2.0 ** 40, 2.0 ** 70, -2.0 ** 70, 2.0 ** 100, -2.0 ** 100, 1.5 * 2.0 ** 126, -1.5 * 2.0 ** 126, -2.0 ** -100]
UPS = [1.0, -3.0, 2.0 ** -100, 2.0 ** 20, -2.0 ** 20, 2.0 ** 60, 1.5 * 2.0 ** 100, -2.0 ** 120]


def row_of(value):
    """Codes and the scale byte of a block of 32 whose sum is `value` (exactly)."""
    index = {m: i for i, m in enumerate(mx.MAGNITUDES)}
    left = abs(value)
    s = int(np.ceil(np.log2(left / (6 * K)))) if left else 0  # the smallest that holds it
    left /= 2.0 ** s
    codes = np.zeros(mx.padded(K), np.uint8)
    for k in range(K):
        part = max(m for m in mx.MAGNITUDES if m <= left)
        codes[k] = index[part] | (8 if value < 0 else 0)
        left -= part
    assert left == 0, value
    scales = np.zeros(mx.padded(K) // 32, np.uint8)
    scales[0] = 127 + s
    return codes[0::2] | codes[1::2] << 4, scales


def matrix(q38m, values):
    rows = [row_of(v) for v in values]
    return Encoded(q38m, np.stack([c for c, _ in rows]), np.stack([s for _, s in rows]), K)


def ones(q38m, rows):
    codes, scales = np.zeros((rows, mx.padded(K) // 2), np.uint8), np.zeros((rows, mx.padded(K) // 32), np.uint8)
    codes[:, :K // 2], scales[:, 0] = 0x22, 127
    return Encoded(q38m, codes, scales, K)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_swiglu_range(q38m, dtype):
    pairs = [(g, u) for g in GATES for u in UPS]
    w = matrix(q38m, [g for g, _ in pairs] + [u for _, u in pairs])
    a = ones(q38m, 5)
    assert (a.values == 1).all()
    offsets = device(np.array([0, 5], np.uint32))
    _, got = run_experts(q38m, w, a, offsets, None, 1, 5, True, dtype)
    g, u = (np.array(v, np.float64) for v in zip(*pairs))
    assert np.array_equal(w.values.sum(1), np.concatenate((g, u)))
    want = mx.swiglu(g, u)
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    least = 2.0 ** -134 if dtype == "bf16" else 2.0 ** -150
    top = np.finfo(np.float32).max if dtype == "f32" else 255 * 2.0 ** 120
    relative = 8 * 2.0 ** -24 + (np.minimum(np.abs(g), 90.0) * 2.0 ** -24 if dtype == "bf16" else 0.0)
    inside = -g < np.log(2.0) * 128
    bound = relative * np.abs(want) + np.abs(g * u) * 2.0 ** -150 + np.abs(u) * 2.0 ** -150 + 2.0 ** -150
    bound = np.where(inside, bound, np.abs(want))
    for row in got:
        beyond = np.abs(want) > top * (1 + half)
        assert np.array_equal(np.isinf(row), beyond)
        off = np.abs(row - want)[~beyond]
        limit = (bound * (1 + half) + half * np.abs(want) + least)[~beyond]
        worst = np.argmax(off / limit)
        assert off[worst] <= limit[worst], (np.array(pairs)[~beyond][worst], row[~beyond][worst], want[~beyond][worst])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_swiglu_infinite_and_nan(q38m, dtype):
    """A gate or an up value past fp32, and NaN: what the formula gives."""
    t = torch()
    huge = 6 * 2.0 ** 127  # of scale byte 254: infinite in fp32, as K - 1 more of them
    codes = np.zeros((6, 64), np.uint8)
    scales = np.zeros((6, 4), np.uint8)
    codes[:, :16] = 0x77
    #       gate: +inf, -inf, NaN; up: 1 .. each
    scales[:, 0] = [254, 254, 255, 127, 127, 127]
    codes[1, :16] = 0xff
    w = Encoded(q38m, codes, scales, K)
    assert w.values[0, 0] == huge
    _, got = run_experts(q38m, w, ones(q38m, 1), device(np.array([0, 1], np.uint32)), None, 1, 1, True, dtype)
    t.cuda.synchronize()
    assert got[0, 0] == np.inf and np.isnan(got[0, 1]) and np.isnan(got[0, 2])
