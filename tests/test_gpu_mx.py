"""Microscaled 4-bit rows on the GPU against the plain 64-bit forms
(oracle/mx_oracle.py): the quantiser bit for bit, the products within a bound
on their fp32 sums.

Bound of a product: its terms are exact in fp32 (two significant bits each,
power-of-two scales).  Each matrix instruction covers at least 64 values of K
and adds its terms to an fp32 accumulator; one such step, and each addition of
partial sums, is taken to be off by at most 2^-23 of the magnitudes it adds
(twice a rounding: bits below the largest term may be cut off).  With at most
eight partial sums, S the sum of all terms' magnitudes: (ceil(K / 64) + 8)
2^-23 S, then half a step of the output type.
"""
import ctypes

import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, host, stream, torch

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu

BF16_HALF, F32_HALF = 2.0 ** -8, 2.0 ** -24


def bf16_words(x):
    """float64 -> bf16 words, to nearest even (through fp32: inputs only)."""
    t = torch()
    return host(t.from_numpy(np.asarray(x, np.float32)).to(t.bfloat16).view(t.int16), np.uint16)


def widen(words):
    return (words.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def product_bound(k, size):
    return (-(-k // 64) + 8) * 2.0 ** -23 * size


def close(got, want, bound, dtype, what):
    """got within bound of want, then half a step of dtype; infinities and NaN in the same places."""
    half = BF16_HALF if dtype == "bf16" else F32_HALF
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    live = ~np.isnan(want)
    limit = bound[live] * (1 + half) + half * np.abs(want[live]) + 1e-44
    off = np.abs(got[live] - want[live])
    assert (off <= limit).all(), (what, float((off / limit).max()))


# ---- quantisation -----------------------------------------------------------

def run_quantize(q38m, words, rows, columns, stride, dtype, rounded=True, shift=0):
    """Quantises rows of `words` (flat uint16 or float32, `shift` elements in front); returns
    codes, scales, values and checks that nothing around them is written."""
    t = torch()
    buffer = device(np.concatenate((np.zeros(shift, words.dtype), words)))
    row, scale = q38m.lib().q38m_mx_row_bytes(columns), q38m.lib().q38m_mx_scale_bytes(columns)
    codes = t.full((rows * row + 64,), 0xa5, dtype=t.uint8, device="cuda")
    scales = t.full((rows * scale + 64,), 0xa5, dtype=t.uint8, device="cuda")
    values = t.full((rows * columns + 64,), 7777, dtype=t.int16 if dtype == "bf16" else t.int32,
                    device="cuda")
    desc = q38m.MxMatrix(codes.data_ptr(), scales.data_ptr(), 1, rows, columns)
    x = buffer.data_ptr() + shift * words.itemsize
    q38m.call("q38m_mx_quantize_v1", x, q38m.DTYPE_BF16 if dtype == "bf16" else q38m.DTYPE_F32,
              stride, ctypes.byref(desc), values.data_ptr() if rounded else None, stream(), 0)
    t.cuda.synchronize()
    assert (codes[rows * row:] == 0xa5).all() and (scales[rows * scale:] == 0xa5).all()
    assert (values[rows * columns:] == 7777).all()
    if not rounded:
        assert (values == 7777).all()
    v = host(values, np.uint16 if dtype == "bf16" else np.float32)[:rows * columns]
    v = widen(v) if dtype == "bf16" else v.astype(np.float64)
    return (host(codes, np.uint8)[:rows * row].reshape(rows, row),
            host(scales, np.uint8)[:rows * scale].reshape(rows, scale), v.reshape(rows, columns))


def check_quantize(q38m, x, columns, dtype, rounded=True, shift=0):
    """x [rows][stride] float64 whose values the type holds."""
    rows, stride = x.shape
    words = bf16_words(x) if dtype == "bf16" else x.astype(np.float32)
    exact = (widen(words) if dtype == "bf16" else words.astype(np.float64)).reshape(rows, stride)
    codes, scales, values = mx.quantize(exact[:, :columns])
    got = run_quantize(q38m, words.reshape(-1), rows, columns, stride, dtype, rounded, shift)
    assert np.array_equal(got[1], scales)
    assert np.array_equal(got[0], codes)
    if rounded:
        assert np.array_equal(got[2], values, equal_nan=True)
        assert np.array_equal(np.signbit(got[2]), np.signbit(values)) or np.isnan(values).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,columns,spare,shift", [
    (1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (2, 33, 7, 1), (5, 100, 0, 0), (9, 128, 8, 0),
    (17, 129, 0, 3), (10, 512, 0, 0), (7, 1000, 24, 0), (3, 2048, 0, 8), (2, 2050, 1, 0),
    (1, 8193, 0, 0), (300, 64, 0, 0), (1025, 40, 0, 4)])
def test_quantize(q38m, dtype, rows, columns, spare, shift):
    print(f"quantize {rows} x {columns} + {spare}, shift {shift}, {dtype}", flush=True)
    rng = np.random.default_rng(rows * 7919 + columns)
    x = rng.normal(size=(rows, columns + spare)) * np.exp(4 * rng.normal(size=(rows, 1)))
    x[rng.random(x.shape) < 0.1] = 0.0
    check_quantize(q38m, x, columns, dtype, shift=shift)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_every_bf16(q38m, dtype):
    """Every bf16 pattern (NaN and the infinities among them) beside a value of every eighth
    exponent: roundings, ties, saturation and subnormals under many scales."""
    words = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    patterns = widen(words).reshape(-1, 16)
    blocks = []
    for field in range(1, 255, 8):
        top = widen(np.full((4096, 1), field << 7, np.uint16))
        blocks.append(np.concatenate((patterns, np.broadcast_to(top, (4096, 16))), 1))
    x = np.concatenate(blocks, 1)
    with np.errstate(invalid="ignore"):
        check_quantize(q38m, x, x.shape[1], dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_not_finite(q38m, dtype):
    """A NaN or an infinity takes its block and no other; the padding's scale stays."""
    x = np.random.default_rng(5).normal(size=(4, 300))
    x[0, 0], x[1, 31], x[2, 299], x[3, 128] = np.nan, np.inf, -np.inf, np.nan
    x[3, 160:192] = 0.0
    x[3, 161] = -0.0
    check_quantize(q38m, x, 300, dtype)
    check_quantize(q38m, x, 290, dtype, rounded=False)


# ---- products ---------------------------------------------------------------

def encoded(rng, rows, columns, low=119, high=135):
    """Random codes and scales in the stored layout, their padding zero."""
    k = mx.padded(columns)
    both = rng.integers(0, 16, size=(rows, k), dtype=np.uint8)
    both[:, columns:] = 0
    scales = rng.integers(low, high, size=(rows, k // 32), dtype=np.uint8)
    scales[:, -(-columns // 32):] = 0
    return both[:, 0::2] | both[:, 1::2] << 4, scales


class Encoded:
    def __init__(self, q38m, codes, scales, columns, experts=1):
        self.codes, self.scales = device(codes), device(scales)
        self.desc = q38m.MxMatrix(self.codes.data_ptr(), self.scales.data_ptr(), experts,
                                  codes.shape[0] // experts, columns)
        self.values = mx.decode(codes, scales, columns)


def output(rows, stride, dtype):
    t = torch()
    out = t.full((rows * stride + 64,), 0x4a4a, dtype=t.int16 if dtype == "bf16" else t.int32,
                 device="cuda")
    return out, (None, out.data_ptr()) if dtype == "bf16" else (out.data_ptr(), None)


def read_output(out, rows, stride, dtype):
    torch().cuda.synchronize()
    words = host(out, np.uint16 if dtype == "bf16" else np.uint32)
    assert (words[rows * stride:] == 0x4a4a).all(), "written past the end"
    words = words[:rows * stride].reshape(rows, stride)
    values = widen(words) if dtype == "bf16" else words.view(np.float32).astype(np.float64)
    return words, values


def check_product(q38m, a, b, k, dtype, spare=0):
    m, n = a.desc.rows, b.desc.rows
    out, args = output(m, n + spare, dtype)
    q38m.call("q38m_mx_gemm_v1", ctypes.byref(a.desc), ctypes.byref(b.desc), *args, n + spare,
              stream(), 0)
    words, got = read_output(out, m, n + spare, dtype)
    assert (words[:, n:] == 0x4a4a).all(), "written between the rows"
    want, size = mx.product(a.values, b.values)
    close(got[:, :n], want, product_bound(k, size), dtype, (m, n, k, dtype))


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 17, 33), (2, 100, 64), (3, 5, 2048), (7, 130, 257),
          (16, 64, 640), (17, 16, 128), (31, 33, 500), (32, 256, 2048), (33, 65, 129),
          (64, 64, 384), (65, 200, 1111), (100, 300, 256), (128, 128, 512), (129, 127, 4096),
          (200, 513, 896), (255, 257, 130), (256, 256, 1024), (300, 520, 768), (513, 1024, 2048),
          (1, 8192, 256), (700, 1, 384), (1, 512, 8192), (4, 2048, 1920),
          # whole rounds of the larger tiles, with and without an edge
          (1030, 4090, 300), (1024, 2050, 1024), (4096, 4096, 512), (4100, 4090, 384), (5000, 4444, 130)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(q38m, m, n, k, dtype):
    print(f"product {m} x {n} x {k} {dtype}", flush=True)
    rng = np.random.default_rng(m * 131 + n * 17 + k)
    a = Encoded(q38m, *encoded(rng, m, k), k)
    b = Encoded(q38m, *encoded(rng, n, k), k)
    check_product(q38m, a, b, k, dtype, spare=(m + n) % 3 * 5)


@pytest.mark.parametrize("m", [2, 40, 150])
def test_product_scales_at_the_ends(q38m, m):
    """Scale bytes over most of their range in both operands (products below the smallest
    normal and up to 2^120), and 255: NaN in its row or column only."""
    rng = np.random.default_rng(m)
    k = 320
    a_codes, a_scales = encoded(rng, m, k, 20, 180)
    b_codes, b_scales = encoded(rng, 70, k, 60, 180)
    a_scales[1, 3] = 255
    b_scales[7, 9] = 255
    check_product(q38m, Encoded(q38m, a_codes, a_scales, k), Encoded(q38m, b_codes, b_scales, k),
                  k, "f32")


# ---- experts' products --------------------------------------------------------

def routing(rng, tokens, top_k, experts, kind):
    """Expert ids [tokens][top_k]: even, one expert only, skewed, with dropped routes, none kept."""
    if kind == "one":
        return np.full((tokens, top_k), experts // 2, np.int32)
    if kind == "none":
        return np.full((tokens, top_k), -1, np.int32)
    if kind == "skewed":
        p = 1.0 / np.arange(1, experts + 1) ** 1.2
        ids = rng.choice(experts, size=(tokens, top_k), p=p / p.sum())
    else:
        ids = rng.integers(0, experts, size=(tokens, top_k))
    ids = ids.astype(np.int32)
    if kind == "dropped":
        ids[rng.random(ids.shape) < 0.4] = -1
        ids[0] = experts + 3
    return ids


def run_experts(q38m, w, rows, offsets, packed, top_k, routes, swiglu, dtype):
    columns = w.desc.rows // 2 if swiglu else w.desc.rows
    out, args = output(routes, columns, dtype)
    q38m.call("q38m_mx_grouped_gemm_v1", ctypes.byref(w.desc), ctypes.byref(rows.desc),
              offsets.data_ptr(), None if packed is None else packed.data_ptr(), top_k, routes,
              q38m.MX_EPILOGUE_SWIGLU if swiglu else q38m.MX_EPILOGUE_NONE, *args, stream(), 0)
    return read_output(out, routes, columns, dtype)


def want_experts(w_values, rows, offsets, packed, top_k, experts, k, swiglu):
    """The plain form and its bound, float64 [routes][columns]; nan where no expert writes."""
    n = w_values.shape[0] // experts
    routes = packed.size
    columns = n // 2 if swiglu else n
    want, bound = np.full((routes, columns), np.nan), np.zeros((routes, columns))
    for e in range(experts):
        p = np.arange(offsets[e], offsets[e + 1])
        if p.size == 0:
            continue
        y, size = mx.product(rows[packed[p] // top_k] if top_k else rows[p], w_values[e * n:(e + 1) * n])
        b = product_bound(k, size)
        if swiglu:
            # |d silu / d g| <= 1.1; exp within 3 units of its last place, the sum, the division and
            # the product one rounding each: 8 roundings cover them
            g, u, bg, bu = y[:, :columns], y[:, columns:], b[:, :columns], b[:, columns:]
            y = mx.swiglu(g, u)
            b = 1.1 * bg * (np.abs(u) + bu) + np.abs(mx.swiglu(g, 1.0)) * bu + 8 * F32_HALF * np.abs(y)
            b += 2.0 ** -126 * np.abs(g * u)  # below g = -88 the exponential is held
        want[p], bound[p] = y, b
    return want, bound


@pytest.mark.parametrize("swiglu,dtype", [(False, "f32"), (False, "bf16"), (True, "bf16"), (True, "f32")])
@pytest.mark.parametrize("tokens,top_k,experts,n,k,kind", [
    (1, 1, 1, 2, 1, "even"), (1, 10, 512, 64, 256, "even"), (3, 2, 5, 34, 100, "dropped"),
    (17, 4, 8, 96, 640, "skewed"), (40, 10, 60, 130, 129, "dropped"), (33, 3, 7, 64, 512, "one"),
    (64, 10, 512, 32, 128, "even"), (150, 2, 4, 256, 384, "skewed"), (20, 1, 1024, 18, 64, "even"),
    (300, 8, 16, 192, 256, "dropped"), (9, 2, 3, 48, 96, "none"), (513, 1, 2, 260, 1280, "even"),
    # many rows an expert: the larger tiles
    (700, 4, 12, 512, 512, "skewed"), (2400, 8, 8, 2048, 128, "dropped"), (1500, 8, 7, 1030, 640, "even")])
def test_experts(q38m, swiglu, dtype, tokens, top_k, experts, n, k, kind):
    print(f"experts {tokens} x {top_k} of {experts}, {n} x {k} {kind} swiglu {swiglu} {dtype}", flush=True)
    rng = np.random.default_rng(tokens * 31 + experts)
    offsets, packed, _ = mx.sort_routes(routing(rng, tokens, top_k, experts, kind), experts)
    w = Encoded(q38m, *encoded(rng, experts * n, k, 122, 126), k, experts)
    routes = packed.size
    for gather in (True, False):
        rows = Encoded(q38m, *encoded(rng, tokens if gather else routes, k, 122, 126), k)
        words, got = run_experts(q38m, w, rows, device(offsets), device(packed) if gather else None,
                                 top_k, routes, swiglu, dtype)
        want, bound = want_experts(w.values, rows.values, offsets, packed, top_k if gather else 0,
                                   experts, k, swiglu)
        kept = int(offsets[-1])
        assert (words[kept:] == 0x4a4a).all(), "a dropped route's row was written"
        close(got[:kept], want[:kept], bound[:kept], dtype, (tokens, kind, gather))


def test_swiglu_far_ends(q38m):
    """Gates from -1500 to 1500: the exponential at and beyond the ends of its range."""
    rng = np.random.default_rng(11)
    experts, n, k, routes = 2, 64, 128, 40
    offsets, packed = np.array([0, 17, 40], np.uint32), np.arange(40, dtype=np.uint32)
    w = Encoded(q38m, *encoded(rng, experts * n, k, 126, 131), k, experts)
    rows = Encoded(q38m, *encoded(rng, routes, k, 120, 128), k)
    words, got = run_experts(q38m, w, rows, device(offsets), None, 1, routes, True, "f32")
    want, bound = want_experts(w.values, rows.values, offsets, packed, 0, experts, k, True)
    gate = np.concatenate([mx.product(rows.values[:17], w.values[:32])[0], mx.product(rows.values[17:], w.values[64:96])[0]])
    assert gate.min() < -150 and gate.max() > 150 and (np.abs(gate) < 5).any()
    close(got, want, bound, "f32", "far ends")


def test_experts_bad_plan(q38m):
    """Offsets past the routes count as the routes, falling ones as no rows; a source row past
    the last reads the last one."""
    rng = np.random.default_rng(3)
    experts, n, k, routes = 4, 40, 256, 24
    w = Encoded(q38m, *encoded(rng, experts * n, k), k, experts)
    rows = Encoded(q38m, *encoded(rng, 12, k), k)
    packed = np.arange(routes, dtype=np.uint32)[::-1].copy()
    packed[3] = 0xffffffff
    packed[5] = 24  # token 12 of 12
    offsets = np.array([0, 10, 0x7fffffff, 16, 16], np.uint32)
    words, got = run_experts(q38m, w, rows, device(offsets), device(packed), 2, routes, False, "f32")
    values = rows.values[np.minimum(packed // 2, 11)]
    for p0, p1, e in ((0, 10, 0), (10, 24, 1)):
        want, size = mx.product(values[p0:p1], w.values[e * n:(e + 1) * n])
        close(got[p0:p1], want, product_bound(k, size), "f32", (p0, e))
