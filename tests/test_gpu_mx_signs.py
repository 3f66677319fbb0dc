"""Signs of what the quantiser's codes stand for, zeros among them, wherever the
value is no NaN, and fp32 values beside every border between two codes."""
import numpy as np
import pytest

from conftest import load_oracle
from test_gpu_mx import bf16_words, run_quantize, widen

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu


def check(q38m, x, dtype):
    words = bf16_words(x) if dtype == "bf16" else x.astype(np.float32)
    exact = widen(words) if dtype == "bf16" else words.astype(np.float64)
    codes, scales, values = mx.quantize(exact)
    got = run_quantize(q38m, words.reshape(-1), *x.shape, x.shape[1], dtype)
    assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales)
    live = ~np.isnan(values)
    assert np.array_equal(np.isnan(got[2]), ~live)
    assert np.array_equal(got[2][live], values[live])
    assert np.array_equal(np.signbit(got[2])[live], np.signbit(values)[live])
    return values


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_signs_of_every_bf16(q38m, dtype):
    """Every bf16 pattern beside values of many exponents, in blocks with and without NaN."""
    patterns = widen(np.arange(65536, dtype=np.uint32).astype(np.uint16)).reshape(-1, 16)
    blocks = []
    for field in range(1, 255, 12):
        top = widen(np.full((4096, 1), field << 7, np.uint16))
        blocks.append(np.concatenate((patterns, np.broadcast_to(top, (4096, 16))), 1))
    x = np.concatenate(blocks, 1)
    with np.errstate(invalid="ignore"):
        values = check(q38m, x, dtype)
    zero = values == 0
    assert np.isnan(values).any() and np.signbit(values)[zero].any() and (~np.signbit(values)[zero]).any()


def test_values_beside_the_borders(q38m):
    """Under scales from the least to nearly the largest: each border between two codes, and one
    and two steps of fp32 to either side of it, of both signs."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    near = [borders]
    for direction in (np.float32(0), np.float32(np.inf)):
        step = borders
        for _ in range(2):
            step = np.nextafter(step, direction, dtype=np.float32)
            near.append(step)
    near = np.concatenate(near)
    near = np.concatenate((near, -near))
    rows = []
    for exponent in (-126, -125, -100, -20, 0, 20, 100, 124):
        for first in range(0, near.size, 31):
            block = np.zeros(32, np.float32)
            part = near[first:first + 31]
            block[:part.size] = part * np.float32(2.0) ** np.float32(exponent)
            block[31] = np.float32(4.0) * np.float32(2.0) ** np.float32(exponent)  # the scale is 2^exponent
            rows.append(block)
    check(q38m, np.stack(rows).astype(np.float64), "f32")
