"""Pins of the plain 64-bit forms that the GPU tests of the microscaled rows
and the sorted tokens compare with (oracle/mx_oracle.py): the roundings of
the 4-bit format one by one, scales at the ends of their range, and the sort
and its way back on small cases worked by hand."""
import numpy as np
import pytest

from conftest import load_oracle

load_oracle()
import mx_oracle as mx  # noqa: E402


def codes_of(x):
    codes, scales, values = mx.quantize(np.asarray([x]))
    both = np.stack((codes & 15, codes >> 4), -1).reshape(-1)
    return both[:len(x)], scales[0], values[0]


@pytest.mark.parametrize("value,index", [
    (0.0, 0), (0.25, 0), (0.2500001, 1), (0.5, 1), (0.75, 2), (1.0, 2), (1.25, 2), (1.26, 3),
    (1.5, 3), (1.75, 4), (2.0, 4), (2.5, 4), (2.51, 5), (3.0, 5), (3.5, 6), (4.0, 6), (5.0, 6),
    (5.01, 7), (6.0, 7), (7.9, 7)])
def test_every_rounding(value, index):
    """A 4.0 in the block fixes the scale at 1 (byte 127)."""
    code, scales, values = codes_of([value, -value, 4.0])
    assert scales[0] == 127
    assert code[0] == index and code[1] == index + 8
    assert values[0] == mx.MAGNITUDES[index] and values[1] == -mx.MAGNITUDES[index]


@pytest.mark.parametrize("top,byte", [
    (0.0, 0), (2.0 ** -149, 0), (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1),
    (1.0, 125), (7.99, 127), (8.0, 128), (3.3895313892515355e38, 252)])
def test_scale_bytes(top, byte):
    assert codes_of([0.0, -top])[1][0] == byte


def test_blocks_that_are_not_finite():
    x = np.ones(96)
    x[5], x[70] = np.nan, -np.inf
    _, scales, values = codes_of(x)
    assert list(scales[:3]) == [255, 125, 255]
    assert np.isnan(values[:32]).all() and np.isnan(values[64:]).all()
    assert (values[32:64] == 1).all()


def test_decode_is_the_inverse():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(7, 200)) * np.exp(rng.normal(size=(7, 1)) * 20)
    codes, scales, values = mx.quantize(x)
    assert codes.shape == (7, 128) and scales.shape == (7, 8)
    assert np.array_equal(mx.decode(codes, scales, 200), values)
    again = mx.quantize(values)
    assert np.array_equal(mx.decode(again[0], again[1], 200), values)
    assert (codes[:, 100:] == 0).all() and (scales[:, 7:] == 0).all()


def test_sort_by_hand():
    ids = [[2, 0], [-1, 2], [5, 0]]
    offsets, packed, inverse = mx.sort_routes(ids, 3)
    assert list(offsets) == [0, 2, 2, 4]
    assert list(packed) == [1, 5, 0, 3, 2, 4]
    assert list(inverse) == [2, 0, mx.DROPPED, 3, mx.DROPPED, 1]
    rows = np.arange(6.0)[:, None] + [[0.0, 10.0]]
    weights = [[1.0, 2.0], [np.nan, 3.0], [np.inf, -1.0]]
    y, _ = mx.unpermute(rows, inverse, weights, 3)
    assert np.array_equal(y, [[2.0, 32.0], [9.0, 39.0], [-1.0, -11.0]])
    dy = np.array([[1.0, 1.0], [2.0, 0.0], [0.0, 3.0]])
    d_rows, d_weights, _ = mx.unpermute_backward(dy, rows, inverse, weights)
    assert np.array_equal(d_rows[:4], [[2, 2], [0, -3], [1, 1], [6, 0]])
    assert np.isnan(d_rows[4:]).all()
    assert np.array_equal(d_weights, [[14, 10], [0, 6], [0, 33]])
