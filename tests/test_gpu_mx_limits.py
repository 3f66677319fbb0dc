"""The largest calls that the header allows, and rows just past them."""
import ctypes

import numpy as np
import pytest

from conftest import load_oracle
from helpers import host, stream, torch

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu


def test_most_rows_of_a_quantisation(q38m):
    """2^23 rows in one call; one more is refused, and is two calls on parts of the buffers."""
    t = torch()
    rows, columns = (1 << 23) + 1, 2
    x = t.empty(rows, columns, dtype=t.float32, device="cuda").normal_()
    codes = t.full((rows, 64), 0xa5, dtype=t.uint8, device="cuda")
    scales = t.full((rows, 4), 0xa5, dtype=t.uint8, device="cuda")

    def quantise(first, count):
        desc = q38m.MxMatrix(codes[first].data_ptr(), scales[first].data_ptr(), 1, count, columns)
        q38m.call("q38m_mx_quantize_v1", x[first].data_ptr(), q38m.DTYPE_F32, columns, ctypes.byref(desc), None,
                  stream(), 0)

    with pytest.raises(q38m.InvalidArgument):
        quantise(0, rows)
    quantise(0, rows - 1)
    assert (codes[-1] == 0xa5).all() and (scales[-1] == 0xa5).all()
    quantise(rows - 1, 1)
    at = np.concatenate((np.arange(300), np.arange(0, rows, 7919), np.arange(rows - 300, rows)))
    some = t.as_tensor(at, device="cuda")
    want_codes, want_scales, _ = mx.quantize(host(x[some], np.float32))
    assert np.array_equal(host(codes[some], np.uint8), want_codes)
    assert np.array_equal(host(scales[some], np.uint8), want_scales)
    assert not codes[:, 1:].any() and not scales[:, 1:].any()


def test_rows_one_over_the_other_are_refused(q38m):
    t = torch()
    x = t.zeros(6, 64, dtype=t.bfloat16, device="cuda")
    for view in (x[:1].expand(4, 64), x.view(-1).as_strided((5, 64), (63, 1))):
        with pytest.raises(q38m.InvalidArgument):
            q38m.mx_quantize(view)
