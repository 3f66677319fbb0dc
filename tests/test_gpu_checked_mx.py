"""The checked build (libq38m_checked.so) on the microscaled experts' products
and the sorted rows: the same results as the product library's, dropped routes
and places out of range among them, and a status bit for each value that no
valid plan holds."""
import ctypes

import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, stream, torch
from test_gpu_mx import Encoded, encoded, output

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu


def both(q38m, run):
    """run(call) through both libraries; its outputs, equal, and the status."""
    t = torch()
    q38m.checked_status(reset=True)
    want, got = run(q38m.call), run(q38m.call_checked)
    t.cuda.synchronize()
    for w, g in zip(want, got):
        assert t.equal(w.view(t.uint8), g.view(t.uint8))
    return q38m.checked_status(reset=True)


@pytest.mark.parametrize("routes,experts,n,k,swiglu", [
    (40, 24, 34, 130, True), (300, 130, 130, 450, False), (5000, 3, 1100, 512, True), (6000, 5, 300, 900, False)])
def test_experts(q38m, routes, experts, n, k, swiglu):
    rng = np.random.default_rng(routes)
    ids = rng.integers(-1, experts, size=(routes, 1)).astype(np.int32)
    ids[:2] = 0
    offsets, packed, _ = mx.sort_routes(ids, experts)
    tokens = (routes + 1) // 2
    w = Encoded(q38m, *encoded(rng, experts * n, k, 122, 126), k, experts)
    rows = Encoded(q38m, *encoded(rng, tokens, k, 122, 126), k)

    def status(offsets, packed):
        at, order = device(offsets), device(packed)

        def run(call):
            out, args = output(routes, n // 2 if swiglu else n, "bf16")
            call("q38m_mx_grouped_gemm_v1", ctypes.byref(w.desc), ctypes.byref(rows.desc), at.data_ptr(),
                 order.data_ptr(), 2, routes, int(swiglu), *args, stream(), 0)
            return [out]
        return both(q38m, run)

    assert status(offsets, packed) == 0
    wrong = packed.copy()
    wrong[int(offsets[-1]) // 2] = 2 * tokens
    assert status(offsets, wrong) == q38m.CHECK_TOKEN
    wrong = packed.copy()
    wrong[int(offsets[-1]):] = 0xffffffff  # behind the experts' rows nothing is read
    assert status(offsets, wrong) == 0
    wrong = offsets.copy()
    wrong[-1] = routes + 1
    assert status(wrong, packed) == q38m.CHECK_OFFSETS
    wrong = offsets.copy()
    wrong[2:] = offsets[1] // 2  # the second expert's end lies in front of its begin, behind it there are no rows
    assert offsets[1] > 0
    assert status(wrong, packed) == q38m.CHECK_OFFSETS


@pytest.mark.parametrize("dtype,width", [("bf16", 200), ("bf16", 5), ("f32", 70)])
def test_rows(q38m, dtype, width):
    t = torch()
    tokens, top_k = 37, 3
    routes = tokens * top_k
    rng = np.random.default_rng(width)
    ids = rng.integers(-1, 6, size=(tokens, top_k)).astype(np.int32)
    _, _, inverse = mx.sort_routes(ids, 6)
    kind = t.bfloat16 if dtype == "bf16" else t.float32
    code = q38m.DTYPE_BF16 if dtype == "bf16" else q38m.DTYPE_F32
    x, rows = (t.randn(n, width, device="cuda").to(kind) for n in (tokens, routes))
    w = t.rand(tokens, top_k, device="cuda")

    def status(inverse):
        at = device(inverse)

        def run(call):
            out, y, d_rows, d_w = t.zeros_like(rows), t.zeros_like(x), t.zeros_like(rows), t.zeros_like(w)
            shape = (tokens, top_k, width)
            call("q38m_moe_permute_rows_v1", x.data_ptr(), code, at.data_ptr(), *shape, out.data_ptr(), stream(), 0)
            call("q38m_moe_unpermute_rows_v1", rows.data_ptr(), code, at.data_ptr(), w.data_ptr(), *shape,
                 y.data_ptr(), stream(), 0)
            call("q38m_moe_unpermute_backward_v1", x.data_ptr(), rows.data_ptr(), code, at.data_ptr(), w.data_ptr(),
                 *shape, d_rows.data_ptr(), d_w.data_ptr(), stream(), 0)
            return [out, y, d_rows, d_w]
        return both(q38m, run)

    assert (inverse == mx.DROPPED).any() and status(inverse) == 0
    wrong = inverse.copy()
    wrong[np.nonzero(inverse != mx.DROPPED)[0][-1]] = routes
    assert status(wrong) == q38m.CHECK_ROUTE
