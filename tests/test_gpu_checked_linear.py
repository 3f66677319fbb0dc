"""The checked build's bf16 products: the product's results bit for bit with a clear
status, and the bits of what the experts' products hold to the range."""
import pytest

from helpers import stream, torch
from linear_cases import Matrix, Sorted, output, scratch_for, sync

pytestmark = pytest.mark.gpu

N, K = 136, 72


def operands(q38m, s, spare):
    return (Matrix(q38m, 1, s.routes, K, spare=spare), Matrix(q38m, 2, s.routes, N, spare=spare),
            Matrix(q38m, 3, N, K, experts=s.experts))


def run(q38m, call, s, rows, dc, w):
    c, d = output(q38m, s.routes, N), output(q38m, s.routes, K, "f32")
    dw = output(q38m, N, K, "f32", experts=s.experts)
    call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, *s.args(), 0, c.arg, None, stream(), 0)
    call("q38m_moe_expert_backward_rows_v1", w.arg, dc.arg, s.args()[0], None, d.arg, stream(), 0)
    call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, *s.args(), None, dw.arg, stream(), 0)
    sync()
    return c.view, d.view, dw.view


@pytest.mark.parametrize("spare", [0, 1])
def test_clear_status_and_equal_results(q38m, spare):
    t = torch()
    s = Sorted([40, 0, 3, 70, 1], 5, 119, 1, 2)
    q38m.checked_status()
    both = [run(q38m, call, s, *operands(q38m, s, spare)) for call in (q38m.call, q38m.call_checked)]
    assert q38m.checked_status() == 0
    for a, b in zip(*both):
        assert t.equal(a, b)
    x, v = Matrix(q38m, 4, 61, 2056, spare=spare), Matrix(q38m, 5, N, 2056)
    outs = []
    for call in (q38m.call, q38m.call_checked):
        y = output(q38m, 61, N)
        _, at, nbytes = scratch_for(q38m, 61, N, 2056)
        call("q38m_linear_v1", x.arg, v.arg, None, 4, None, y.arg, None, at, nbytes, stream(), 0)
        sync()
        outs.append(y.view)
    assert t.equal(*outs) and q38m.checked_status() == 0


@pytest.mark.parametrize("spare", [0, 1])
def test_what_is_held_to_the_range_is_reported(q38m, spare):
    s = Sorted([40, 0, 3, 70, 1], 5, 119, 1, 2)
    q38m.checked_status()
    s.packed[7] = 119
    run(q38m, q38m.call_checked, s, *operands(q38m, s, spare))
    assert q38m.checked_status() == q38m.CHECK_TOKEN
    s.packed[7] = 0
    s.offsets_on[2] = 30
    run(q38m, q38m.call_checked, s, *operands(q38m, s, spare))
    assert q38m.checked_status() == q38m.CHECK_OFFSETS
    s.offsets_on[2], s.offsets_on[5] = 40, 200
    run(q38m, q38m.call_checked, s, *operands(q38m, s, spare))
    assert q38m.checked_status() & q38m.CHECK_OFFSETS
