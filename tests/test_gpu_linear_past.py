"""Dense products whose rows stay in the caches and ones whose rows go past them: C and what
is added to it just below, at and above 128 MB together.  The operands are small whole
numbers, so that an output is the exact sum and the residual, rounded: bit for bit."""
import pytest

from helpers import stream, torch
from linear_cases import Matrix, arg, output, scratch_for, sync
from linear_tiles import tiles_of
from test_gpu_linear_residual import typed, whole

pytestmark = pytest.mark.gpu

STAY = 1 << 27  # bytes


@pytest.mark.parametrize("name", ["q38m_linear_v1", "q38m_linear_backward_input_v1"])
@pytest.mark.parametrize("columns,k,tile", [(8192, 1032, 256), (128, 64, 128)])
@pytest.mark.parametrize("out,residual", [("bf16", None), ("f32", None), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"),
                                          ("f32", "bf16")])
def test_both_sides(q38m, name, columns, k, tile, out, residual):
    t = torch()
    size = {None: 0, "bf16": 2, "f32": 4}
    at = STAY // (columns * (size[out] + size[residual]))
    forward = name == "q38m_linear_v1"
    w = whole(q38m, 2, columns, k) if forward else whole(q38m, 2, k, columns)
    for rows in (at - 3, at, at + 5):
        assert tiles_of(rows, columns, k, along=forward)[:2] == (tile, tile)
        print(name, rows, columns, k, out, residual, flush=True)
        x = whole(q38m, 1, rows, k)
        r = residual and Matrix(q38m, 3, rows, columns, residual, sigma=2.0 ** 20)
        y = output(q38m, rows, columns, out)
        _, room, nbytes = scratch_for(q38m, rows, columns, k) if forward else scratch_for(q38m, rows, k, columns)
        q38m.call(name, x.arg, w.arg, None, 0, arg(r), y.arg, *((None,) if forward else ()), room, nbytes, stream(), 0)
        sync()
        want = x.values @ (w.values.T.contiguous() if forward else w.values)
        if r:
            want = want + r.values
        assert t.equal(y.got(), typed(want, out).double())
