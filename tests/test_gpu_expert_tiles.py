"""The experts' forward products on every tile shape, as the library plans them: sizes
whose products run on tiles, and not on the form for few rows that small ones of the
same shape's rule would take."""
import random

import pytest

from linear_cases import Sorted, check_experts
from linear_tiles import SHAPES, tiles_of
from test_gpu_linear_tiles import counts_of, found

pytestmark = pytest.mark.gpu

EXPERTS = 24


def sizes(rng):
    return max(1, int(2 ** rng.uniform(0, 14))), 16 * rng.randint(1, 160), 8 * rng.randint(1, 100)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows,columns,several", [(*s, several) for s in sorted(SHAPES) for several in (False, True)])
def test_forward(q38m, rows, columns, several, swiglu):
    """several: more tiles than the card holds workgroups."""
    def plan(routes, n, k):
        return tiles_of(routes, n, k, EXPERTS, swiglu, along=True)

    def wanted(t):
        return t[:2] == (rows, columns) and t.waves == 0 and (t.at_most > t.held) == several

    routes, n, k = found(wanted, sizes, plan)
    rng = random.Random(rows + several)
    s = Sorted(counts_of(rng, EXPERTS, routes), 3, routes + 3, 1, 5)
    assert plan(s.routes, n, k)[:2] == (rows, columns) and plan(s.routes, n, k).waves == 0
    check_experts(q38m, 1, s, n, k, swiglu, "bf16", "bf16" if swiglu else None, tokens=routes + 3)
    check_experts(q38m, 2, s, n, k, swiglu, "f32", None, tokens=routes + 3)
    check_experts(q38m, 3, Sorted(counts_of(rng, EXPERTS, routes)), n, k, swiglu, "f32", "f32" if swiglu else None)
