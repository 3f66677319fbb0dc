"""The bf16 products on every tile shape, with K cut and whole, several tiles a
workgroup, and edges of rows, columns and K inside a tile."""
import random

import pytest

from linear_cases import Sorted, check_backward_input, check_backward_weight, check_experts, check_experts_rows, \
    check_experts_weights, check_linear
from linear_tiles import FEW, SHAPES, tiles_of

pytestmark = pytest.mark.gpu


def found(wanted, sizes, plan, tries=40000):
    """Sizes of the least work whose plan is wanted."""
    rng, best = random.Random(7), None
    for _ in range(tries):
        s = sizes(rng)
        if min(s[1:]) < 72 or max(s) < 200:  # a few stages of K, an edge of the columns
            continue
        work = s[0] * s[1] * s[2]
        if (best is None or work < best[0]) and work < 2e11 and wanted(plan(*s)):
            best = work, s
    assert best, "no product"
    return best[1]


def spread(rng):
    """Odd sizes of rows, rows that start at 16 bytes."""
    def one(top):
        return max(1, int(2 ** rng.uniform(0, top)))
    return one(13), 8 * one(9.5), 8 * one(10)


# so many rows of 16 that they are more tiles than workgroups run on larger ones
KINDS = [(*s, cut, several) for s in sorted(SHAPES) for cut, several in ((False, False), (True, False), (False, True))
         if not (several and s[0] == 16)]


@pytest.mark.parametrize("rows,columns,cut,several", KINDS)
def test_dense(q38m, rows, columns, cut, several):
    """cut: K in parts; several: more tiles than the card holds workgroups."""
    def wanted(t):
        return t[:2] == (rows, columns) and (t.parts > 1) == cut and (t.at_most > t.held) == several

    m, n, k = found(wanted, spread, tiles_of)
    if not tiles_of(m, n, k, along=True).waves:
        check_linear(q38m, 1, m, n, k, "gelu", "f32", "bf16", "bf16", "bf16")
        check_linear(q38m, 2, m, n, k, "none", None, "f32", "f32")
    check_backward_input(q38m, 3, m, k, n, "silu", "bf16", "bf16")
    check_backward_input(q38m, 4, m, k, n, "none", None, "f32")
    if rows <= 64:  # forward products of such tiles: with more workgroups than the form for few rows takes
        m, n, k = found(lambda t: wanted(t) and not t.waves, spread, lambda m, n, k: tiles_of(m, n, k, along=True)) \
            if rows > 16 and not cut else (24, 8 * 1100, 200)
        check_linear(q38m, 8, m, n, k, "gelu", "f32", "bf16", "bf16", "bf16")
        check_linear(q38m, 9, m, n, k, "none", None, "f32", "f32")
    if rows >= 64 and not (several and cut):
        def transposed(m, n, k):
            return tiles_of(n, k, m, ragged=True)
        m, n, k = found(wanted, lambda rng: tuple(spread(rng)), transposed)
        check_backward_weight(q38m, 5, m, n, k, "f32", "f32")
        check_backward_weight(q38m, 6, m, n, k, None, "bf16")
        check_backward_weight(q38m, 7, m, n, k, "bf16", "bf16", spare=(8, 8, 3))


@pytest.mark.parametrize("rows,columns,waves", sorted(FEW))
def test_few_rows(q38m, rows, columns, waves):
    """Dense and by expert: one row, tiles just full and begun, K of less than a stage a wave, odd K."""
    for m, n, k in ((1, 8 * 40, 2048), (1, 300, 8), (16, 1000, 520), (17, 64, 2056), (40, 3000, 136), (100, 2000, 72),
                    (129, 72, 1000), (1, 8192, 264), (9, 4100, 600)):
        t = tiles_of(m, n, k, along=True)
        if (t.columns, t.waves) == (columns, waves):
            check_linear(q38m, 1, m, n, k, "gelu", "f32", "bf16", "bf16", "bf16")
            check_linear(q38m, 2, m, n, k, "none", None, "f32", "f32", spare=(8, 16, 3))
    seen = 0
    for counts, n, k in (([1, 0, 2], 72, 520), ([16, 17, 1, 0], 136, 72), ([5] * 8, 544, 200), ([1] * 10, 1024, 136),
                         ([3, 40, 8], 1600, 1000), ([7, 0, 9, 15], 320, 8)):
        s = Sorted(counts, 2, sum(counts) + 2, 1, 3)
        for swiglu in (False, True):
            t = tiles_of(s.routes, n, k, len(counts), swiglu, along=True)
            if (t.columns, t.waves) == (columns, waves):
                seen += 1
                check_experts(q38m, 3, s, n, k, swiglu, "bf16", "bf16" if swiglu else None, tokens=s.routes)
                check_experts(q38m, 4, s, n, k, swiglu, "f32", "f32" if swiglu else None, spare=(0, 8, 0),
                              tokens=s.routes)
    assert seen


def counts_of(rng, experts, routes):
    cuts = sorted(rng.randint(0, routes) for _ in range(experts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [routes])]


GROUPED = [(*s, several) for s in sorted(SHAPES) for several in (False, True)]


@pytest.mark.parametrize("rows,columns,several", GROUPED)
def test_experts(q38m, rows, columns, several):
    experts = 24
    rng = random.Random(rows + several)

    def sizes(rng):
        return max(1, int(2 ** rng.uniform(0, 14))), 16 * rng.randint(1, 160), 8 * rng.randint(1, 100)

    for swiglu in (False, True):
        def wanted(t):
            return t[:2] == (rows, columns) and (t.at_most > t.held) == several
        routes, n, k = found(wanted, sizes, lambda r, n, k: tiles_of(r, n, k, experts, swiglu))
        s = Sorted(counts_of(rng, experts, routes), 3, routes + 3, 1, 5)
        check_experts(q38m, 1, s, n, k, swiglu, "bf16", "bf16" if swiglu else None, tokens=routes + 3)
        check_experts(q38m, 2, s, n, k, swiglu, "f32", None, tokens=routes + 3)
        if swiglu and rows == 256:
            continue
        routes, k, n = found(wanted, sizes, lambda r, k, n: tiles_of(r, k, n, experts, False, False, not swiglu))
        s = Sorted(counts_of(rng, experts, routes), 3)
        check_experts_rows(q38m, 3, s, n, k, "bf16" if swiglu else None, "bf16")
        check_experts_rows(q38m, 4, s, n, k, "f32" if swiglu else None, "f32")
    if rows < 64:
        return
    n, k, routes = found(wanted, lambda rng: (8 * rng.randint(1, 200), 8 * rng.randint(1, 200), rng.randint(1, 8000)),
                         lambda n, k, r: tiles_of(n, k, r, experts, ragged=True))
    counts = counts_of(rng, experts, routes)
    counts[3] += counts[4]
    counts[4] = 0
    s = Sorted(counts, 5, routes + 5, 1, 6)
    check_experts_weights(q38m, 5, s, n, k, "f32", "f32", tokens=routes + 5)
    check_experts_weights(q38m, 6, Sorted(counts), n, k, "bf16", "bf16")
    check_experts_weights(q38m, 7, s, n, k, None, "bf16", tokens=routes + 5)
