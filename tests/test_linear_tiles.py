"""The bf16 products' tile rule: every shape is some product's, parts of K are whole and
not empty, and the scratch that a layer is told to bring is what its products need."""
import random

from linear_tiles import FEW, SHAPES, tiles_of


def sizes(rng):
    def one(top):
        return max(1, int(2 ** rng.uniform(0, top)))
    return one(17), one(15), one(15)


def test_every_shape_is_taken():
    rng = random.Random(1)
    dense, ragged, grouped, few = set(), set(), set(), set()
    for _ in range(4000):
        m, n, k = sizes(rng)
        dense.add(tiles_of(m, n, k)[:2])
        ragged.add(tiles_of(n, k, m, ragged=True)[:2])
        experts = rng.choice((1, 8, 60, 512))
        grouped.add(tiles_of(m, n, k, experts)[:2])
        assert tiles_of(n, k, m, experts, ragged=True).rows >= 64
        assert tiles_of(m, n, k, experts, wide=False)[:2] != (256, 256)
        forward = tiles_of(m, n, k, along=True)
        if forward.waves:
            few.add((*forward[:2], forward.waves))
            assert forward.workgroups <= 512 and forward.parts == 1
        else:
            assert forward == tiles_of(m, n, k)
            assert -(-m // 16) * -(-n // 32) > 256
        swiglu = tiles_of(m, 2 * n, k, experts, True, along=True)
        assert not swiglu.waves or swiglu.columns == 32
    assert dense == grouped == SHAPES and few == FEW
    assert ragged == {(256, 256), (128, 128), (64, 64)}


def test_parts_of_k():
    rng = random.Random(2)
    cut = 0
    for _ in range(4000):
        m, n, k = sizes(rng)
        t = tiles_of(m, n, k)
        cut += t.parts > 1
        assert t.parts == 1 or t.each % 64 == 0
        assert (t.parts - 1) * t.each < k <= t.parts * t.each
        assert t.workgroups % 8 == 0 and t.workgroups <= t.held
        assert t.workgroups >= min(t.held, t.parts * t.at_most)
        assert t.parts == 1 or t.parts * m * n * 4 <= 1.1 * 2 ** 28
    assert cut > 400


def test_scratch_holds_the_parts(q38m):
    rng = random.Random(3)
    for _ in range(2000):
        m, n, k = sizes(rng)
        scratch = q38m.lib().q38m_linear_scratch_bytes(m, n, k)
        for t, values in ((tiles_of(m, n, k, along=True), m * n), (tiles_of(m, k, n), m * k),
                          (tiles_of(n, k, m, ragged=True), n * k)):
            assert scratch >= (4 * t.parts * values if t.parts > 1 else 0)


def test_bounds_of_the_experts_tiles():
    """No routing has more tiles than the launch counts with."""
    rng = random.Random(4)
    for _ in range(500):
        experts, routes = rng.choice((1, 7, 64, 512)), int(2 ** rng.uniform(0, 16))
        counts = [0] * experts
        for _ in range(rng.randint(1, 40)):
            counts[rng.randrange(experts)] += routes // 40
        counts[rng.randrange(experts)] += routes - sum(counts)
        n, k = 8 * rng.randint(1, 300), 8 * rng.randint(1, 300)
        t = tiles_of(routes, n, k, experts)
        assert sum(-(-c // t.rows) for c in counts) * -(-n // t.columns) <= t.at_most
        t = tiles_of(n, k, routes, experts, ragged=True)
        assert sum(c > 0 for c in counts) * -(-n // t.rows) * -(-k // t.columns) <= t.at_most
