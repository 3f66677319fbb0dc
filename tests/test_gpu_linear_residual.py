"""What a residual costs a sum: one rounding, on every kernel.  The operands are small
whole numbers, so that every order of a product's sum is exact in fp32 (at most 8,200
terms of 4), and an output is the fp32 rounding of the exact sum and the residual, then
its type's: compared bit for bit, with residuals 2^5 times the largest sums and more."""
import random

import pytest

from helpers import stream, torch
from linear_cases import Matrix, Sorted, generator, lin, output, scratch_for, sync
from linear_tiles import tiles_of
from test_gpu_linear_tiles import KINDS, counts_of, found, spread

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")]  # of the output and the residual


def whole(q38m, seed, rows, columns, **more):
    t = torch()
    values = t.randint(-2, 3, (rows, columns), generator=generator(seed), device="cuda")
    return Matrix(q38m, seed, rows, columns, fill=values.bfloat16(), **more)


def typed(values, dtype):
    t = torch()
    return values.float() if dtype == "f32" else values.float().bfloat16()


def check(q38m, name, operands, product, rows, columns, types, room, experts=1, after=(), spare=0):
    """The call with the residual apart, and in place where the types are one."""
    out, residual = types
    scratch = room[1:]
    r = Matrix(q38m, 3, rows, columns, residual, sigma=2.0 ** 20, spare=spare, experts=experts)
    want = typed(product.reshape(r.values.shape) + r.values, out)
    y = output(q38m, rows, columns, out, spare, experts=experts)
    places = [(r, y)] + ([(r, r)] if out == residual else [])
    for given, to in places:
        q38m.call(name, *operands, given.arg, to.arg, *after, *scratch, stream(), 0)
        sync()
        got = to.got()
        assert torch().equal(got, want.double()), (name, rows, columns, types, given is to,
                                                   float((got - want.double()).abs().max()))


def check_forward(q38m, m, n, k, types, **spares):
    print("forward", m, n, k, types, flush=True)
    x, w = whole(q38m, 1, m, k, **spares), whole(q38m, 2, n, k, **spares)
    check(q38m, "q38m_linear_v1", (x.arg, w.arg, None, 0), x.values @ w.values.T, m, n, types,
          scratch_for(q38m, m, n, k), after=(None,))


def check_input(q38m, m, n, k, types, **spares):
    print("input", m, n, k, types, flush=True)
    dz, w = whole(q38m, 1, m, n, **spares), whole(q38m, 2, n, k, **spares)
    check(q38m, "q38m_linear_backward_input_v1", (dz.arg, w.arg, None, 0), dz.values @ w.values, m, k, types,
          scratch_for(q38m, m, n, k))


def check_weight(q38m, m, n, k, types, **spares):
    print("weight", m, n, k, types, flush=True)
    dz, x = whole(q38m, 1, m, n, **spares), whole(q38m, 2, m, k, **spares)
    check(q38m, "q38m_linear_backward_weight_v1", (dz.arg, x.arg), dz.values.T.contiguous() @ x.values, n, k, types,
          scratch_for(q38m, m, n, k), after=(None,))


@pytest.mark.parametrize("rows,columns,cut,several", KINDS)
def test_on_tiles(q38m, rows, columns, cut, several):
    def wanted(t):
        return t[:2] == (rows, columns) and (t.parts > 1) == cut and (t.at_most > t.held) == several

    m, n, k = found(wanted, spread, tiles_of)
    for types in TYPES:
        check_input(q38m, m, k, n, types)
        if not tiles_of(m, n, k, along=True).waves:
            check_forward(q38m, m, n, k, types)
    if rows >= 64 and not (several and cut):
        m, n, k = found(wanted, spread, lambda m, n, k: tiles_of(n, k, m, ragged=True))
        for types in TYPES:
            check_weight(q38m, m, n, k, types)


# long K on few rows; K in parts; rows that start anywhere, copied and not; edges of every tile
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 8192), (5, 264, 2048), (61, 1024, 2056), (300, 256, 8192), (1030, 520, 640),
                                   (17, 333, 501), (131, 1001, 1003), (700, 513, 65)])
def test_on_the_others(q38m, m, n, k, types):
    for spares in ({}, {"spare": 3, "shift": 1}):
        check_forward(q38m, m, n, k, types, **spares)
        check_input(q38m, m, n, k, types, **spares)
        check_weight(q38m, m, n, k, types, **spares)


@pytest.mark.parametrize("rows,columns,several", [(256, 256, False), (256, 256, True), (128, 128, False), (128, 128, True),
                                                  (64, 64, False), (64, 64, True)])
@pytest.mark.parametrize("types", TYPES)
def test_experts_weights(q38m, rows, columns, several, types):
    """Weight gradients added to what was there, experts without rows among them, on tiles and (rows that
    start anywhere) on the kernel for those."""
    t, experts = torch(), 24
    rng = random.Random(rows + several)

    def wanted(p):
        return p[:2] == (rows, columns) and (p.at_most > p.held) == several

    n, k, routes = found(wanted, lambda rng: (8 * rng.randint(1, 200), 8 * rng.randint(1, 200), rng.randint(1, 8000)),
                         lambda n, k, r: tiles_of(n, k, r, experts, ragged=True))
    counts = counts_of(rng, experts, routes)
    counts[3] += counts[4]
    counts[4] = 0
    for spare in (0, 1):
        for tokens in (0, routes + 5):
            s = Sorted(counts, 5, tokens, 1, 6)
            print("experts", n, k, routes, types, spare, tokens, flush=True)
            dc, x = whole(q38m, 1, s.routes, n, spare=spare), whole(q38m, 2, tokens or s.routes, k, spare=spare)
            product = lin.experts_backward_weights(dc.values, x.values, s.offsets, experts, s.source)
            assert not product[4].any()
            check(q38m, "q38m_moe_expert_backward_weights_v1", (dc.arg, x.arg, *s.args()), product, n, k, types, (None,),
                  experts, spare=spare)
