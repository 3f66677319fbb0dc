"""The experts' products in bf16 over sorted rows and their gradients, against plain
forms in 64 bits (oracle/linear_oracle.py).  Operands lie among NaN, outputs among
guards; the bounds are derived in linear_cases.py."""
import ctypes

import numpy as np
import pytest

from helpers import stream, torch
from linear_cases import (Matrix, Sorted, check_experts, check_experts_rows, check_experts_weights, close,
                          lin, output, sync)

pytestmark = pytest.mark.gpu


def ragged(count, total, seed):
    """`total` rows over `count` experts, unevenly, some without any."""
    rng = np.random.default_rng(seed)
    p = rng.random(count) ** 4
    p[rng.random(count) < 0.3] = 0
    if p.sum() == 0:
        p[:] = 1
    return rng.multinomial(total, p / p.sum()).tolist()


# counts, dropped, tokens (0: rows as they lie), top_k
SORTS = [([1], 0, 0, 1), ([0, 3, 0], 0, 4, 1), ([0, 0], 5, 5, 1), ([1] * 10, 0, 1, 10), ([63, 64, 65, 0, 1], 7, 0, 1),
         ([15, 16, 17, 31, 33], 3, 60, 2), ([127, 0, 128, 129], 1, 200, 4), (ragged(60, 1000, 1), 24, 512, 2),
         (ragged(1024, 3000, 2), 0, 1500, 2), ([255, 257, 256, 700], 20, 0, 1), ([2000], 0, 300, 8)]
SHAPES = [(2, 8), (16, 16), (64, 72), (130, 136), (256, 264), (72, 520)]


@pytest.mark.parametrize("counts,dropped,tokens,top_k", SORTS)
def test_forward(q38m, counts, dropped, tokens, top_k):
    s = Sorted(counts, dropped, tokens, top_k, 3)
    for i, (n, k) in enumerate(SHAPES):
        check_experts(q38m, i, s, n, k, out=("bf16", "f32")[i % 2], tokens=tokens)
        check_experts(q38m, i, s, n, k, True, ("f32", "bf16")[i % 2], (None, "bf16", "f32")[i % 3], tokens=tokens)


@pytest.mark.parametrize("counts,dropped,tokens,top_k", SORTS)
def test_row_gradient(q38m, counts, dropped, tokens, top_k):
    s = Sorted(counts, dropped)
    for i, (n, k) in enumerate(SHAPES):
        check_experts_rows(q38m, i, s, n, k, out=("bf16", "f32")[i % 2])
        check_experts_rows(q38m, i, s, n, k, ("bf16", "f32")[i // 2 % 2], ("f32", "bf16")[i % 2])


@pytest.mark.parametrize("counts,dropped,tokens,top_k", SORTS)
def test_weight_gradient(q38m, counts, dropped, tokens, top_k):
    s = Sorted(counts, dropped, tokens, top_k, 4)
    for i, (n, k) in enumerate(SHAPES if len(counts) < 100 else SHAPES[:3]):
        check_experts_weights(q38m, i, s, n, k, out=("bf16", "f32")[i % 2], tokens=tokens)
        check_experts_weights(q38m, i, s, n, k, ("f32", "bf16")[i % 2], ("f32", "bf16")[i % 2], tokens=tokens)


@pytest.mark.parametrize("spare,shift", [((8, 0, 0), (0, 0, 0)), ((0, 16, 8), (8, 8, 0)), ((24, 8, 3), (0, 0, 1)),
                                         ((1, 0, 0), (0, 0, 0)), ((0, 3, 0), (0, 0, 0)), ((13, 5, 1), (3, 7, 1))])
@pytest.mark.parametrize("tokens", [0, 150])
def test_strides(q38m, spare, shift, tokens):
    s = Sorted([3, 0, 70, 130, 9], 11, tokens, 2, 5)
    for n, k in ((136, 72), (36, 39)):
        check_experts(q38m, 6, s, n, k, spare=spare, shift=shift, tokens=tokens)
        check_experts(q38m, 7, s, n, k, True, "f32", "bf16", spare, shift, tokens)
        check_experts_rows(q38m, 8, s, n, k, None, "f32", spare, shift)
        check_experts_rows(q38m, 9, s, n, k, "bf16", "bf16", spare, shift)
        check_experts_weights(q38m, 10, s, n, k, "bf16", "bf16", spare, shift, tokens)


def test_model_geometry(q38m):
    """Gate/up and down of the library's layer, ten experts a token, 64 of the 512 experts."""
    s = Sorted(ragged(64, 700, 7), 20, 72, 10, 8)
    plain = Sorted(ragged(64, 700, 7), 20)
    check_experts(q38m, 1, s, 1024, 2048, True, "bf16", "bf16", tokens=72)
    check_experts(q38m, 2, plain, 2048, 512)
    check_experts_rows(q38m, 3, plain, 2048, 512, "bf16")
    check_experts_rows(q38m, 4, plain, 1024, 2048)
    check_experts_weights(q38m, 5, plain, 2048, 512)
    check_experts_weights(q38m, 6, s, 1024, 2048, "f32", "f32", tokens=72)


def test_masked_places_do_not_count(q38m):
    """NaN and infinities in rows of no expert, in weights of experts without rows and in the rows of
    other experts do not reach an expert's results."""
    t = torch()
    s = Sorted([5, 0, 40, 19], 6)
    n, k = 72, 136
    rows, dc = Matrix(q38m, 1, s.routes, k), Matrix(q38m, 2, s.routes, n)
    w = Matrix(q38m, 3, n, k, experts=4)
    rows.view[64:], dc.view[64:] = float("nan"), float("inf")  # of no expert
    rows.view[2], dc.view[3] = float("inf"), float("nan")       # of expert 0
    w.view[n:2 * n] = float("nan")                              # of expert 1, without rows
    c, d, dw = output(q38m, s.routes, n, "f32"), output(q38m, s.routes, k, "f32"), output(q38m, n, k, "f32", experts=4)
    q38m.call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, *s.args(), 0, c.arg, None, stream(), 0)
    q38m.call("q38m_moe_expert_backward_rows_v1", w.arg, dc.arg, s.args()[0], None, d.arg, stream(), 0)
    q38m.call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, *s.args(), None, dw.arg, stream(), 0)
    sync()
    c, d, dw = c.got(), d.got(), dw.got()
    clean = [i for i in range(64) if i != 2]
    assert c[clean].isfinite().all() and not c[2].isfinite().any() and (c[64:] == 7777).all()
    clean = [i for i in range(64) if i != 3]
    assert d[clean].isfinite().all() and d[3].isnan().all() and (d[64:] == 7777).all()
    assert dw[0].isnan().all() and (dw[1] == 0).all() and dw[2:].isfinite().all()


def test_offsets_that_fall_or_pass_the_routes(q38m):
    """Offsets past the routes are taken as them, an end not behind its begin has no rows."""
    t = torch()
    n, k, routes = 40, 64, 30
    w = Matrix(q38m, 1, n, k, experts=4)
    rows, dc = Matrix(q38m, 2, routes, k), Matrix(q38m, 3, routes, n)
    for offsets in ([0, 10, 5, 5, 5], [4, 4, 20, 99, 1000], [50, 60, 70, 80, 90]):
        at = t.tensor(offsets, dtype=t.int32, device="cuda")
        c, d, dw = output(q38m, routes, n, "f32"), output(q38m, routes, k, "f32"), output(q38m, n, k, "f32", experts=4)
        q38m.call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, at.data_ptr(), None, 1, 0, c.arg, None, stream(), 0)
        q38m.call("q38m_moe_expert_backward_rows_v1", w.arg, dc.arg, at.data_ptr(), None, d.arg, stream(), 0)
        q38m.call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, at.data_ptr(), None, 1, None, dw.arg,
                  stream(), 0)
        sync()
        for got, want in ((c.got(), lin.experts(rows.values, w.values, offsets, routes)),
                          (d.got(), lin.experts_backward_rows(dc.values, w.values, offsets)),
                          (dw.got(), lin.experts_backward_weights(dc.values, rows.values, offsets, 4))):
            live = ~want.isnan()
            close(got[live], want[live], (1 + want[live].abs()) * 2.0 ** -14, "f32", offsets)
            assert (got[~live] == 7777).all()


def test_sources_past_the_rows(q38m):
    """A gathered row past the last one is the last one."""
    t = torch()
    s = Sorted([4, 4], 0, 4, 2, 1)
    s.packed[1], s.packed[6] = 2 ** 20, 9
    source = (s.packed.long() // 2).clamp_max(3)
    rows, w, dc = Matrix(q38m, 1, 4, 72), Matrix(q38m, 2, 40, 72, experts=2), Matrix(q38m, 3, 8, 40)
    c, dw = output(q38m, 8, 40, "f32"), output(q38m, 40, 72, "f32", experts=2)
    q38m.call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, *s.args(), 0, c.arg, None, stream(), 0)
    q38m.call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, *s.args(), None, dw.arg, stream(), 0)
    sync()
    want = lin.experts(rows.values, w.values, s.offsets, 8, source)
    close(c.got(), want, 72 * 2.0 ** -18 + want * 0, "f32", "c")
    want = lin.experts_backward_weights(dc.values, rows.values, s.offsets, 2, source)
    close(dw.got(), want, 72 * 2.0 ** -18 + want * 0, "f32", "dw")


def layer(q38m, t, x, wg, wd, route, weights, room, on):
    """A layer's forward and backward as a training step calls them."""
    call, d = q38m.call, lambda v: ctypes.byref(q38m.describe(v))
    tokens, top_k = weights.shape
    f = {k: v.data_ptr() for k, v in (("offsets", route.offsets), ("packed", route.packed), ("inverse", route.inverse),
                                      ("weights", weights))}
    hidden = x.shape[1]
    call("q38m_moe_expert_gemm_v1", d(wg), d(x), f["offsets"], f["packed"], top_k, q38m.EPILOGUE_SWIGLU, d(room["h"]),
         d(room["pre"]), on, 0)
    call("q38m_moe_expert_gemm_v1", d(wd), d(room["h"]), f["offsets"], None, 1, q38m.EPILOGUE_NONE, d(room["rows"]),
         None, on, 0)
    call("q38m_moe_unpermute_rows_v1", room["rows"].data_ptr(), q38m.DTYPE_BF16, f["inverse"], f["weights"], tokens,
         top_k, hidden, room["y"].data_ptr(), on, 0)
    call("q38m_moe_unpermute_backward_v1", room["dy"].data_ptr(), room["rows"].data_ptr(), q38m.DTYPE_BF16,
         f["inverse"], f["weights"], tokens, top_k, hidden, room["d_rows"].data_ptr(), room["d_weights"].data_ptr(),
         on, 0)
    call("q38m_moe_expert_backward_weights_v1", d(room["d_rows"]), d(room["h"]), f["offsets"], None, 1, None,
         d(room["d_wd"]), on, 0)
    call("q38m_moe_expert_backward_rows_v1", d(wd), d(room["d_rows"]), f["offsets"], d(room["pre"]), d(room["d_pre"]),
         on, 0)
    call("q38m_moe_expert_backward_weights_v1", d(room["d_pre"]), d(x), f["offsets"], f["packed"], top_k, None,
         d(room["d_wg"]), on, 0)
    call("q38m_moe_expert_backward_rows_v1", d(wg), d(room["d_pre"]), f["offsets"], None, d(room["dx_rows"]), on, 0)
    call("q38m_moe_unpermute_rows_v1", room["dx_rows"].data_ptr(), q38m.DTYPE_BF16, f["inverse"], None, tokens, top_k,
         hidden, room["dx"].data_ptr(), on, 0)


@pytest.mark.parametrize("tokens,top_k,experts,hidden,middle,lost", [(1, 4, 8, 128, 64, 0.0), (50, 3, 12, 136, 72, 0.1),
                                                                     (400, 2, 4, 256, 128, 0.05)])
def test_a_layer_in_training(q38m, tokens, top_k, experts, hidden, middle, lost):
    """Sort, gate/up, down and rows back with all gradients, eager and captured, against autograd in 64
    bits.  Each bf16 output between the calls is off by half a step, 2^-8: the results by a few of them
    (at most eight behind one another: h, rows, y; d_rows, pre, d_pre, dx rows, dx) in the norm."""
    t = torch()
    g = t.Generator("cuda").manual_seed(tokens)

    def normal(*shape, sigma=1.0):
        return (sigma * t.randn(*shape, generator=g, device="cuda")).bfloat16()

    x, wg = normal(tokens, hidden), normal(experts, 2 * middle, hidden, sigma=hidden ** -0.5)
    wd = normal(experts, hidden, middle, sigma=middle ** -0.5)
    logits = t.randn(tokens, experts, generator=g, device="cuda")
    best = t.topk(logits, top_k, dim=1)
    ids = best.indices.int()
    ids[t.rand(ids.shape, generator=g, device="cuda") < lost] = -1
    weights = t.softmax(best.values, 1).contiguous()
    routes = tokens * top_k
    route = q38m.SortedRoutes(tokens, top_k, experts)

    def rooms():
        def zeros(*shape, dtype=t.bfloat16):
            return t.zeros(*shape, dtype=dtype, device="cuda")
        return {"h": zeros(routes, middle), "pre": zeros(routes, 2 * middle), "rows": zeros(routes, hidden),
                "y": zeros(tokens, hidden), "dy": dy, "d_rows": zeros(routes, hidden),
                "d_weights": zeros(tokens, top_k, dtype=t.float32), "d_wd": zeros(experts, hidden, middle, dtype=t.float32),
                "d_pre": zeros(routes, 2 * middle), "d_wg": zeros(experts, 2 * middle, hidden, dtype=t.float32),
                "dx_rows": zeros(routes, hidden), "dx": zeros(tokens, hidden)}

    dy = normal(tokens, hidden)
    room, again = rooms(), rooms()

    def step(into):
        route.sort(ids)
        layer(q38m, t, x, wg, wd, route, weights, into, stream())

    step(room)
    sync()
    leaves = [v.double().requires_grad_() for v in (x, wg, wd, weights)]
    x64, wg64, wd64, r64 = leaves
    y64 = t.zeros(tokens, hidden, dtype=t.float64, device="cuda")
    for e in range(experts):
        token, rank = (ids == e).nonzero(as_tuple=True)
        if len(token):
            out = lin.swiglu(x64[token] @ wg64[e].T) @ wd64[e].T
            y64 = y64.index_add(0, token, r64[token, rank].unsqueeze(1) * out)
    grads = t.autograd.grad(y64, leaves, dy.double())
    for name, want in (("y", y64.detach()), ("dx", grads[0]), ("d_wg", grads[1]), ("d_wd", grads[2]),
                       ("d_weights", grads[3])):
        off = (room[name].double() - want).norm() / want.norm()
        assert off < 8 * 2.0 ** -8, (name, float(off))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        step(again)
    for i in range(3):
        x.copy_(normal(tokens, hidden))
        step(room)
        graph.replay()
        sync()
        for name in room:
            assert t.equal(room[name], again[name]), (name, i)


def test_streams(q38m):
    """The same calls on two streams at once equal the ones alone."""
    t = torch()
    s = Sorted(ragged(32, 900, 3), 0)
    n, k = 264, 256
    rows, dc, w = Matrix(q38m, 1, 900, k), Matrix(q38m, 2, 900, n), Matrix(q38m, 3, n, k, experts=32)

    def outs():
        return output(q38m, 900, n), output(q38m, 900, k), output(q38m, n, k, experts=32)

    def run(o, on):
        q38m.call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, *s.args(), 0, o[0].arg, None, on, 0)
        q38m.call("q38m_moe_expert_backward_rows_v1", w.arg, dc.arg, s.args()[0], None, o[1].arg, on, 0)
        q38m.call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, *s.args(), None, o[2].arg, on, 0)

    alone = outs()
    run(alone, stream())
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    both = [[outs() for _ in range(5)] for _ in streams]
    sync()
    for i in range(5):
        for on, o in zip(streams, both):
            run(o[i], on.cuda_stream)
    sync()
    for o in both:
        for i in range(5):
            for a, b in zip(alone, o[i]):
                assert t.equal(a.view, b.view)


@pytest.mark.parametrize("tokens,top_k,experts", [(3, 4, 24), (90, 6, 96)])
def test_graphs_with_other_routes(q38m, tokens, top_k, experts):
    """A layer's products captured once and replayed with routes that change between the replays, experts
    with and without rows among them: every replay equals the eager calls bit for bit."""
    t = torch()
    hidden, middle, routes = 136, 72, tokens * top_k
    x, dy = Matrix(q38m, 1, tokens, hidden), Matrix(q38m, 2, routes, hidden)
    up = Matrix(q38m, 3, 2 * middle, hidden, sigma=0.1, experts=experts)
    down = Matrix(q38m, 4, hidden, middle, sigma=0.1, experts=experts)
    routing = q38m.SortedRoutes(tokens, top_k, experts)
    at, packed = q38m.ptr(routing.offsets), q38m.ptr(routing.packed)

    def buffers():
        return (output(q38m, routes, middle), output(q38m, routes, 2 * middle, "f32"), output(q38m, routes, hidden),
                output(q38m, routes, 2 * middle), output(q38m, routes, hidden),
                output(q38m, 2 * middle, hidden, "f32", experts=experts), output(q38m, hidden, middle, experts=experts))

    def run(o):
        h, pre, y, dgu, dx, dup, ddown = o
        q38m.call("q38m_moe_expert_gemm_v1", up.arg, x.arg, at, packed, top_k, 1, h.arg, pre.arg, stream(), 0)
        q38m.call("q38m_moe_expert_gemm_v1", down.arg, h.arg, at, None, 1, 0, y.arg, None, stream(), 0)
        q38m.call("q38m_moe_expert_backward_rows_v1", down.arg, dy.arg, at, pre.arg, dgu.arg, stream(), 0)
        q38m.call("q38m_moe_expert_backward_rows_v1", up.arg, dgu.arg, at, None, dx.arg, stream(), 0)
        q38m.call("q38m_moe_expert_backward_weights_v1", dgu.arg, x.arg, at, packed, top_k, dup.arg, dup.arg, stream(), 0)
        q38m.call("q38m_moe_expert_backward_weights_v1", dy.arg, h.arg, at, None, 1, None, ddown.arg, stream(), 0)

    def ids(seed):
        some = t.randperm(experts, generator=t.Generator().manual_seed(seed))[:max(top_k, experts // (seed + 1))]
        picks = t.rand(tokens, len(some), generator=t.Generator().manual_seed(seed)).argsort(1)[:, :top_k]
        return some[picks].int().cuda()

    eager, replayed = buffers(), buffers()
    routing.sort(ids(0))
    run(eager)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        run(replayed)
    for seed in range(4):
        routing.sort(ids(seed))
        for o in (eager, replayed):
            o[5].view.fill_(1.0)
        run(eager)
        graph.replay()
        sync()
        for a, b in zip(eager, replayed):
            assert t.equal(a.view, b.view), seed


@pytest.mark.parametrize("n,k,counts", [(2, 1100001, [0, 5, 0]), (700, 3, [0] * 130 + [1] + [0] * 77), (1, 1, [0] * 70)])
def test_weight_gradient_of_experts_without_rows(q38m, n, k, counts):
    """Rows of more pieces than there are threads, many experts' zeros, and no rows at all."""
    s = Sorted(counts, 0 if sum(counts) else 3)
    for spare in ((0, 0, 0), (-n % 8, -k % 8, 0)):  # on either kernel
        check_experts_weights(q38m, 11, s, n, k, None, "bf16", spare)
        check_experts_weights(q38m, 12, s, n, k, "f32", "f32", spare)
