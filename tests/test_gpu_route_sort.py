"""Tokens sorted by expert and back on the GPU against the plain 64-bit forms
(oracle/mx_oracle.py).  The sort is exact.  A row summed back over k ranks is
k fp32 fused multiply-adds, each off by at most 2^-24 of the magnitudes added
so far: k 2^-24 S with S the sum of the terms' magnitudes, then half a step of
the output type.  A weight's gradient sums `width` terms in some fixed order:
width 2^-24 S covers any order of fused multiply-adds and additions."""
import ctypes

import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, host, stream, torch

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
GUARD = 0x4a4a


def words_of(x, dtype):
    t = torch()
    f = np.asarray(x, np.float32)
    if dtype == "f32":
        return f
    return host(t.from_numpy(f).to(t.bfloat16).view(t.int16), np.uint16)


def values_of(words):
    if words.dtype == np.uint16:
        return (words.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return words.astype(np.float64)


class Rows:
    """[rows][width] values on the device, `shift` elements behind a 16-byte aligned start."""

    def __init__(self, x, dtype, shift=0):
        words = words_of(x, dtype)
        self.values = values_of(words)
        flat = np.concatenate((np.zeros(shift, words.dtype), words.reshape(-1)))
        self.buffer = device(flat)
        self.ptr = self.buffer.data_ptr() + shift * words.itemsize


class Out:
    """A guarded output buffer, filled with a pattern."""

    def __init__(self, rows, width, dtype, shift=0):
        t = torch()
        self.shape, self.dtype, self.shift = (rows, width), dtype, shift
        self.buffer = t.full((shift + rows * width + 32,), GUARD,
                             dtype=t.int16 if dtype == "bf16" else t.int32, device="cuda")
        self.ptr = self.buffer.data_ptr() + shift * self.buffer.element_size()

    def read(self):
        torch().cuda.synchronize()
        words = host(self.buffer, np.uint16 if self.dtype == "bf16" else np.uint32)
        n = self.shape[0] * self.shape[1]
        assert (words[:self.shift] == GUARD).all() and (words[self.shift + n:] == GUARD).all()
        words = words[self.shift:self.shift + n].reshape(self.shape)
        return words, values_of(words if self.dtype == "bf16" else words.view(np.float32))


def code(q38m, dtype):
    return q38m.DTYPE_BF16 if dtype == "bf16" else q38m.DTYPE_F32


def draw_ids(rng, tokens, top_k, experts, kind):
    if kind == "none":
        return np.full((tokens, top_k), -1, np.int32)
    if kind == "one":
        return np.full((tokens, top_k), experts - 1, np.int32)
    ids = rng.integers(0, experts, size=(tokens, top_k)).astype(np.int32)
    if kind == "skewed":
        ids = (rng.random(ids.shape) ** 4 * experts).astype(np.int32)
    if kind == "dropped":
        ids[rng.random(ids.shape) < 0.3] = rng.choice([-1, experts, 0x7fffffff, -0x80000000])
        ids[tokens // 2] = -5
    return ids


# the largest sort of one workgroup is 8,192 routes; 1,024 is a chunk of the larger ones
SORTS = [(1, 1, 1, "even"), (1, 10, 512, "even"), (1, 32, 3, "dropped"), (63, 1, 5, "even"),
         (64, 1, 1024, "skewed"), (65, 1, 64, "one"), (100, 10, 60, "dropped"), (512, 10, 512, "even"),
         (819, 10, 512, "none"), (1024, 8, 256, "skewed"), (8192, 1, 1024, "dropped"),
         (8193, 1, 1024, "dropped"), (1639, 5, 7, "one"), (1300, 7, 1023, "skewed"),
         (4096, 10, 512, "dropped"), (9000, 3, 1, "none"), (32768, 10, 512, "skewed"),
         (70000, 2, 1024, "even")]


def run_sort(q38m, ids, experts, guard=16):
    t = torch()
    tokens, top_k = ids.shape
    routes = tokens * top_k
    outs = [t.full((n + guard,), GUARD, dtype=t.int32, device="cuda") for n in (experts + 1, routes, routes)]
    nbytes = q38m.lib().q38m_moe_sort_scratch_bytes(tokens, top_k, experts)
    scratch = t.full((nbytes // 4 + guard,), GUARD, dtype=t.int32, device="cuda")
    ids = device(ids)
    q38m.call("q38m_moe_sort_routes_v1", ids.data_ptr(), tokens, top_k, experts,
              *(o.data_ptr() for o in outs), scratch.data_ptr() if nbytes else None, nbytes, stream(), 0)
    t.cuda.synchronize()
    assert (scratch[nbytes // 4:] == GUARD).all()
    for o, n in zip(outs, (experts + 1, routes, routes)):
        assert (o[n:] == GUARD).all()
    return [host(o, np.uint32)[:-guard] for o in outs]


@pytest.mark.parametrize("tokens,top_k,experts,kind", SORTS)
def test_sort(q38m, tokens, top_k, experts, kind):
    print(f"sort {tokens} x {top_k} of {experts} {kind}", flush=True)
    ids = draw_ids(np.random.default_rng(tokens + experts), tokens, top_k, experts, kind)
    for got, want in zip(run_sort(q38m, ids, experts), mx.sort_routes(ids, experts)):
        assert np.array_equal(got, want)


def test_sort_is_the_route_plan_order(q38m):
    """512 experts, top-10: the same order, inverse and offsets as the route plan's."""
    t = torch()
    ids = np.argsort(np.random.default_rng(9).random((200, 512)), axis=1)[:, :10].astype(np.int32)
    offsets, packed, inverse = run_sort(q38m, np.ascontiguousarray(ids), 512)
    nbytes = q38m.route_plan_bytes(200)
    buf = t.empty(nbytes + 256, dtype=t.uint8, device="cuda")
    base = (buf.data_ptr() + 255) // 256 * 256
    plan = q38m.bind_plan(base, nbytes, 200)
    ids = device(ids)
    q38m.call("q38m_moe_build_route_plan_v1", ids.data_ptr(), 200, ctypes.byref(plan), 0, stream(), 0)
    t.cuda.synchronize()
    image = host(buf, np.uint8)
    at = lambda p, n: image[p - buf.data_ptr():][:4 * n].view(np.uint32)  # noqa: E731
    assert np.array_equal(at(plan.expert_offsets, 513), offsets)
    assert np.array_equal(at(plan.packed_assignment, 2000), packed)
    assert np.array_equal(at(plan.assignment_to_packed, 2000), inverse)


ROWS = [(1, 1, 1, 1, "even", 0), (1, 10, 512, 2048, "even", 0), (5, 2, 3, 7, "dropped", 0),
        (33, 10, 60, 44, "dropped", 0), (64, 4, 8, 520, "skewed", 0), (17, 8, 16, 2048, "dropped", 1),
        (100, 3, 4, 600, "one", 3), (10, 32, 9, 4104, "even", 0), (300, 1, 64, 8, "dropped", 0),
        (8, 10, 512, 2050, "even", 0), (40, 5, 12, 129, "none", 0), (1000, 10, 512, 256, "skewed", 0),
        (3, 33, 40, 1000, "dropped", 0), (2, 7, 9, 20000, "dropped", 0)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,top_k,experts,width,kind,shift", ROWS)
def test_rows(q38m, dtype, tokens, top_k, experts, width, kind, shift):
    """There, back with and without weights, and the gradients; what a dropped route's weight, or
    a row behind the kept ones, holds does not matter (NaN here)."""
    print(f"rows {tokens} x {top_k} of {experts}, width {width} {kind} {dtype} shift {shift}", flush=True)
    rng = np.random.default_rng(tokens * 13 + width)
    ids = draw_ids(rng, tokens, top_k, experts, kind)
    offsets, _, inverse = mx.sort_routes(ids, experts)
    kept, routes = int(offsets[-1]), tokens * top_k
    at = device(inverse)
    x = Rows(rng.normal(size=(tokens, width)), dtype, shift)
    rows_in = rng.normal(size=(routes, width))
    rows_in[kept:] = np.nan
    rows = Rows(rows_in, dtype, shift)
    weights = rng.random((tokens, top_k)).astype(np.float32) * 2 - 0.5
    weights[inverse.reshape(tokens, top_k) == mx.DROPPED] = np.nan
    w = device(weights)
    dt = code(q38m, dtype)

    packed = Out(routes, width, dtype, shift)
    q38m.call("q38m_moe_permute_rows_v1", x.ptr, dt, at.data_ptr(), tokens, top_k, width, packed.ptr, stream(), 0)
    words, values = packed.read()
    assert (words[kept:] == GUARD).all()
    live = np.nonzero(inverse != mx.DROPPED)[0]
    assert np.array_equal(values[inverse[live]], x.values[live // top_k])

    for use in (weights, None):
        y = Out(tokens, width, dtype, shift)
        q38m.call("q38m_moe_unpermute_rows_v1", rows.ptr, dt, at.data_ptr(), None if use is None else w.data_ptr(),
                  tokens, top_k, width, y.ptr, stream(), 0)
        want, size = mx.unpermute(rows.values, inverse, use, tokens)
        off = np.abs(y.read()[1] - want)
        assert (off <= top_k * 2.0 ** -24 * size * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want)).all()

    for with_rows, with_weights in ((True, True), (True, False), (False, True)):
        d_rows, d_weights = Out(routes, width, dtype, shift), Out(tokens, top_k, "f32")
        q38m.call("q38m_moe_unpermute_backward_v1", x.ptr, rows.ptr if with_weights else None, dt, at.data_ptr(),
                  w.data_ptr(), tokens, top_k, width, d_rows.ptr if with_rows else None,
                  d_weights.ptr if with_weights else None, stream(), 0)
        want_rows, want_weights, size = mx.unpermute_backward(x.values, rows.values, inverse, weights)
        words, values = d_rows.read()
        if with_rows:
            assert (words[kept:] == GUARD).all()
            off = np.abs(values[:kept] - want_rows[:kept])
            assert (off <= HALF[dtype] * np.abs(want_rows[:kept]) * (1 + 2.0 ** -20)).all()
        else:
            assert (words == GUARD).all()
        words, values = d_weights.read()
        if with_weights:
            assert (np.abs(values - want_weights) <= width * 2.0 ** -24 * size).all()
        else:
            assert (words == GUARD).all()


def test_gradients_against_differences(q38m):
    """L = <g, y>: y is linear in the rows and in the weights, so a difference quotient of any
    step is the gradient, up to the rounding of y (fp32 rows, k fused multiply-adds) and of L's sum,
    which is formed in 64 bits.  Bound: 2 (k + 1) 2^-24 sum(|g| S) / step, S as for y."""
    t = torch()
    rng = np.random.default_rng(77)
    tokens, top_k, experts, width, step = 6, 3, 4, 40, 1.0
    ids = draw_ids(rng, tokens, top_k, experts, "dropped")
    offsets, _, inverse = mx.sort_routes(ids, experts)
    at, routes = device(inverse), tokens * top_k
    rows = rng.normal(size=(routes, width)).astype(np.float32)
    weights = rng.normal(size=(tokens, top_k)).astype(np.float32)
    g = rng.normal(size=(tokens, width)).astype(np.float32)

    def loss(rows, weights):
        y = Out(tokens, width, "f32")
        r, w = device(rows), device(weights)
        q38m.call("q38m_moe_unpermute_rows_v1", r.data_ptr(), q38m.DTYPE_F32, at.data_ptr(), w.data_ptr(),
                  tokens, top_k, width, y.ptr, stream(), 0)
        _, size = mx.unpermute(rows, inverse, weights, tokens)
        return float((g * y.read()[1]).sum()), float((np.abs(g) * size).sum())

    d_rows, d_weights = Out(routes, width, "f32"), Out(tokens, top_k, "f32")
    on_device = [device(a) for a in (g, rows, weights)]
    q38m.call("q38m_moe_unpermute_backward_v1", on_device[0].data_ptr(), on_device[1].data_ptr(), q38m.DTYPE_F32,
              at.data_ptr(), on_device[2].data_ptr(), tokens, top_k, width, d_rows.ptr, d_weights.ptr, stream(), 0)
    got_rows, got_weights = d_rows.read()[1], d_weights.read()[1]
    base, size = loss(rows, weights)
    for t0 in range(tokens):
        for r in range(top_k):
            moved = weights.copy()
            moved[t0, r] += step
            there, more = loss(rows, moved)
            bound = 2 * (top_k + 1) * 2.0 ** -24 * (size + more) / step
            assert abs((there - base) / step - got_weights[t0, r]) <= bound + 2.0 ** -18 * abs(got_weights[t0, r])
    for p in range(int(offsets[-1])):
        moved = rows.copy()
        moved[p, p % width] += step
        moved_by = float(moved[p, p % width]) - float(rows[p, p % width])
        there, more = loss(moved, weights)
        bound = 2 * (top_k + 1) * 2.0 ** -24 * (size + more) / step
        assert abs((there - base) / moved_by - got_rows[p, p % width]) <= bound + 2.0 ** -18 * abs(got_rows[p, p % width])


def test_bad_inverse_is_skipped(q38m):
    """Entries past the routes are no places: nothing is read or written for them."""
    tokens, top_k, width = 4, 2, 16
    inverse = np.array([0, 8, 1, 0xfffffffe, 2, 3, 0x80000000, 4], np.uint32)
    rng = np.random.default_rng(2)
    x, rows = Rows(rng.normal(size=(tokens, width)), "f32"), Rows(rng.normal(size=(8, width)), "f32")
    at, w = device(inverse), device(np.ones((tokens, top_k), np.float32))
    out, y, d = Out(8, width, "f32"), Out(tokens, width, "f32"), Out(tokens, top_k, "f32")
    dt = q38m.DTYPE_F32
    q38m.call("q38m_moe_permute_rows_v1", x.ptr, dt, at.data_ptr(), tokens, top_k, width, out.ptr, stream(), 0)
    words, values = out.read()
    assert np.array_equal(values[:5], x.values[[0, 1, 2, 2, 3]]) and (words[5:] == GUARD).all()
    q38m.call("q38m_moe_unpermute_rows_v1", rows.ptr, dt, at.data_ptr(), w.data_ptr(), tokens, top_k, width, y.ptr,
              stream(), 0)
    want, _ = mx.unpermute(rows.values, inverse, None, tokens)
    assert np.allclose(y.read()[1], want, rtol=2.0 ** -23, atol=2.0 ** -22)
    q38m.call("q38m_moe_unpermute_backward_v1", x.ptr, rows.ptr, dt, at.data_ptr(), w.data_ptr(), tokens, top_k,
              width, None, d.ptr, stream(), 0)
    assert (d.read()[1].reshape(-1)[[1, 3, 6]] == 0).all()
