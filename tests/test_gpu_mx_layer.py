"""The microscaled products and the sorted routes together, as a layer of
experts uses them: routes sorted, tokens quantised, gate/up with SwiGLU,
quantised again, down, the rows brought back with the router's weights, and
the gradients of the way there and back.  Each step is compared with the plain
64-bit form of what the step before left, so each bound is that of one step
(test_gpu_mx.py and test_gpu_route_sort.py derive them).

Then the same calls captured into a graph, on several streams, from several
threads and on the default stream, which give the same bits; and sizes past 32
bits, compared at rows spread over their length."""
import ctypes
import threading

import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, host, torch
from test_gpu_mx import close, encoded, product_bound, want_experts, widen

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu

BF16_HALF, F32_HALF = 2.0 ** -8, 2.0 ** -24


class Layer:
    """A layer's weights and the buffers of one call of `tokens` tokens."""

    def __init__(self, q38m, tokens, top_k, experts, hidden, middle, seed):
        t, rng = torch(), np.random.default_rng(seed)
        self.q38m, self.tokens, self.top_k, self.experts = q38m, tokens, top_k, experts
        self.hidden, self.middle, self.routes = hidden, middle, tokens * top_k
        self.rng = rng
        # gate/up and down weights of a size that keeps the layer's values near one
        self.gate_up = self.weights(experts, 2 * middle, hidden)
        self.down = self.weights(experts, hidden, middle)
        bf16, f32 = dict(dtype=t.bfloat16, device="cuda"), dict(dtype=t.float32, device="cuda")
        self.x, self.dy = t.zeros(tokens, hidden, **bf16), t.zeros(tokens, hidden, **bf16)
        self.ids = t.zeros(tokens, top_k, dtype=t.int32, device="cuda")
        self.w = t.zeros(tokens, top_k, **f32)
        self.sorted = q38m.SortedRoutes(tokens, top_k, experts)
        self.a, self.b = q38m.MxRows(1, tokens, hidden), q38m.MxRows(1, self.routes, middle)
        self.h = t.zeros(self.routes, middle, **bf16)  # zeros behind the kept routes too
        self.rows, self.y = t.zeros(self.routes, hidden, **bf16), t.zeros(tokens, hidden, **bf16)
        self.d_rows, self.dx = t.zeros(self.routes, hidden, **bf16), t.zeros(tokens, hidden, **bf16)
        self.d_w = t.zeros(tokens, top_k, **f32)

    def weights(self, experts, rows, columns):
        codes, scales = encoded(self.rng, experts * rows, columns, 122, 125)
        out = self.q38m.MxRows(experts, rows, columns)
        out.codes.copy_(torch().from_numpy(codes))
        out.scales.copy_(torch().from_numpy(scales))
        out.values = mx.decode(codes, scales, columns)
        return out

    def draw(self, seed, dropped=0.1):
        """New inputs; an expert may come twice in a token, some routes have none."""
        t, rng = torch(), np.random.default_rng(seed)
        ids = rng.integers(0, self.experts, size=(self.tokens, self.top_k)).astype(np.int32)
        ids[rng.random(ids.shape) < dropped] = -1
        ids[self.tokens // 2] = -1
        for to, x in ((self.x, rng.normal(size=self.x.shape)), (self.dy, rng.normal(size=self.dy.shape)),
                      (self.w, rng.random(self.w.shape)), (self.ids, ids)):
            to.copy_(t.from_numpy(x))

    def run(self, handle=None):
        q, t = self.q38m, torch()
        handle = t.cuda.current_stream().cuda_stream if handle is None else handle
        s, ref = self.sorted, ctypes.byref
        shape = (self.tokens, self.top_k, self.hidden)
        q.call("q38m_moe_sort_routes_v1", self.ids.data_ptr(), self.tokens, self.top_k, self.experts,
               s.offsets.data_ptr(), s.packed.data_ptr(), s.inverse.data_ptr(), s.scratch.data_ptr(),
               s.scratch.numel(), handle, 0)
        q.call("q38m_mx_quantize_v1", self.x.data_ptr(), q.DTYPE_BF16, self.hidden, ref(self.a.desc), None, handle, 0)
        q.call("q38m_mx_grouped_gemm_v1", ref(self.gate_up.desc), ref(self.a.desc), s.offsets.data_ptr(),
               s.packed.data_ptr(), self.top_k, self.routes, q.MX_EPILOGUE_SWIGLU, None, self.h.data_ptr(), handle, 0)
        q.call("q38m_mx_quantize_v1", self.h.data_ptr(), q.DTYPE_BF16, self.middle, ref(self.b.desc), None, handle, 0)
        q.call("q38m_mx_grouped_gemm_v1", ref(self.down.desc), ref(self.b.desc), s.offsets.data_ptr(), None, 1,
               self.routes, q.MX_EPILOGUE_NONE, None, self.rows.data_ptr(), handle, 0)
        q.call("q38m_moe_unpermute_rows_v1", self.rows.data_ptr(), q.DTYPE_BF16, s.inverse.data_ptr(),
               self.w.data_ptr(), *shape, self.y.data_ptr(), handle, 0)
        q.call("q38m_moe_unpermute_backward_v1", self.dy.data_ptr(), self.rows.data_ptr(), q.DTYPE_BF16,
               s.inverse.data_ptr(), self.w.data_ptr(), *shape, self.d_rows.data_ptr(), self.d_w.data_ptr(), handle, 0)
        q.call("q38m_moe_unpermute_rows_v1", self.d_rows.data_ptr(), q.DTYPE_BF16, s.inverse.data_ptr(), None,
               *shape, self.dx.data_ptr(), handle, 0)

    OUTPUTS = ("h", "rows", "y", "d_rows", "d_w", "dx")

    def clear(self):
        for name in self.OUTPUTS:
            getattr(self, name).zero_()

    def outputs(self):
        """Copies of what a run wrote.  What lies behind the kept routes is a run's input too."""
        s = self.sorted
        return [x.clone() for x in (s.offsets, s.packed, s.inverse, self.a.codes, self.a.scales, self.b.codes,
                                    self.b.scales, *(getattr(self, n) for n in self.OUTPUTS))]

    def eager(self):
        self.clear()
        self.run()
        return self.outputs()


def same(got, want):
    return all(torch().equal(g, w) for g, w in zip(got, want))


def values(x):
    t = torch()
    return host(x, np.float32).astype(np.float64) if x.dtype == t.float32 else widen(host(x.view(t.int16), np.uint16))


@pytest.mark.parametrize("tokens,top_k,experts,hidden,middle", [
    (1, 10, 64, 512, 128), (7, 3, 5, 200, 72), (100, 10, 32, 512, 160), (1200, 8, 6, 256, 512)])
def test_layer(q38m, tokens, top_k, experts, hidden, middle):
    print(f"layer {tokens} x {top_k} of {experts}, {hidden} x {middle}", flush=True)
    layer = Layer(q38m, tokens, top_k, experts, hidden, middle, tokens)
    layer.draw(tokens + 1)
    if tokens == 1:
        layer.ids.copy_(torch().arange(10, dtype=torch().int32).view(1, 10) * 5 % 64)
    layer.eager()
    torch().cuda.synchronize()
    offsets, packed, inverse = mx.sort_routes(host(layer.ids, np.int32), experts)
    s = layer.sorted
    for got, want in ((s.offsets, offsets), (s.packed, packed), (s.inverse, inverse)):
        assert np.array_equal(host(got, np.uint32), want)
    kept = int(offsets[-1])

    def quantised(rows, x):
        codes, scales, decoded = mx.quantize(x)
        assert np.array_equal(host(rows.codes, np.uint8), codes) and np.array_equal(host(rows.scales, np.uint8), scales)
        return decoded

    a = quantised(layer.a, values(layer.x))
    want, bound = want_experts(layer.gate_up.values, a, offsets, packed, top_k, experts, hidden, True)
    h = values(layer.h)
    close(h[:kept], want[:kept], bound[:kept], "bf16", "gate/up")
    assert (h[kept:] == 0).all()
    want, bound = want_experts(layer.down.values, quantised(layer.b, h), offsets, packed, 0, experts, middle, False)
    rows = values(layer.rows)
    close(rows[:kept], want[:kept], bound[:kept], "bf16", "down")
    w, dy = values(layer.w), values(layer.dy)
    want, size = mx.unpermute(rows, inverse, w, tokens)
    close(values(layer.y), want, top_k * F32_HALF * size, "bf16", "y")
    d_rows, d_w, size = mx.unpermute_backward(dy, rows, inverse, w)
    got = values(layer.d_rows)
    # w dy rounded in fp32, then to bf16
    close(got[:kept], d_rows[:kept], F32_HALF * np.abs(d_rows[:kept]), "bf16", "d_rows")
    assert (got[kept:] == 0).all()
    close(values(layer.d_w), d_w, hidden * F32_HALF * size, "f32", "d_w")
    want, size = mx.unpermute(got, inverse, None, tokens)
    close(values(layer.dx), want, top_k * F32_HALF * size, "bf16", "dx")


SMALL, LARGE = (40, 10, 24, 256, 96), (1500, 8, 12, 512, 256)  # 400 and 12,000 routes: both sorts


@pytest.mark.parametrize("shape", [SMALL, LARGE], ids=["small", "large"])
def test_graph(q38m, shape):
    """Captured once, replayed on other inputs, with eager runs of the same buffers between."""
    t = torch()
    layer = Layer(q38m, *shape, 5)
    layer.draw(0)
    layer.eager()
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=side):
        layer.run()
    for seed in range(1, 6):
        layer.draw(seed)
        want = layer.eager()
        layer.clear()
        graph.replay()
        got = layer.outputs()
        t.cuda.synchronize()
        assert same(got, want), seed


def test_two_graphs_share_the_buffers(q38m):
    """Two captured runs of the same buffers, one behind the other on a stream."""
    t = torch()
    layer = Layer(q38m, *LARGE, 6)
    layer.draw(0)
    layer.eager()
    graphs = [t.cuda.CUDAGraph(), t.cuda.CUDAGraph()]
    for graph in graphs:
        with t.cuda.graph(graph):
            layer.run()
    for seed in range(1, 4):
        layer.draw(seed)
        want = layer.eager()
        layer.clear()
        for graph in graphs:
            graph.replay()
        got = layer.outputs()
        assert same(got, want), seed


def test_streams(q38m):
    """Four layers of their own on a stream each, their calls in turn; one on the default stream."""
    t = torch()
    layers = [Layer(q38m, *(SMALL, LARGE)[i % 2], 20 + i) for i in range(4)]
    want = []
    for i, layer in enumerate(layers):
        layer.draw(30 + i)
        want.append(layer.eager())
    t.cuda.synchronize()
    streams = [t.cuda.Stream() for _ in layers[1:]]
    for _ in range(3):
        for layer in layers:
            layer.clear()
        t.cuda.synchronize()
        for _ in range(5):
            layers[0].run(0)  # the default stream's handle
            for layer, s in zip(layers[1:], streams):
                layer.run(s.cuda_stream)
        t.cuda.synchronize()
        assert all(same(layer.outputs(), w) for layer, w in zip(layers, want))


def test_threads(q38m):
    """Calls from two threads at once, each with its stream and buffers."""
    t = torch()
    layers = [Layer(q38m, *SMALL, 40), Layer(q38m, *LARGE, 41)]
    want = []
    for i, layer in enumerate(layers):
        layer.draw(50 + i)
        want.append(layer.eager())
        layer.clear()
    streams = [t.cuda.Stream() for _ in layers]
    t.cuda.synchronize()
    failed = []

    def work(layer, handle):
        try:
            for _ in range(20):
                layer.run(handle)
        except Exception as error:  # noqa: BLE001  (reported by the test's own thread)
            failed.append(error)

    threads = [threading.Thread(target=work, args=(l, s.cuda_stream)) for l, s in zip(layers, streams)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    t.cuda.synchronize()
    assert not failed
    assert all(same(layer.outputs(), w) for layer, w in zip(layers, want))


def test_python_rows(q38m):
    """The Python conveniences: a strided view, a single row of any stride, raw words, a stream."""
    t = torch()
    x = t.randn(12, 300, device="cuda").to(t.bfloat16)
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    for view, stream in ((x, None), (x[:, 7:230], None), (x[::3], side), (x[4:5].as_strided((1, 300), (3, 1)), None),
                         (x.view(t.int16), side), (x.float(), None)):
        rounded = t.empty_like(view, memory_format=t.contiguous_format)
        out = q38m.mx_quantize(view, rounded=rounded, stream=stream)
        t.cuda.synchronize()
        v = view.contiguous()
        codes, scales, decoded = mx.quantize(values(v.view(t.bfloat16) if v.dtype == t.int16 else v))
        assert np.array_equal(host(out.codes, np.uint8), codes) and np.array_equal(host(out.scales, np.uint8), scales)
        assert np.array_equal(values(rounded.view(t.bfloat16) if v.dtype == t.int16 else rounded), decoded)
    ids = device(np.array([[3, 1], [3, 3], [-1, 0]], np.int32))
    routes = q38m.SortedRoutes(3, 2, 4).sort(ids)
    t.cuda.synchronize()
    for got, want in zip((routes.offsets, routes.packed, routes.inverse), mx.sort_routes(host(ids, np.int32), 4)):
        assert np.array_equal(host(got, np.uint32), want)


# ---- past 32 bits -------------------------------------------------------------

def spread(rows, count=24):
    return np.unique(np.concatenate((np.linspace(0, rows - 1, count).astype(np.int64), [rows - 1, rows // 2 + 1])))


def random_rows(q38m, experts, rows, columns, low=122, high=126):
    """Random codes and scales made on the device; columns a multiple of 128."""
    t = torch()
    out = q38m.MxRows(experts, rows, columns)
    out.codes.random_(0, 256)
    out.scales.random_(low, high)
    return out


def decode_rows(rows, at, columns):
    at = torch().as_tensor(at, device="cuda")
    return mx.decode(host(rows.codes[at], np.uint8), host(rows.scales[at], np.uint8), columns)


def test_large_quantize(q38m):
    """4.6 billion elements, 2.2 million rows."""
    t = torch()
    rows, columns, stride = (1 << 21) + 99, 2180, 2200
    x = t.empty(rows, stride, dtype=t.bfloat16, device="cuda")
    x.normal_()
    rounded = t.empty(rows, columns, dtype=t.bfloat16, device="cuda")
    out = q38m.mx_quantize(x[:, :columns], rounded=rounded)
    at = t.as_tensor(spread(rows), device="cuda")
    codes, scales, decoded = mx.quantize(values(x[at][:, :columns].contiguous()))
    assert np.array_equal(host(out.codes[at], np.uint8), codes) and np.array_equal(host(out.scales[at], np.uint8), scales)
    assert np.array_equal(values(rounded[at]), decoded)


@pytest.mark.parametrize("m,n,k", [(70000, 65600, 128), ((1 << 22) + 70, 40, 2048), (40, (1 << 22) + 70, 2048)])
def test_large_product(q38m, m, n, k):
    """C of 4.6 billion values; 4.3 GB of codes in A and in B."""
    t = torch()
    a, b = random_rows(q38m, 1, m, k), random_rows(q38m, 1, n, k)
    c = t.empty(m, n, dtype=t.bfloat16, device="cuda")
    q38m.call("q38m_mx_gemm_v1", ctypes.byref(a.desc), ctypes.byref(b.desc), None, c.data_ptr(), n,
              t.cuda.current_stream().cuda_stream, 0)
    rows, columns = spread(m), spread(n, 300)
    want, size = mx.product(decode_rows(a, rows, k), decode_rows(b, columns, k))
    got = values(c[t.as_tensor(rows, device="cuda")][:, t.as_tensor(columns, device="cuda")].contiguous())
    close(got, want, product_bound(k, size), "bf16", (m, n, k))


def test_large_experts(q38m):
    """4.3 GB of the experts' codes: 1,024 experts, the last ones in use."""
    t = torch()
    experts, n, k, routes = 1024, 2050, 4096, 3000
    w, rows = random_rows(q38m, experts, n, k), random_rows(q38m, 1, routes, k)
    ids = np.random.default_rng(1).integers(0, experts, size=(routes, 1)).astype(np.int32)
    ids[:9] = experts - 1
    offsets, packed, _ = mx.sort_routes(ids, experts)
    c = t.empty(routes, n, dtype=t.float32, device="cuda")
    at, order = device(offsets), device(packed)
    q38m.call("q38m_mx_grouped_gemm_v1", ctypes.byref(w.desc), ctypes.byref(rows.desc), at.data_ptr(),
              order.data_ptr(), 1, routes, q38m.MX_EPILOGUE_NONE, c.data_ptr(), None,
              t.cuda.current_stream().cuda_stream, 0)
    places, columns = spread(routes), spread(n, 40)
    got = values(c[t.as_tensor(places, device="cuda")][:, t.as_tensor(columns, device="cuda")].contiguous())
    a = decode_rows(rows, packed[places].astype(np.int64), k)
    for i, p in enumerate(places):
        expert = int(ids[packed[p], 0])
        want, size = mx.product(a[i:i + 1], decode_rows(w, expert * n + columns, k))
        close(got[i:i + 1], want, product_bound(k, size), "f32", (p, expert))


@pytest.mark.parametrize("width", [8192, 1201])
def test_large_rows(q38m, width):
    """560,000 routes of bf16 rows, 9.2 GB of them at 8,192 values and an odd start for every
    second row at 1,201: there, back and the gradients."""
    t = torch()
    tokens, top_k, experts = 70000, 8, 300
    routes = tokens * top_k
    ids = t.randint(-20, experts, (tokens, top_k), dtype=t.int32, device="cuda")
    s = q38m.SortedRoutes(tokens, top_k, experts).sort(ids)
    x = t.empty(tokens, width, dtype=t.bfloat16, device="cuda").normal_()
    rows = t.zeros(routes, width, dtype=t.bfloat16, device="cuda")
    w = t.rand(tokens, top_k, device="cuda")
    y, d_rows, d_w = t.empty_like(x), t.zeros_like(rows), t.empty_like(w)
    shape, handle = (tokens, top_k, width), t.cuda.current_stream().cuda_stream
    dt, inverse = q38m.DTYPE_BF16, s.inverse.data_ptr()
    q38m.call("q38m_moe_permute_rows_v1", x.data_ptr(), dt, inverse, *shape, rows.data_ptr(), handle, 0)
    q38m.call("q38m_moe_unpermute_rows_v1", rows.data_ptr(), dt, inverse, w.data_ptr(), *shape, y.data_ptr(), handle, 0)
    q38m.call("q38m_moe_unpermute_backward_v1", x.data_ptr(), rows.data_ptr(), dt, inverse, w.data_ptr(), *shape,
              d_rows.data_ptr(), d_w.data_ptr(), handle, 0)
    at = s.inverse.view(tokens, top_k).long()
    kept = int(s.offsets[-1])
    assert kept < routes and not rows[kept:].any() and not d_rows[kept:].any()
    for r in range(top_k):
        has = at[:, r] >= 0
        for part in has.nonzero()[:, 0].split(16384):
            assert t.equal(rows[at[part, r]], x[part])
    some = t.as_tensor(spread(tokens), device="cuda")
    x64, w64, held = values(x[some]), values(w[some]), host(at[some] >= 0, np.bool_)
    share = w64 * held
    want, size = share.sum(1, keepdims=True) * x64, share.sum(1, keepdims=True) * np.abs(x64)
    close(values(y[some]), want, top_k * F32_HALF * size, "bf16", "y")
    size = (x64 * x64).sum(1, keepdims=True) * held
    close(values(d_w[some]), size, width * F32_HALF * size, "f32", "d_w")
    for r in range(top_k):
        has = np.nonzero(held[:, r])[0]
        want = w64[has, r, None] * x64[has]
        got = values(d_rows[at[some[t.as_tensor(has, device="cuda")], r]])
        close(got, want, F32_HALF * np.abs(want), "bf16", "d_rows")


def test_most_routes(q38m):
    """2^24 - 1 routes, the most there may be, and a row of one value for each."""
    t = torch()
    tokens, experts = (1 << 24) - 1, 1024
    ids = np.random.default_rng(8).integers(-3, experts + 3, size=(tokens, 1)).astype(np.int32)
    s = q38m.SortedRoutes(tokens, 1, experts).sort(device(ids))
    x = t.randn(tokens, 1, device="cuda")
    rows, y, dw = t.zeros_like(x), t.empty_like(x), t.empty_like(x)
    handle, inverse = t.cuda.current_stream().cuda_stream, s.inverse.data_ptr()
    q38m.call("q38m_moe_permute_rows_v1", x.data_ptr(), q38m.DTYPE_F32, inverse, tokens, 1, 1, rows.data_ptr(), handle, 0)
    q38m.call("q38m_moe_unpermute_rows_v1", rows.data_ptr(), q38m.DTYPE_F32, inverse, None, tokens, 1, 1, y.data_ptr(),
              handle, 0)
    q38m.call("q38m_moe_unpermute_backward_v1", x.data_ptr(), rows.data_ptr(), q38m.DTYPE_F32, inverse, x.data_ptr(),
              tokens, 1, 1, None, dw.data_ptr(), handle, 0)
    t.cuda.synchronize()
    offsets, packed, want = mx.sort_routes(ids, experts)
    for got, right in ((s.offsets, offsets), (s.packed, packed), (s.inverse, want)):
        assert np.array_equal(host(got, np.uint32), right)
    held = t.as_tensor((ids >= 0) & (ids < experts), device="cuda")
    assert t.equal(y, t.where(held, x, 0.0)) and t.equal(dw, t.where(held, x * x, 0.0))
