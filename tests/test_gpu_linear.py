"""Dense bf16 products with bias, activation and residual, and their gradients,
against plain forms in 64 bits (oracle/linear_oracle.py).  Operands lie among NaN,
outputs among guards; the bounds are derived in linear_cases.py."""
import ctypes

import pytest

from helpers import stream, torch
from linear_cases import (ACT_ERROR, F32_ROUND, Matrix, check_backward_input, check_backward_weight, check_linear,
                          close, lin, output, product_bound, run_linear, scratch_for, sync)

pytestmark = pytest.mark.gpu

# rows, outputs, inputs: one of everything, tiles just full, just begun, odd, long and short K
SIZES = [(1, 1, 1), (1, 8, 8), (1, 2048, 512), (2, 17, 33), (3, 1, 100), (15, 16, 64), (16, 64, 72), (17, 65, 63),
         (31, 130, 127), (64, 64, 64), (65, 100, 8), (100, 257, 200), (128, 128, 128), (129, 127, 520), (255, 256, 64),
         (257, 264, 136), (512, 40, 1000), (300, 520, 2048), (513, 512, 192), (61, 1024, 2056), (1, 4096, 2048),
         (700, 7, 9), (1030, 1032, 256)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward(q38m, m, n, k):
    check_linear(q38m, m + n + k, m, n, k)
    check_linear(q38m, m + n + k, m, n, k, "silu", "bf16", "f32", "f32", "bf16")


@pytest.mark.parametrize("m,n,k", SIZES)
def test_input_gradient(q38m, m, n, k):
    check_backward_input(q38m, m + n + k, m, n, k)
    check_backward_input(q38m, m + n + k, m, n, k, "gelu_tanh", "bf16", "f32")


@pytest.mark.parametrize("m,n,k", SIZES)
def test_weight_gradient(q38m, m, n, k):
    check_backward_weight(q38m, m + n + k, m, n, k)
    check_backward_weight(q38m, m + n + k, m, n, k, "f32", "f32", "bf16")


# rows that start at 16 bytes without being so long; rows that start anywhere
STRIDES = [((8, 0, 0), (0, 0, 0)), ((0, 16, 8), (8, 8, 0)), ((24, 8, 3), (0, 0, 1)), ((1, 0, 0), (0, 0, 0)),
           ((0, 3, 0), (0, 0, 0)), ((0, 0, 5), (1, 0, 0)), ((13, 5, 1), (3, 7, 1))]


@pytest.mark.parametrize("spare,shift", STRIDES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 136), (50, 72, 264), (130, 136, 200)])
def test_strides(q38m, m, n, k, spare, shift):
    check_linear(q38m, 5, m, n, k, "gelu", "f32", "bf16", "bf16", "f32", spare=spare, shift=shift)
    check_backward_input(q38m, 6, m, n, k, "silu", "f32", "bf16", "f32", spare=spare, shift=shift)
    check_backward_weight(q38m, 7, m, n, k, "bf16", "bf16", spare=spare, shift=shift)


@pytest.mark.parametrize("act", lin.ACTIVATIONS)
@pytest.mark.parametrize("m,n,k", [(5, 80, 64), (200, 136, 128)])
def test_activations(q38m, act, m, n, k):
    check_linear(q38m, 8, m, n, k, act, "f32", None, "f32", "f32", sigma=4.0)
    check_linear(q38m, 9, m, n, k, act, None, "bf16", "bf16", sigma=4.0)
    check_backward_input(q38m, 10, m, n, k, act, None, "f32", "bf16")
    check_backward_input(q38m, 11, m, n, k, act, "bf16", "bf16", "f32")


@pytest.mark.parametrize("m", [33, 256, 257, 511, 5000, 70001])
@pytest.mark.parametrize("n", [1, 8, 77, 640])
def test_bias_gradient_alone(q38m, m, n):
    check_backward_weight(q38m, m + n, m, n, 1, db="f32", dw=False, spare=(n % 3, 0, 0))


def one_by_one(q38m, act, z, slope):
    """act(z) through a product with the one-by-one identity, or act'(z) of a gradient of ones."""
    t = torch()
    rows = z.numel()
    one = Matrix(q38m, 0, 1, 1, fill=1.0)
    if slope:
        dz = Matrix(q38m, 0, rows, 1, fill=1.0)
        pre = Matrix(q38m, 0, rows, 1, "f32", fill=z.float().view(-1, 1))
        out = output(q38m, rows, 1, "f32")
        q38m.call("q38m_linear_backward_activation_v1", dz.arg, pre.arg, q38m.ACTIVATIONS[act], out.arg, stream(), 0)
    else:
        x = Matrix(q38m, 0, rows, 1, fill=z.view(-1, 1))
        out = output(q38m, rows, 1, "f32")
        run_linear(q38m, x, one, None, act, None, out, None)
    sync()
    return out.view.double().view(-1), t


@pytest.mark.parametrize("act", lin.ACTIVATIONS)
@pytest.mark.parametrize("slope", [False, True])
def test_every_bf16(q38m, act, slope):
    """Every bf16 pattern: the header's bound for finite ones, NaN for NaN, the limits far out."""
    t = torch()
    z = t.arange(65536, device="cuda").to(t.int32).to(t.int16).view(t.bfloat16)
    got, _ = one_by_one(q38m, act, z, slope)
    exact = z.double()
    finite = exact.isfinite()
    want = (lin.slope if slope else lin.activation)(act, t.where(finite, exact, 0.0).clamp(-1e4, 1e4))
    if not slope and act != "sigmoid":  # beyond: 0 or z
        want = t.where(exact > 1e4, exact, want)
        if act == "none":
            want = exact
    off = (got - want).abs()
    limit = ACT_ERROR * exact.abs().clamp_min(1) + F32_ROUND * want.abs() + 2.0 ** -126
    bad = finite & (off > limit)
    assert not bad.any(), (exact[bad][:5], got[bad][:5], want[bad][:5])
    if not (slope and act in ("none", "relu")):
        assert got[exact.isnan()].isnan().all()
    if act != "none":
        assert (off[finite & (exact < -200)] <= 2.0 ** -126).all()


def test_masked_places_do_not_count(q38m):
    """Infinities and NaN in rows of x reach their own rows of y and no other; in weight rows their
    own columns; zeros times infinity are NaN as in the formula."""
    t = torch()
    x, w = Matrix(q38m, 1, 70, 136), Matrix(q38m, 2, 90, 136)
    x.view[3, 5], x.view[66, 135], w.view[7, 0], w.view[89, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    y = output(q38m, 70, 90, "f32")
    run_linear(q38m, x, w, None, "none", None, y, None)
    want = x.view.double() @ w.view.double().T
    got = y.got()
    assert t.equal(got.isnan(), want.isnan()) and t.equal(got.isinf(), want.isinf())
    rows = [i for i in range(70) if i not in (3, 66)]
    columns = [j for j in range(90) if j not in (7, 89)]
    assert got[rows][:, columns].isfinite().all()


@pytest.mark.parametrize("out,residual", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,k", [(1, 100, 256), (61, 200, 72), (300, 264, 128)])
def test_residual_in_place(q38m, m, n, k, out, residual):
    """y, dx and d_weight may be the residual that they are added to."""
    def outputs(rows, columns):
        return Matrix(q38m, 4, rows, columns, out, spare=8)

    x, w = Matrix(q38m, 1, m, k), Matrix(q38m, 2, n, k, sigma=k ** -0.5)
    dz = Matrix(q38m, 3, m, n, sigma=n ** -0.5)
    scratch, at, nbytes = scratch_for(q38m, m, n, k)
    for name, rows, columns, args in (
            ("q38m_linear_v1", m, n, lambda r, c: (x.arg, w.arg, None, 0, r, c, None)),
            ("q38m_linear_backward_input_v1", m, k, lambda r, c: (dz.arg, w.arg, None, 0, r, c)),
            ("q38m_linear_backward_weight_v1", n, k, lambda r, c: (dz.arg, x.arg, r, c, None))):
        apart, place = outputs(rows, columns), output(q38m, rows, columns, out, 8)
        q38m.call(name, *args(apart.arg, place.arg), at, nbytes, stream(), 0)
        q38m.call(name, *args(apart.arg, apart.arg), at, nbytes, stream(), 0)
        sync()
        assert torch().equal(apart.view, place.view), name


def test_a_layer_against_differences(q38m):
    """dx, dW and db against central differences of sum(dy * y) in 64 bits."""
    t = torch()
    m, n, k, act = 6, 10, 24, "silu"
    x, w = Matrix(q38m, 1, m, k), Matrix(q38m, 2, n, k, sigma=0.3)
    b, dy = Matrix(q38m, 3, 1, n, "f32"), Matrix(q38m, 4, m, n)
    y, pre, dz = output(q38m, m, n, "f32"), output(q38m, m, n, "f32"), output(q38m, m, n)
    run_linear(q38m, x, w, b, act, None, y, pre)
    q38m.call("q38m_linear_backward_activation_v1", dy.arg, pre.arg, q38m.ACTIVATIONS[act], dz.arg, stream(), 0)
    dx, dw, db = output(q38m, m, k, "f32"), output(q38m, n, k, "f32"), output(q38m, 1, n, "f32")
    scratch, at, nbytes = scratch_for(q38m, m, n, k)
    q38m.call("q38m_linear_backward_input_v1", dz.arg, w.arg, None, 0, None, dx.arg, at, nbytes, stream(), 0)
    q38m.call("q38m_linear_backward_weight_v1", dz.arg, x.arg, None, dw.arg, db.arg, at, nbytes, stream(), 0)
    sync()

    def value(x_, w_, b_):
        return (dy.values * lin.linear(x_, w_, b_, act)[0]).sum()

    h = 2.0 ** -12
    given = {"x": x.values, "w": w.values, "b": b.values}
    for name, got in (("x", dx.got()), ("w", dw.got()), ("b", db.got())):
        flat = t.empty(got.numel(), dtype=t.float64, device="cuda")
        for i in range(got.numel()):
            def moved(step):
                v = {key: p.clone() for key, p in given.items()}
                v[name].view(-1)[i] += step
                return value(v["x"], v["w"], v["b"])
            flat[i] = (moved(h) - moved(-h)) / (2 * h)
        # dz is rounded to bf16: half a step of each of its terms; the differences are off by h^2 times a
        # third derivative of at most a few units per term
        size = {"x": dy.values.abs() @ w.values.abs(), "w": dy.values.abs().T @ x.values.abs(),
                "b": dy.values.abs().sum(0, keepdim=True)}[name]
        third = (1 + x.values.abs().max() ** 3) * h * h * size.max() * 4
        close(got, flat.view_as(got), size * (1.13 * 2.0 ** -8 + 2.0 ** -18) + third, "f32", name)


def test_streams_and_graphs(q38m):
    """The three products and the bias gradient on a stream of their own, and captured with inputs
    that change between replays; every replay equals the eager call bit for bit."""
    t = torch()
    for m, n, k in ((1, 2048, 512), (61, 520, 2048), (300, 512, 256), (1000, 136, 64)):
        x, w, dz = Matrix(q38m, 1, m, k), Matrix(q38m, 2, n, k, sigma=k ** -0.5), Matrix(q38m, 3, m, n)
        b, r = Matrix(q38m, 4, 1, n, "f32"), Matrix(q38m, 5, m, n)

        def buffers():
            return (output(q38m, m, n), output(q38m, m, n, "f32"), output(q38m, m, k), output(q38m, n, k, "f32"),
                    output(q38m, 1, n, "f32"), scratch_for(q38m, m, n, k))

        def run(o, on):
            y, pre, dx, dw, db, (_, at, nbytes) = o
            q38m.call("q38m_linear_v1", x.arg, w.arg, b.arg, 2, r.arg, y.arg, pre.arg, at, nbytes, on, 0)
            q38m.call("q38m_linear_backward_input_v1", dz.arg, w.arg, None, 0, None, dx.arg, at, nbytes, on, 0)
            q38m.call("q38m_linear_backward_weight_v1", dz.arg, x.arg, None, dw.arg, db.arg, at, nbytes, on, 0)

        eager, other, replayed = buffers(), buffers(), buffers()
        side = t.cuda.Stream()
        side.wait_stream(t.cuda.current_stream())
        run(other, side.cuda_stream)
        run(eager, stream())
        sync()
        for a, c in zip(eager[:5], other[:5]):
            assert t.equal(a.view, c.view)
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            run(replayed, stream())
        for i in range(4):
            x.view.copy_(t.randn(m, k, generator=t.Generator("cuda").manual_seed(i), device="cuda").bfloat16())
            run(eager, stream())
            graph.replay()
            sync()
            for a, c in zip(eager[:5], replayed[:5]):
                assert t.equal(a.view, c.view), (m, n, k, i)


def test_two_scratches_at_once(q38m):
    """Calls on two streams with a scratch each."""
    t = torch()
    m, n, k = 61, 256, 4096
    x, w = Matrix(q38m, 1, m, k), Matrix(q38m, 2, n, k)
    alone = output(q38m, m, n, "f32")
    run_linear(q38m, x, w, None, "none", None, alone, None)
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    outs = [[output(q38m, m, n, "f32") for _ in range(20)] for _ in streams]
    rooms = [scratch_for(q38m, m, n, k) for _ in streams]
    sync()
    for i in range(20):
        for s, o, (_, at, nbytes) in zip(streams, outs, rooms):
            q38m.call("q38m_linear_v1", x.arg, w.arg, None, 0, None, o[i].arg, None, at, nbytes, s.cuda_stream, 0)
    sync()
    for o in outs:
        for y in o:
            assert t.equal(y.view, alone.view)


def test_long_rows_past_32_bits(q38m):
    """A matrix of more than 4 GB: offsets of its last rows are past 32 bits."""
    t = torch()
    rows, k, n = (1 << 31) // 1024 + 70, 1024, 24
    x = t.zeros(rows, k, dtype=t.bfloat16, device="cuda")
    g = t.Generator("cuda").manual_seed(3)
    x[-100:] = t.randn(100, k, generator=g, device="cuda").bfloat16()
    w = t.randn(n, k, generator=g, device="cuda").bfloat16()
    y = t.empty(rows, n, dtype=t.float32, device="cuda")
    _, at, nbytes = scratch_for(q38m, rows, n, k)
    d = [q38m.describe(v) for v in (x, w, y)]
    q38m.call("q38m_linear_v1", *(ctypes.byref(v) for v in d[:2]), None, 0, None, ctypes.byref(d[2]), None, at, nbytes,
              stream(), 0)
    sync()
    a, b = x[-100:].double(), w.double()
    close(y[-100:].double(), a @ b.T, (a.abs() @ b.abs().T) * (k / 8 + 32) * 2.0 ** -23, "f32", "y")
    assert not y[:-100].any()
    # the gradient of x, as long
    dz = t.zeros(rows, n, dtype=t.bfloat16, device="cuda")
    dz[-100:] = t.randn(100, n, generator=g, device="cuda").bfloat16()
    e = q38m.describe(dz)
    q38m.call("q38m_linear_backward_input_v1", ctypes.byref(e), ctypes.byref(d[1]), None, 0, None, ctypes.byref(d[0]),
              at, nbytes, stream(), 0)
    sync()
    a = dz[-100:].double()
    close(x[-100:].double(), a @ b, (a.abs() @ b.abs()) * (n / 8 + 32) * 2.0 ** -23, "bf16", "dx")
    assert not x[:-100].any()
    dw = t.empty(n, k, dtype=t.float32, device="cuda")
    f = q38m.describe(dw)
    q38m.call("q38m_linear_backward_weight_v1", ctypes.byref(e), ctypes.byref(d[0]), None, ctypes.byref(f), None, at,
              nbytes, stream(), 0)
    sync()
    b = x[-100:].double()
    # zeros add nothing and no error
    close(dw.double(), a.T @ b, (a.abs().T @ b.abs()) * 300 * 2.0 ** -23, "f32", "dw")


@pytest.mark.parametrize("m,n,k", [(1, 333, 2001), (17, 401, 333), (700, 513, 65), (131, 1001, 1003)])
def test_odd_rows_copied_and_not(q38m, m, n, k):
    """Contiguous odd rows: with the scratch that a layer is told to bring, and with none where that
    is taken too; strides that the scratch was not sized for, with room and without."""
    t = torch()
    big = t.empty(1 << 26, dtype=t.uint8, device="cuda")
    for spare in (0, 3):
        x, w = Matrix(q38m, 1, m, k, spare=spare, shift=spare), Matrix(q38m, 2, n, k, sigma=k ** -0.5, spare=spare)
        dz = Matrix(q38m, 3, m, n, spare=spare)
        _, at, nbytes = scratch_for(q38m, m, n, k)
        for place, room in ((at, nbytes), (None, 0), (big.data_ptr(), big.numel())):
            y, dx = output(q38m, m, n, "f32", 1), output(q38m, m, k, "f32", 1)
            dw = output(q38m, n, k, "f32", 1)
            q38m.call("q38m_linear_v1", x.arg, w.arg, None, 0, None, y.arg, None, place, room, stream(), 0)
            q38m.call("q38m_linear_backward_input_v1", dz.arg, w.arg, None, 0, None, dx.arg, place, room, stream(), 0)
            q38m.call("q38m_linear_backward_weight_v1", dz.arg, x.arg, None, dw.arg, None, place, room, stream(), 0)
            sync()
            for got, a, b in ((y, x.values, w.values.T), (dx, dz.values, w.values), (dw, dz.values.T, x.values)):
                close(got.got(), a @ b, product_bound(a.shape[1], a.abs() @ b.abs()), "f32", (spare, room))


@pytest.mark.parametrize("m,n,k", [(300, 256, 8192), (5, 264, 2048), (1030, 520, 640)])
def test_residual_larger_than_the_sums(q38m, m, n, k):
    """A residual of a thousand times the sums' size is a term of them at most: the bound of a sum of
    one term more, whichever it begins with."""
    t = torch()
    for rows, outputs, inputs, name in ((m, n, k, "forward"), (m, k, n, "input"), (k, m, n, "weight")):
        if name == "forward":
            a, b = Matrix(q38m, 1, rows, inputs), Matrix(q38m, 2, outputs, inputs, sigma=inputs ** -0.5)
            shape, product = (rows, outputs), lambda a, b: a @ b.T
        elif name == "input":
            a, b = Matrix(q38m, 1, rows, outputs), Matrix(q38m, 2, outputs, inputs, sigma=outputs ** -0.5)
            shape, product = (rows, inputs), lambda a, b: a @ b
        else:
            a, b = Matrix(q38m, 1, rows, outputs), Matrix(q38m, 2, rows, inputs, sigma=rows ** -0.5)
            shape, product = (outputs, inputs), lambda a, b: a.T @ b
        depth = {"forward": inputs, "input": outputs, "weight": rows}[name]
        r, y = Matrix(q38m, 3, *shape, "f32", sigma=1000.0), output(q38m, *shape, "f32")
        _, at, nbytes = scratch_for(q38m, rows, outputs, inputs)
        if name == "forward":
            q38m.call("q38m_linear_v1", a.arg, b.arg, None, 0, r.arg, y.arg, None, at, nbytes, stream(), 0)
        elif name == "input":
            q38m.call("q38m_linear_backward_input_v1", a.arg, b.arg, None, 0, r.arg, y.arg, at, nbytes, stream(), 0)
        else:
            q38m.call("q38m_linear_backward_weight_v1", a.arg, b.arg, r.arg, y.arg, None, at, nbytes, stream(), 0)
        sync()
        size = product(a.values.abs(), b.values.abs()) + r.values.abs()
        close(y.got(), product(a.values, b.values) + r.values, product_bound(depth + 1, size), "f32", (name, m, n, k))
