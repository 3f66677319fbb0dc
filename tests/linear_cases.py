"""Plumbing of the tests of the bf16 products with epilogues and gradients:
operands in larger buffers whose other values are NaN, outputs with guards around
them, and the bounds.

A product's terms are exact in fp32 (16 significant bits).  A matrix instruction
is taken to add at least eight of them at a time to an fp32 sum, each time off by
at most 2^-23 of the magnitudes added (twice a rounding: bits below the largest
term may be cut off), and at most 32 partial sums to be joined the same way: with
S the sum of all terms' magnitudes, (ceil(K / 8) + 32) 2^-23 S.  An activation is
within 8 2^-24 max(1, |z|) of the formula at its argument, as its header says, and
has a slope of at most 1.13, its derivative one of at most 0.8 (gelu's: 2 phi(0));
each fp32 operation behind adds a rounding, and the output half a step.
"""
import ctypes

from conftest import load_oracle
from helpers import stream, torch

load_oracle()
import linear_oracle as lin  # noqa: E402

F32_ROUND = 2.0 ** -24
ACT_ERROR = 8 * F32_ROUND


def generator(seed):
    g = torch().Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Matrix:
    """rows x columns (experts times) of a type, `spare` elements from row to row and `shift`
    elements in front; everything else is NaN.  values: float64 of what it holds."""

    def __init__(self, q38m, seed, rows, columns, dtype="bf16", sigma=1.0, spare=0, shift=0, experts=1, fill=None):
        t = torch()
        kind = t.bfloat16 if dtype == "bf16" else t.float32
        self.stride, self.rows, self.columns, self.experts, self.dtype = columns + spare, rows, columns, experts, dtype
        all_rows = experts * rows
        self.buffer = t.full((shift + all_rows * self.stride + 64,), float("nan"), dtype=kind, device="cuda")
        self.shift = shift
        if fill is not None:
            self.view[:] = fill
        else:
            self.view[:] = (sigma * t.randn(all_rows, columns, generator=generator(seed), device="cuda")).to(kind)
        self.values = self.view.double().view(experts, rows, columns)
        if experts == 1:
            self.values = self.values[0]
        self.q38m = q38m
        self.desc = q38m.Tensor(self.buffer.data_ptr() + shift * self.buffer.element_size(), self.stride,
                                q38m.DTYPE_BF16 if dtype == "bf16" else q38m.DTYPE_F32, experts, rows, columns)

    @property
    def view(self):
        n = self.experts * self.rows
        return self.buffer[self.shift:self.shift + n * self.stride].view(n, self.stride)[:, :self.columns]

    @property
    def arg(self):
        return ctypes.byref(self.desc)

    def got(self):
        """float64 values; checks that nothing around them was written."""
        t = torch()
        n = self.experts * self.rows
        rest = t.ones(self.buffer.shape, dtype=t.bool, device="cuda")
        rest[self.shift:self.shift + n * self.stride].view(n, self.stride)[:, :self.columns] = False
        assert self.buffer[rest].isnan().all(), "written outside of the output"
        v = self.view.double()
        return v if self.experts == 1 else v.view(self.experts, self.rows, self.columns)


def output(q38m, rows, columns, dtype="bf16", spare=0, shift=0, experts=1):
    """An output that holds 7777 until it is written."""
    return Matrix(q38m, 0, rows, columns, dtype, spare=spare, shift=shift, experts=experts, fill=7777.0)


def arg(m):
    return None if m is None else m.arg


def product_bound(k, size):
    return (-(-k // 8) + 32) * 2.0 ** -23 * size



def close(got, want, bound, dtype, what):
    """got within bound of want, then half a step of the output's type (2^-9 of the value for bf16's
    8 significant bits; eps / 2), and 2^-126 for results below the smallest normal."""
    t = torch()
    got, want, bound = got.reshape(-1), want.reshape(-1), bound.expand_as(want).reshape(-1)
    assert t.equal(got.isnan(), want.isnan()), (what, int(got.isnan().sum()), int(want.isnan().sum()))
    ends = want.isinf()
    assert t.equal(got[ends], want[ends]), what
    live = ~(want.isnan() | ends)
    half = t.finfo(t.bfloat16 if dtype == "bf16" else t.float32).eps / 2
    limit = (bound * (1 + half) + half * want.abs() + 2.0 ** -126)[live]
    off = (got - want).abs()[live]
    assert (off <= limit).all(), (what, float((off / limit).max()), int((off > limit).sum()))


def sync():
    torch().cuda.synchronize()


def scratch_for(q38m, m, n, k):
    t = torch()
    nbytes = q38m.lib().q38m_linear_scratch_bytes(m, n, k)
    buffer = t.full((max(nbytes, 16) // 4 + 4,), float("nan"), dtype=t.float32, device="cuda")
    return buffer, buffer.data_ptr() if nbytes else None, nbytes


def run_linear(q38m, x, w, bias, act, residual, y, pre):
    scratch, at, nbytes = scratch_for(q38m, x.rows, w.rows, x.columns)
    q38m.call("q38m_linear_v1", x.arg, w.arg, arg(bias), q38m.ACTIVATIONS[act], arg(residual), y.arg, arg(pre), at,
              nbytes, stream(), 0)
    sync()


def check_linear(q38m, seed, m, n, k, act="none", bias=None, residual=None, out="bf16", keep=None, spare=(0, 0, 0),
                 shift=(0, 0, 0), sigma=1.0):
    """bias, residual, keep: their types, or None."""
    print(f"linear {m} x {n} x {k} {act} bias {bias} residual {residual} out {out} keep {keep} spare {spare} "
          f"shift {shift}", flush=True)
    x = Matrix(q38m, seed, m, k, spare=spare[0], shift=shift[0])
    w = Matrix(q38m, seed + 1, n, k, sigma=sigma * k ** -0.5, spare=spare[1], shift=shift[1])
    b = bias and Matrix(q38m, seed + 2, 1, n, bias, shift=shift[2])
    r = residual and Matrix(q38m, seed + 3, m, n, residual, spare=spare[2], shift=shift[2])
    y = output(q38m, m, n, out, spare[2], shift[2])
    p = keep and output(q38m, m, n, keep, spare[2], shift[2])
    run_linear(q38m, x, w, b, act, r, y, p)
    want, pre = lin.linear(x.values, w.values, b and b.values, act, r and r.values)
    size = x.values.abs() @ w.values.abs().T
    off = product_bound(k, size)
    if b:
        off = off + F32_ROUND * pre.abs() * (1 + 2.0 ** -20)
    if p:
        close(p.got(), pre, off, keep, "pre")
    off = 1.13 * off + (0 if act in ("none", "relu") else ACT_ERROR * pre.abs().clamp_min(1))
    if r:
        off = off + 2 * F32_ROUND * want.abs()
    close(y.got(), want, off, out, "y")
    return y


def check_backward_input(q38m, seed, m, n, k, act="none", residual=None, out="bf16", pre="bf16", spare=(0, 0, 0),
                         shift=(0, 0, 0)):
    print(f"input gradient {m} x {n} x {k} {act} residual {residual} out {out} pre {pre} spare {spare} shift {shift}",
          flush=True)
    dz = Matrix(q38m, seed, m, n, spare=spare[0], shift=shift[0])
    w = Matrix(q38m, seed + 1, n, k, sigma=n ** -0.5, spare=spare[1], shift=shift[1])
    z = None if act == "none" else Matrix(q38m, seed + 2, m, k, pre, sigma=2.0, spare=spare[2], shift=shift[2])
    r = residual and Matrix(q38m, seed + 3, m, k, residual, spare=spare[2], shift=shift[2])
    dx = output(q38m, m, k, out, spare[2], shift[2])
    scratch, at, nbytes = scratch_for(q38m, m, n, k)
    q38m.call("q38m_linear_backward_input_v1", dz.arg, w.arg, arg(z), q38m.ACTIVATIONS[act], arg(r), dx.arg, at,
              nbytes, stream(), 0)
    sync()
    want = dz.values @ w.values
    off = product_bound(n, dz.values.abs() @ w.values.abs())
    if z:
        slope = lin.slope(act, z.values)
        off = off * slope.abs() + want.abs() * ACT_ERROR * z.values.abs().clamp_min(1) + off * 2.0 ** -10
        want = want * slope
    if r:
        want = want + r.values
    off = off + 2 * F32_ROUND * (want.abs() + (r.values.abs() if r else 0))
    close(dx.got(), want, off, out, "dx")


def check_backward_weight(q38m, seed, m, n, k, residual=None, out="bf16", db="f32", spare=(0, 0, 0),
                          shift=(0, 0, 0), dw=True):
    print(f"weight gradient {m} x {n} x {k} residual {residual} out {out} db {db} spare {spare} shift {shift}",
          flush=True)
    dz = Matrix(q38m, seed, m, n, spare=spare[0], shift=shift[0])
    x = Matrix(q38m, seed + 1, m, k, sigma=m ** -0.5, spare=spare[1], shift=shift[1])
    r = residual and Matrix(q38m, seed + 2, n, k, residual, spare=spare[2], shift=shift[2])
    d = output(q38m, n, k, out, spare[2], shift[2]) if dw else None
    b = db and output(q38m, 1, n, db, shift=shift[2])
    scratch, at, nbytes = scratch_for(q38m, m, n, k)
    q38m.call("q38m_linear_backward_weight_v1", dz.arg, x.arg if dw else None, arg(r), arg(d), arg(b), at, nbytes,
              stream(), 0)
    sync()
    if dw:
        want = dz.values.T @ x.values
        off = product_bound(m, dz.values.abs().T @ x.values.abs())
        if r:
            off = off + 2 * F32_ROUND * (want.abs() + r.values.abs())
            want = want + r.values
        close(d.got(), want, off, out, "dw")
    if b:  # at most m additions behind one another
        close(b.got()[0], dz.values.sum(0), m * F32_ROUND * 2 * dz.values.abs().sum(0), db, "db")


class Sorted:
    """Rows sorted by expert: `counts` of each, then `dropped` of none, gathered from `tokens`."""

    def __init__(self, counts, dropped=0, tokens=0, top_k=1, seed=0):
        t = torch()
        self.experts, self.top_k = len(counts), top_k
        self.offsets = [0]
        for c in counts:
            self.offsets.append(self.offsets[-1] + c)
        self.routes = self.offsets[-1] + dropped
        self.offsets_on = t.tensor(self.offsets, dtype=t.int32, device="cuda")
        self.packed = self.source = None
        if tokens:
            assert tokens * top_k >= self.routes
            order = t.randperm(tokens * top_k, generator=generator(seed), device="cuda")[:self.routes]
            self.packed = order.int().contiguous()
            self.source = order // top_k

    def args(self):
        return (self.offsets_on.data_ptr(), None if self.packed is None else self.packed.data_ptr(), self.top_k)


def check_experts(q38m, seed, s, n, k, swiglu=False, out="bf16", keep=None, spare=(0, 0, 0), shift=(0, 0, 0),
                  tokens=0):
    """n: weight rows."""
    print(f"experts {s.experts} routes {s.routes} {n} x {k} swiglu {swiglu} out {out} keep {keep} tokens {tokens} "
          f"spare {spare} shift {shift}", flush=True)
    rows = Matrix(q38m, seed, tokens or s.routes, k, spare=spare[0], shift=shift[0])
    w = Matrix(q38m, seed + 1, n, k, sigma=k ** -0.5, spare=spare[1], shift=shift[1], experts=s.experts)
    weights = w.values if s.experts > 1 else w.values.unsqueeze(0)
    c = output(q38m, s.routes, n // 2 if swiglu else n, out, spare[2], shift[2])
    p = keep and output(q38m, s.routes, n, keep, spare[2], shift[2])
    q38m.call("q38m_moe_expert_gemm_v1", w.arg, rows.arg, *s.args(),
              q38m.EPILOGUE_SWIGLU if swiglu else q38m.EPILOGUE_NONE, c.arg, arg(p), stream(), 0)
    sync()
    t = torch()
    want = lin.experts(rows.values, weights, s.offsets, s.routes, s.source)
    off = product_bound(k, lin.experts(rows.values.abs(), weights.abs(), s.offsets, s.routes, s.source))
    live = ~want[:, 0].isnan()

    def left(m, value):  # rows of no expert stay as they were
        got = m.got()
        assert (got[~live] == 7776.0 if m.dtype == "bf16" else got[~live] == 7777.0).all()
        return got[live], value[live]

    if p:
        got, value = left(p, want)
        close(got, value, off[live], keep, "pre")
    if swiglu:
        gate, up = want.chunk(2, 1)
        d_gate, d_up = off.chunk(2, 1)
        silu = lin.activation("silu", gate)
        # eight roundings of h, |g| more (2^-17 of h at most) with a bf16 output
        off = 1.13 * d_gate * up.abs() + silu.abs() * d_up + d_gate * d_up + \
            (silu * up).abs() * (8 * F32_ROUND + (2.0 ** -17 if out == "bf16" else 0))
        want = silu * up
    got, value = left(c, want)
    close(got, value, off[live], out, "c")
    return t


def check_experts_rows(q38m, seed, s, n, k, pre=None, out="bf16", spare=(0, 0, 0), shift=(0, 0, 0)):
    print(f"experts' row gradient {s.experts} routes {s.routes} {n} x {k} pre {pre} out {out} spare {spare} "
          f"shift {shift}", flush=True)
    dc = Matrix(q38m, seed, s.routes, n, spare=spare[0], shift=shift[0])
    w = Matrix(q38m, seed + 1, n, k, sigma=n ** -0.5, spare=spare[1], shift=shift[1], experts=s.experts)
    weights = w.values if s.experts > 1 else w.values.unsqueeze(0)
    p = pre and Matrix(q38m, seed + 2, s.routes, 2 * k, pre, sigma=2.0, spare=spare[2], shift=shift[2])
    d = output(q38m, s.routes, 2 * k if pre else k, out, spare[2], shift[2])
    q38m.call("q38m_moe_expert_backward_rows_v1", w.arg, dc.arg, s.offsets_on.data_ptr(), arg(p), d.arg, stream(), 0)
    sync()
    want = lin.experts_backward_rows(dc.values, weights, s.offsets)
    off = product_bound(n, lin.experts_backward_rows(dc.values.abs(), weights.abs(), s.offsets))
    live = ~want[:, 0].isnan()
    if p:
        gate, up = p.values.chunk(2, 1)
        factor = torch().cat((up * lin.slope("silu", gate), lin.activation("silu", gate)), 1)
        scale = torch().cat((up.abs(), torch().ones_like(up)), 1) * ACT_ERROR * gate.abs().clamp_min(1).repeat(1, 2)
        off, want = off.repeat(1, 2) * (factor.abs() + scale) + want.repeat(1, 2).abs() * scale, want.repeat(1, 2) * factor
        off = off + 4 * F32_ROUND * want.abs()
    got = d.got()
    assert (got[~live] == (7776.0 if out == "bf16" else 7777.0)).all()
    close(got[live], want[live], off[live], out, "d_rows")


def check_experts_weights(q38m, seed, s, n, k, residual=None, out="bf16", spare=(0, 0, 0), shift=(0, 0, 0), tokens=0):
    print(f"experts' weight gradient {s.experts} routes {s.routes} {n} x {k} residual {residual} out {out} "
          f"tokens {tokens} spare {spare} shift {shift}", flush=True)
    dc = Matrix(q38m, seed, s.routes, n, spare=spare[0], shift=shift[0])
    rows = Matrix(q38m, seed + 1, tokens or s.routes, k, spare=spare[1], shift=shift[1])
    r = residual and Matrix(q38m, seed + 2, n, k, residual, spare=spare[2], shift=shift[2], experts=s.experts)
    d = output(q38m, n, k, out, spare[2], shift[2], s.experts)
    q38m.call("q38m_moe_expert_backward_weights_v1", dc.arg, rows.arg, *s.args(), arg(r), d.arg, stream(), 0)
    sync()
    want = lin.experts_backward_weights(dc.values, rows.values, s.offsets, s.experts, s.source)
    size = lin.experts_backward_weights(dc.values.abs(), rows.values.abs(), s.offsets, s.experts, s.source)
    longest = max(1, max(b - a for a, b in zip(s.offsets, s.offsets[1:])))
    off = product_bound(longest, size)
    got = d.got()
    if s.experts == 1:
        got = got.unsqueeze(0)
    if r:
        held = r.values if s.experts > 1 else r.values.unsqueeze(0)
        off = off + 2 * F32_ROUND * (want.abs() + held.abs())
        want = want + held
    close(got, want, off, out, "dw")
    empty = [e for e in range(s.experts) if s.offsets[e + 1] <= s.offsets[e]]
    if empty and not r:
        assert (got[empty] == 0).all()
