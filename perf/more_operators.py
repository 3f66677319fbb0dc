"""bf16 products with their epilogues and gradients, dense and by expert, as
measurable cases.

  linear         q38m_linear_v1: y = act(x W^T + bias) + residual, with the value
                 in front of the activation kept for training
  linear_grad    q38m_linear_backward_input_v1 and q38m_linear_backward_weight_v1:
                 the gradients of x (through the activation in front of it, plus a
                 residual branch's), of W (added to what a batch before left) and of
                 the bias
  experts        q38m_moe_expert_gemm_v1: rows sorted by expert times their expert's
                 matrix; gate/up with the SwiGLU fold, or down
  experts_grad   q38m_moe_expert_backward_rows_v1 and
                 q38m_moe_expert_backward_weights_v1: the gradients of both sides, of
                 down through the SwiGLU in front of it, or of gate/up

The model geometry is the library's (hidden 2048, 512 experts of intermediate
512, top-10) where a case does not say otherwise.
"""
import ctypes
import functools
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "qwen3.8-flash-next-dual-gpu_amd")

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
ACTIVATIONS = ("none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh")
TANH_SCALE, TANH_CUBE = math.sqrt(2 / math.pi), 0.044715


# ---- the cases --------------------------------------------------------------

def _linear(m, n, k, act="none", bias=True, residual=False, keep=False, out="bf16", spare=0):
    return {"kind": "linear", "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual, "keep": keep,
            "out": out, "spare": spare}


def _linear_grad(m, n, k, act="none", residual=False, add=False, out="bf16", dw="bf16", spare=0):
    return {"kind": "linear_grad", "m": m, "n": n, "k": k, "act": act, "residual": residual, "add": add, "out": out,
            "dw": dw, "spare": spare}


def _experts(tokens, up, wide=2048, narrow=512, keep=False, out="bf16", experts=512, top_k=10, zipf=0.0, dropped=0.0):
    return {"kind": "experts", "tokens": tokens, "up": up, "wide": wide, "narrow": narrow, "keep": keep, "out": out,
            "experts": experts, "top_k": top_k, "zipf": zipf, "dropped": dropped}


def _experts_grad(tokens, up, wide=2048, narrow=512, add=False, dw="bf16", experts=512, top_k=10, zipf=0.0,
                  dropped=0.0):
    return {"kind": "experts_grad", "tokens": tokens, "up": up, "wide": wide, "narrow": narrow, "add": add, "dw": dw,
            "experts": experts, "top_k": top_k, "zipf": zipf, "dropped": dropped}


def listed():
    return [
        # one generated token through a dense projection, as wide as the four hyper-connection streams
        {"name": "linear_token", **_linear(1, 8192, 2048, "silu")},
        # those streams back to one row width over a slab that is not full, onto the residual stream
        {"name": "linear_slab", **_linear(509, 2048, 8192, residual=True)},
        # a dense layer over a long training batch, its activation's input kept
        {"name": "linear_large", **_linear(8192, 8192, 8192, "gelu_tanh", keep=True)},
        # a short training batch's gradients, the weight's added up in fp32
        {"name": "linear_grad_batch", **_linear_grad(61, 8192, 2048, "silu", add=True, dw="f32")},
        # the first projection of a dense block over a long batch: the skip connection's gradient comes on top
        {"name": "linear_grad_large", **_linear_grad(8192, 8192, 2048, residual=True)},
        # gate/up of one generated token: ten experts of one row each
        {"name": "experts_token", **_experts(1, True)},
        # gate/up of a prefill slab: nearly every expert active, ten rows each
        {"name": "experts_slab", **_experts(512, True)},
        # down of a chunk that is not full, a skewed routing with dropped routes
        {"name": "experts_down", **_experts(3001, False, zipf=0.8, dropped=0.03)},
        # gate/up of the largest chunk in training: 640 rows for each expert, gate and up kept
        {"name": "experts_chunk", **_experts(32768, True, keep=True)},
        # a short training batch's gradients of down, through the SwiGLU
        {"name": "experts_grad_batch", **_experts_grad(61, False, dropped=0.03)},
        # gate/up's gradients over a long batch, the weights' added up in fp32
        {"name": "experts_grad_up", **_experts_grad(16384, True, add=True, dw="f32")},
        # down's gradients over a long batch
        {"name": "experts_grad_down", **_experts_grad(16384, False)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("linear", "linear_grad", "experts", "experts_grad"))
    if kind in ("linear", "linear_grad"):
        def side():
            return rng.choice((_log(rng, 1, 8192), 8 * _log(rng, 1, 1024), 64 * _log(rng, 1, 128)))
        m, n, k = _log(rng, 1, 8192), side(), side()
        act, spare = rng.choice(ACTIVATIONS), rng.choice((0, 0, 0, 8, 13))
        flag = [rng.choice((True, False)) for _ in range(3)]
        out = rng.choice(("bf16", "bf16", "f32"))
        if kind == "linear":
            return _linear(m, n, k, act, *flag, out, spare)
        return _linear_grad(m, n, k, act, *flag[:2], out, rng.choice(("bf16", "f32")), spare)
    experts = rng.choice((8, 60, 128, 256, 512))
    top_k = rng.choice([k for k in (1, 2, 4, 8, 10) if k <= experts])
    zipf, dropped = rng.choice((0.0, 0.0, 0.8)), rng.choice((0.0, 0.0, 0.05, 0.5))
    up, wide, narrow = rng.choice((True, False)), 8 * rng.randint(8, 256), 8 * rng.randint(4, 64)
    flag = rng.choice((True, False))
    if kind == "experts":
        tokens = _log(rng, 1, 2048 if zipf else 16384)
        return _experts(tokens, up, wide, narrow, flag and up, rng.choice(("bf16", "bf16", "f32")), experts, top_k,
                        zipf, dropped)
    tokens = _log(rng, 1, 2048 if zipf else 8192)
    return _experts_grad(tokens, up, wide, narrow, flag, rng.choice(("bf16", "f32")), experts, top_k, zipf, dropped)


# ---- work -------------------------------------------------------------------

def _matrix(c):
    """Rows and columns of an expert's matrix."""
    return (2 * c["narrow"], c["wide"]) if c["up"] else (c["wide"], c["narrow"])


def _active(c):
    """Experts that have a row, as many as uniform routing is expected to reach."""
    routes = c["tokens"] * c["top_k"] * (1.0 - c["dropped"])
    return c["experts"] * (1.0 - (1.0 - 1.0 / c["experts"]) ** routes)


def work(case):
    c = case
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        outputs = SIZE[c["out"]] + 2 * c["residual"] + 2 * c["keep"]
        return {"bytes": 2 * (m + n) * k + outputs * m * n + 4 * n * c["bias"], "flops": 2 * m * n * k}
    if c["kind"] == "linear_grad":
        m, n, k = c["m"], c["n"], c["k"]
        # dz, W and x read; what dx and dW take besides read; both and the bias' gradient written
        rows = SIZE[c["out"]] + 2 * c["residual"] + 2 * (c["act"] != "none")
        return {"bytes": 2 * (m * n + n * k + m * k) + rows * m * k + SIZE[c["dw"]] * (1 + c["add"]) * n * k + 4 * n,
                "flops": 4 * m * n * k + m * n}
    n, k = _matrix(c)
    routes = c["tokens"] * c["top_k"] * (1.0 - c["dropped"])
    source = c["tokens"] if c["up"] else routes  # rows that the product reads: token rows where they are gathered
    if c["kind"] == "experts":
        columns = c["narrow"] if c["up"] else n
        return {"bytes": 2 * (source + _active(c) * n) * k + routes * (columns * SIZE[c["out"]] + 2 * n * c["keep"]),
                "flops": 2 * routes * n * k}
    # dc, the weights and the rows read, dW (and what it is added to) and the rows' gradient; through the SwiGLU
    # gate and up are read and their two gradients written
    rows = k if c["up"] else 4 * k
    return {"bytes": 2 * (routes * n + _active(c) * n * k + source * k + routes * rows)
            + SIZE[c["dw"]] * (1 + c["add"]) * c["experts"] * n * k, "flops": 4 * routes * n * k}


# ---- inputs -----------------------------------------------------------------

def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 62))
    return g


def _normal(seed, salt, *shape, sigma=1.0, dtype=torch.bfloat16):
    """Normal values, a bounded number of them in fp32 at a time."""
    out = torch.empty(*shape, dtype=dtype, device="cuda")
    flat, step = out.view(-1), 1 << 27
    g = _generator(seed, salt)
    for first in range(0, flat.numel(), step):
        part = flat[first:first + step]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda").mul_(sigma))
    return out


def _ids(seed, c):
    """Expert ids [tokens][top_k], distinct within a token; dropped routes are -1."""
    logits = _normal(seed, 11, c["tokens"], c["experts"], dtype=torch.float32)
    if c["zipf"]:
        rank = torch.randperm(c["experts"], generator=_generator(seed, 12), device="cuda")
        logits = logits - c["zipf"] * torch.log1p(rank.float())
    ids = torch.topk(logits, c["top_k"], dim=1).indices
    if c["dropped"]:
        lost = torch.rand(ids.shape, generator=_generator(seed, 13), device="cuda") < c["dropped"]
        lost[c["tokens"] // 2] = True  # a token that no expert takes
        ids = torch.where(lost, -1, ids)
    return ids


def _sorted(ids, experts):
    """expert_offsets [experts + 1] and packed_assignment [routes], as int32."""
    flat = ids.reshape(-1)
    key, order = torch.sort(torch.where(flat >= 0, flat, experts), stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    return offsets.int(), order.int()


def _empty(rows, columns, dtype):
    return torch.empty(rows, columns, dtype=DTYPES[dtype], device="cuda")


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    if c["kind"] in ("linear", "linear_grad"):
        m, n, k = c["m"], c["n"], c["k"]
        s["x"] = _normal(seed, 1, m, k + c["spare"])[:, :k]
        s["w"] = _normal(seed, 2, n, k, sigma=k ** -0.5)
        if c["kind"] == "linear":
            s["bias"] = _normal(seed, 3, n, sigma=0.5, dtype=torch.float32) if c["bias"] else None
            s["residual"] = _normal(seed, 4, m, n) if c["residual"] else None
            s["y"] = _empty(m, n, c["out"])
            s["pre"] = _empty(m, n, "bf16") if c["keep"] else None
            # partial sums of products that are cut along k: more than a call asks for
            s["scratch"] = _scratch(m, n, k)
            return s
        s["dz"] = _normal(seed, 5, m, n, sigma=n ** -0.5)
        s["pre"] = _normal(seed, 6, m, k, sigma=2.0) if c["act"] != "none" else None
        s["residual"] = _normal(seed, 7, m, k) if c["residual"] else None
        s["add"] = _normal(seed, 8, n, k, dtype=DTYPES[c["dw"]]) if c["add"] else None
        s["dx"], s["dw"] = _empty(m, k, c["out"]), _empty(n, k, c["dw"])
        s["db"] = torch.empty(n, dtype=torch.float32, device="cuda")
        s["scratch"] = _scratch(m, n, k)
        return s
    ids = _ids(seed, c)
    routes, (n, k) = ids.numel(), _matrix(c)
    s["offsets"], s["packed"] = _sorted(ids, c["experts"])
    s["cap"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))
    s["w"] = _normal(seed, 21, c["experts"], n, k, sigma=k ** -0.5)
    s["rows"] = _normal(seed, 22, c["tokens"] if c["up"] else routes, k)
    # rows of dropped routes lie behind the experts' and stay as they are
    if c["kind"] == "experts":
        s["c"] = _empty(routes, c["narrow"] if c["up"] else n, c["out"]).zero_()
        s["pre"] = _empty(routes, n, "bf16").zero_() if c["keep"] else None
        return s
    s["dc"] = _normal(seed, 23, routes, n, sigma=n ** -0.5)
    s["pre"] = None if c["up"] else _normal(seed, 24, routes, 2 * k)
    s["d_rows"] = _empty(routes, k if c["up"] else 2 * k, "bf16").zero_()
    s["add"] = _normal(seed, 25, c["experts"] * n, k, dtype=DTYPES[c["dw"]]) if c["add"] else None
    s["dw"] = _empty(c["experts"] * n, k, c["dw"])
    return s


def _scratch(m, n, k):
    """Room for 16 partial sums of the smallest results, fewer of larger ones, and copies of operands."""
    largest = max(m * n, n * k, m * k)
    return torch.empty(min(64 * largest, 4 * largest + (1 << 29)) + (1 << 20), dtype=torch.uint8, device="cuda")


# ---- plain forms ------------------------------------------------------------

def _activation(act, z):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * TANH_SCALE * (z + TANH_CUBE * z ** 3)))
    if act == "none":
        return z
    s = 1 / (1 + torch.exp(-z))
    return s if act == "sigmoid" else z * s


def _slope(act, z):
    """The activation's derivative."""
    if act == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        s = 1 / (1 + torch.exp(-2 * TANH_SCALE * (z + TANH_CUBE * z ** 3)))
        return s + z * s * (1 - s) * 2 * TANH_SCALE * (1 + 3 * TANH_CUBE * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if act == "sigmoid" else s * (1 + z * (1 - s))


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().T
    if c["bias"]:
        z = z + s["bias"]
    y = _activation(c["act"], z)
    if c["residual"]:
        y = y + s["residual"].float()
    return {"y": y.to(DTYPES[c["out"]]), "pre": z.bfloat16() if c["keep"] else None}


def _plain_linear_grad(s):
    c = s["case"]
    dz = s["dz"].float()
    dx = dz @ s["w"].float()
    if c["act"] != "none":
        dx = dx * _slope(c["act"], s["pre"].float())
    if c["residual"]:
        dx = dx + s["residual"].float()
    dw = dz.T @ s["x"].float()
    if c["add"]:
        dw = dw + s["add"].float()
    return {"dx": dx.to(DTYPES[c["out"]]), "dw": dw.to(DTYPES[c["dw"]]), "db": dz.sum(0)}


def _places(s):
    """Of every sorted row its expert and whether it has one; its place where every expert's rows lie side by side,
    as many places as the fullest has rows, and one place behind them for the rows of no expert."""
    c, place = s["case"], torch.arange(s["packed"].numel(), device="cuda")
    offsets = s["offsets"].long()
    live = place < offsets[-1]
    expert = torch.where(live, torch.searchsorted(offsets, place, right=True) - 1, 0)
    at = torch.where(live, expert * s["cap"] + place - offsets[expert], c["experts"] * s["cap"])
    return expert, live, at


def _beside(s, rows, at):
    c = s["case"]
    out = torch.zeros(c["experts"] * s["cap"] + 1, rows.shape[1], device="cuda")
    out[at] = rows
    out[-1] = 0
    return out[:-1].view(c["experts"], s["cap"], -1)


def _taken(s):
    """fp32 rows of the sorted order."""
    rows = s["rows"].float()
    return rows[s["packed"].long() // s["case"]["top_k"]] if s["case"]["up"] else rows


def _plain_experts(s):
    c = s["case"]
    expert, live, at = _places(s)
    rows = _taken(s)
    if rows.shape[0] < c["experts"]:  # few rows: each with its own copy of its expert
        out = (s["w"][expert].float() @ rows.unsqueeze(2)).squeeze(2)
    else:
        out = torch.bmm(_beside(s, rows, at), s["w"].float().transpose(1, 2).contiguous()).flatten(0, 1)
        out = out[torch.where(live, at, 0)]
    pre = out
    if c["up"]:
        gate, up = out.chunk(2, 1)
        out = gate / (1 + torch.exp(-gate)) * up
    live = live.unsqueeze(1)
    return {"c": torch.where(live, out, s["c"].float()).to(DTYPES[c["out"]]),
            "pre": torch.where(live, pre, s["pre"].float()).bfloat16() if c["keep"] else None}


def _plain_experts_grad(s):
    c = s["case"]
    expert, live, at = _places(s)
    dc = s["dc"].float()
    beside = _beside(s, dc, at)
    if dc.shape[0] < c["experts"]:
        d_rows = (dc.unsqueeze(1) @ s["w"][expert].float()).squeeze(1)
    else:
        d_rows = torch.bmm(beside, s["w"].float()).flatten(0, 1)[torch.where(live, at, 0)]
    if not c["up"]:
        gate, up = s["pre"].float().chunk(2, 1)
        sigmoid = 1 / (1 + torch.exp(-gate))
        d_rows = torch.cat((d_rows * up * sigmoid * (1 + gate * (1 - sigmoid)), d_rows * gate * sigmoid), 1)
    d_rows = torch.where(live.unsqueeze(1), d_rows, s["d_rows"].float()).bfloat16()
    dw = torch.bmm(beside.transpose(1, 2).contiguous(), _beside(s, _taken(s), at)).flatten(0, 1)
    if c["add"]:
        dw = dw + s["add"].float()
    return {"d_rows": d_rows, "dw": dw.to(DTYPES[c["dw"]])}


PLAIN = {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "experts": _plain_experts,
         "experts_grad": _plain_experts_grad}


# ---- the library's calls ----------------------------------------------------

@functools.lru_cache(None)
def _q38m():
    name = "q38m_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(PACKAGE, "__init__.py"), submodule_search_locations=[PACKAGE])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _tensor(q, t, experts=1):
    """A descriptor of a matrix, of experts' matrices one below the other, or of a vector; None of nothing."""
    if t is None:
        return None
    flat = t.flatten(0, -2) if t.dim() > 1 else t.unsqueeze(0)
    dtype = q.DTYPE_BF16 if t.dtype == torch.bfloat16 else q.DTYPE_F32
    return ctypes.byref(q.Tensor(t.data_ptr(), flat.stride(0), dtype, experts, flat.shape[0] // experts,
                                 flat.shape[1]))


def _calls(s):
    """The calls' names and arguments, descriptors and all: a program keeps them beside its buffers."""
    q, c = _q38m(), s["case"]
    t = functools.partial(_tensor, q)
    if c["kind"] in ("linear", "linear_grad"):
        act = q.ACTIVATIONS[c["act"]]
        scratch = (s["scratch"].data_ptr(), s["scratch"].numel())
        if c["kind"] == "linear":
            return [("q38m_linear_v1", t(s["x"]), t(s["w"]), t(s["bias"]), act, t(s["residual"]), t(s["y"]),
                     t(s["pre"]), *scratch)]
        return [("q38m_linear_backward_input_v1", t(s["dz"]), t(s["w"]), t(s["pre"]), act, t(s["residual"]),
                 t(s["dx"]), *scratch),
                ("q38m_linear_backward_weight_v1", t(s["dz"]), t(s["x"]), t(s["add"]), t(s["dw"]), t(s["db"]),
                 *scratch)]
    experts, top_k, offsets = c["experts"], c["top_k"], s["offsets"].data_ptr()
    packed = s["packed"].data_ptr() if c["up"] else None
    if c["kind"] == "experts":
        epilogue = q.EPILOGUE_SWIGLU if c["up"] else q.EPILOGUE_NONE
        return [("q38m_moe_expert_gemm_v1", t(s["w"], experts), t(s["rows"]), offsets, packed, top_k, epilogue,
                 t(s["c"]), t(s["pre"]))]
    return [("q38m_moe_expert_backward_rows_v1", t(s["w"], experts), t(s["dc"]), offsets, t(s["pre"]),
             t(s["d_rows"])),
            ("q38m_moe_expert_backward_weights_v1", t(s["dc"]), t(s["rows"]), offsets, packed, top_k,
             t(s["add"], experts), t(s["dw"], experts))]


OUTPUTS = {"linear": ("y", "pre"), "linear_grad": ("dx", "dw", "db"), "experts": ("c", "pre"),
           "experts_grad": ("d_rows", "dw")}


def _own(s):
    if "calls" not in s:
        s["calls"] = _calls(s)
    call, stream = _q38m().call, _stream()
    for arguments in s["calls"]:
        call(*arguments, stream, 0)
    return {name: s[name] for name in OUTPUTS[s["case"]["kind"]]}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- 64 bits ----------------------------------------------------------------

def _exact_act(act, z):
    """An activation and its derivative, float64."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "gelu":
        below = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        tanh = torch.tanh(TANH_SCALE * (z + TANH_CUBE * z ** 3))
        return (z * (1 + tanh) / 2,
                (1 + tanh) / 2 + z / 2 * (1 - tanh * tanh) * TANH_SCALE * (1 + 3 * TANH_CUBE * z * z))
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if act == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "linear":
        z = torch.matmul(s["x"].double(), s["w"].double().T.contiguous())
        if c["bias"]:
            z += s["bias"].double()
        y = _exact_act(c["act"], z)[0]
        return {"y": y + s["residual"].double() if c["residual"] else y, "pre": z if c["keep"] else None}
    if c["kind"] == "linear_grad":
        dz = s["dz"].double()
        dx = torch.matmul(dz, s["w"].double())
        if c["act"] != "none":
            dx *= _exact_act(c["act"], s["pre"].double())[1]
        if c["residual"]:
            dx += s["residual"].double()
        dw = torch.matmul(dz.T.contiguous(), s["x"].double())
        return {"dx": dx, "dw": dw + s["add"].double() if c["add"] else dw, "db": dz.sum(0)}
    at, n = s["offsets"].tolist(), _matrix(c)[0]
    token = s["packed"].long().div(c["top_k"], rounding_mode="floor") if c["up"] else None
    if c["kind"] == "experts":
        out, pre = s["c"].double(), s["pre"].double() if c["keep"] else None
    else:
        d_rows = s["d_rows"].double()
        dw = s["add"].double() if c["add"] else torch.zeros(s["dw"].shape, dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        p = slice(at[e], at[e + 1])
        if at[e] == at[e + 1]:
            continue
        rows = (s["rows"][token[p]] if c["up"] else s["rows"][p]).double()
        if c["kind"] == "experts":
            y = torch.matmul(rows, s["w"][e].double().T.contiguous())
            if c["keep"]:
                pre[p] = y
            if c["up"]:
                gate, up = y[:, :c["narrow"]], y[:, c["narrow"]:]
                y = _exact_act("silu", gate)[0] * up
            out[p] = y
            continue
        dc = s["dc"][p].double()
        dh = torch.matmul(dc, s["w"][e].double())
        if c["up"]:
            d_rows[p] = dh
        else:
            gate, up = s["pre"][p, :c["narrow"]].double(), s["pre"][p, c["narrow"]:].double()
            silu, slope = _exact_act("silu", gate)
            d_rows[p, :c["narrow"]] = dh * up * slope
            d_rows[p, c["narrow"]:] = dh * silu
        dw[e * n:(e + 1) * n] += torch.matmul(dc.T.contiguous(), rows)
    return {"c": out, "pre": pre} if c["kind"] == "experts" else {"d_rows": d_rows, "dw": dw}
