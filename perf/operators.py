"""Microscaled 4-bit rows, their products, and tokens sorted by expert and back,
as measurable cases.

  quantize  q38m_mx_quantize_v1: rows to 4-bit codes with a power-of-two scale
            for every 32 values, and the values that the codes stand for
  product   q38m_mx_gemm_v1: C = A B^T of two such matrices
  experts   q38m_mx_grouped_gemm_v1: rows sorted by expert times their expert's
            matrix; gate/up with the SwiGLU fold, or down
  route     q38m_moe_sort_routes_v1, q38m_moe_permute_rows_v1 and
            q38m_moe_unpermute_rows_v1: tokens to expert order, and the experts'
            rows back with the router's weights
  gradient  q38m_moe_unpermute_backward_v1 and q38m_moe_unpermute_rows_v1: the
            gradients of both directions

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

BLOCK, PAD = 32, 128
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


# ---- the cases --------------------------------------------------------------

def _quantize(rows, columns, dtype="bf16", spare=0):
    return {"kind": "quantize", "rows": rows, "columns": columns, "dtype": dtype, "spare": spare}


def _product(m, n, k, out="bf16"):
    return {"kind": "product", "m": m, "n": n, "k": k, "out": out}


def _experts(tokens, n, k, swiglu, gather, out="bf16", experts=512, top_k=10, zipf=0.0, dropped=0.0):
    return {"kind": "experts", "tokens": tokens, "n": n, "k": k, "swiglu": swiglu, "gather": gather, "out": out,
            "experts": experts, "top_k": top_k, "zipf": zipf, "dropped": dropped}


def _routes(kind, tokens, width, dtype="bf16", experts=512, top_k=10, zipf=0.0, dropped=0.0):
    return {"kind": kind, "tokens": tokens, "width": width, "dtype": dtype, "experts": experts, "top_k": top_k,
            "zipf": zipf, "dropped": dropped}


def listed():
    return [
        # one generated token: the ten mid rows between its experts' two products
        {"name": "quantize_mid_rows", **_quantize(10, 512)},
        # the token rows of the largest chunk
        {"name": "quantize_chunk", **_quantize(32768, 2048)},
        # a dense projection for one token, as wide as the four hyper-connection streams
        {"name": "product_token", **_product(1, 8192, 2048)},
        # those streams back to one row width over a slab that is not full; fp32 for a sum that follows
        {"name": "product_slab", **_product(509, 2048, 8192, "f32")},
        # a dense layer over a long batch
        {"name": "product_large", **_product(8192, 8192, 8192)},
        # gate/up of one generated token: ten experts of one row each
        {"name": "experts_token", **_experts(1, 1024, 2048, True, True)},
        # gate/up of a prefill slab: nearly every expert active, ten rows each
        {"name": "experts_slab", **_experts(512, 1024, 2048, True, True)},
        # gate/up of the largest chunk: 640 rows for each expert
        {"name": "experts_chunk", **_experts(32768, 1024, 2048, True, True)},
        # a prefill slab's rows to the experts and back, some routes dropped
        {"name": "route_slab", **_routes("route", 512, 2048, dropped=0.03)},
        # the largest chunk
        {"name": "route_chunk", **_routes("route", 32768, 2048, zipf=0.8)},
        # a small training batch in fp32
        {"name": "gradient_batch", **_routes("gradient", 61, 2048, "f32", dropped=0.03)},
        # a long training batch
        {"name": "gradient_chunk", **_routes("gradient", 16384, 2048)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("quantize", "product", "experts", "route", "gradient"))
    if kind == "quantize":
        columns = rng.choice((rng.randint(1, 512), 32 * rng.randint(1, 256)))
        rows = _log(rng, 1, min(65536, (1 << 26) // columns))
        return _quantize(rows, columns, rng.choice(("bf16", "f32")), rng.choice((0, 0, 8, 13)))
    if kind == "product":
        n, k = _log(rng, 1, 8192), rng.choice((_log(rng, 1, 8192), 128 * rng.randint(1, 64)))
        return _product(_log(rng, 1, 8192), n, k, rng.choice(("bf16", "f32")))
    experts = rng.choice((8, 60, 128, 256, 512))
    top_k = rng.choice([k for k in (1, 2, 4, 8, 10) if k <= experts])
    zipf, dropped = rng.choice((0.0, 0.0, 0.8)), rng.choice((0.0, 0.0, 0.05, 0.5))
    if kind == "experts":
        up = rng.choice((True, False))
        wide, narrow = 128 * rng.randint(2, 16), 64 * rng.randint(1, 8)
        n, k = (2 * narrow, wide) if up else (wide, narrow)
        tokens = _log(rng, 1, 2048 if zipf else 16384)
        return _experts(tokens, n, k, up, up, rng.choice(("bf16", "bf16", "f32")), experts, top_k, zipf, dropped)
    width = rng.choice((8 * rng.randint(1, 512), rng.randint(1, 600), 2048))
    tokens = _log(rng, 1, min(32768 if kind == "route" else 16384, (1 << 28) // (width * top_k)))
    return _routes(kind, tokens, width, rng.choice(("bf16", "f32")), experts, top_k, zipf, dropped)


# ---- work -------------------------------------------------------------------

def _mx_bytes(rows, columns):
    return rows * (-(-columns // 2) + -(-columns // BLOCK))


def _active(c):
    """Experts that have a row, as many as uniform routing is expected to reach."""
    routes = c["tokens"] * c["top_k"] * (1.0 - c["dropped"])
    return c["experts"] * (1.0 - (1.0 - 1.0 / c["experts"]) ** routes)


def work(case):
    c = case
    if c["kind"] == "quantize":
        values = c["rows"] * c["columns"]
        return {"bytes": 2 * SIZE[c["dtype"]] * values + _mx_bytes(c["rows"], c["columns"]), "flops": 2 * values}
    if c["kind"] == "product":
        return {"bytes": _mx_bytes(c["m"] + c["n"], c["k"]) + c["m"] * c["n"] * SIZE[c["out"]],
                "flops": 2 * c["m"] * c["n"] * c["k"]}
    routes = c["tokens"] * c["top_k"] * (1.0 - c["dropped"])
    if c["kind"] == "experts":
        rows = c["tokens"] if c["gather"] else routes
        columns = c["n"] // 2 if c["swiglu"] else c["n"]
        return {"bytes": _mx_bytes(rows + _active(c) * c["n"], c["k"]) + routes * columns * SIZE[c["out"]],
                "flops": 2 * routes * c["n"] * c["k"]}
    row = c["width"] * SIZE[c["dtype"]]
    index = 4 * c["tokens"] * c["top_k"]
    if c["kind"] == "route":
        # ids read, both orders written; x read and its routes written; the experts' rows read, y written
        return {"bytes": 4 * index + 2 * (c["tokens"] + routes) * row, "flops": 2 * routes * c["width"]}
    # dy, the experts' rows and the sorted rows' gradient read; the rows' and the tokens' gradients written
    return {"bytes": 3 * index + (2 * c["tokens"] + 3 * routes) * row, "flops": 4 * routes * c["width"]}


# ---- inputs -----------------------------------------------------------------

def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 62))
    return g


def _normal(seed, salt, *shape):
    return torch.randn(*shape, generator=_generator(seed, salt), device="cuda")


def _row_stride(columns):
    return -(-columns // PAD) * PAD


def _encode(x):
    """fp32 [..., columns] -> (codes uint8 [..., padded / 2], scales uint8 [..., padded / 32]), the low nibble first."""
    pad = _row_stride(x.shape[-1]) - x.shape[-1]
    x = torch.nn.functional.pad(x, (0, pad)) if pad else x
    x = x.unflatten(-1, (-1, BLOCK))
    field = x.abs().amax(-1).contiguous().view(torch.int32) >> 23  # the exponent of the largest magnitude
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(bad, 255, (field - 2).clamp_min(0))
    inverse = ((254 - scale) << 23).clamp_min(0).view(torch.float32)
    v = torch.where(bad.unsqueeze(-1), 0.0, x * inverse.unsqueeze(-1))
    mag = v.abs()
    code = torch.where(mag < 2, torch.round(2 * mag),
                       torch.where(mag < 4, torch.round(mag) + 2, (torch.round(mag / 2) + 4).clamp_max(7)))
    code = code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.to(torch.uint8)


def _encoded_normal(seed, salt, rows, columns, sigma):
    """Encoded rows of normal values, a bounded number at a time; the padded values are zero."""
    step = max(1, (1 << 27) // _row_stride(columns))
    parts = [_encode(sigma * _normal(seed, salt + 7 * i, min(step, rows - first), columns))
             for i, first in enumerate(range(0, rows, step))]
    return tuple(torch.cat(p) if len(p) > 1 else p[0].contiguous() for p in zip(*parts))


def _ids(seed, c):
    """Expert ids [tokens][top_k] int32, distinct within a token, best first; dropped routes are -1."""
    logits = _normal(seed, 11, c["tokens"], c["experts"])
    if c["zipf"]:
        rank = torch.randperm(c["experts"], generator=_generator(seed, 12), device="cuda")
        logits = logits - c["zipf"] * torch.log1p(rank.float())
    best = torch.topk(logits, c["top_k"], dim=1)
    ids = best.indices.int()
    if c["dropped"]:
        lost = torch.rand(ids.shape, generator=_generator(seed, 13), device="cuda") < c["dropped"]
        lost[c["tokens"] // 2] = True  # a token that no expert takes
        ids = torch.where(lost, -1, ids)
    return ids.contiguous(), torch.softmax(best.values, dim=1).contiguous()


def _sorted(ids, experts):
    """expert_offsets [experts + 1], packed_assignment and assignment_to_packed [routes], as int32."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device, dtype=key.dtype))
    place = torch.arange(flat.numel(), device=key.device)
    inverse = torch.empty_like(place)
    inverse[order] = torch.where(place < offsets[-1], place, -1)
    return offsets.int(), order.int(), inverse.int()


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    if c["kind"] == "quantize":
        # activations: rows of different size, a few large channels
        x = _normal(seed, 1, c["rows"], c["columns"] + c["spare"])
        x *= torch.exp(_normal(seed, 2, c["rows"], 1))
        x *= 1 + 15 * (torch.rand(x.shape[1], generator=_generator(seed, 3), device="cuda") < 0.01)
        s["x"] = x.to(DTYPES[c["dtype"]])[:, :c["columns"]]
        padded = _row_stride(c["columns"])
        s["codes"] = torch.empty(c["rows"], padded // 2, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(c["rows"], padded // BLOCK, dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty(c["rows"], c["columns"], dtype=DTYPES[c["dtype"]], device="cuda")
        return s
    if c["kind"] == "product":
        s["a"] = _encoded_normal(seed, 1000, c["m"], c["k"], 1.0)
        s["b"] = _encoded_normal(seed, 2000, c["n"], c["k"], c["k"] ** -0.5)
        s["c"] = torch.empty(c["m"], c["n"], dtype=DTYPES[c["out"]], device="cuda")
        return s
    ids, weights = _ids(seed, c)
    routes = ids.numel()
    if c["kind"] == "experts":
        s["offsets"], s["packed"], _ = _sorted(ids, c["experts"])
        s["cap"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["rows"] = _encoded_normal(seed, 3000, c["tokens"] if c["gather"] else routes, c["k"], 1.0)
        s["weights"] = _encoded_normal(seed, 4000, c["experts"] * c["n"], c["k"], c["k"] ** -0.5)
        # rows of dropped routes lie behind the experts' and stay as they are
        s["c"] = torch.zeros(routes, c["n"] // 2 if c["swiglu"] else c["n"], dtype=DTYPES[c["out"]], device="cuda")
        return s
    dtype, width = DTYPES[c["dtype"]], c["width"]
    s["route_weights"] = weights
    s["expert_rows"] = _normal(seed, 21, routes, width).to(dtype)
    if c["kind"] == "route":
        s["ids"] = ids
        s["x"] = _normal(seed, 22, c["tokens"], width).to(dtype)
        s["packed_rows"] = torch.zeros(routes, width, dtype=dtype, device="cuda")
        s["y"] = torch.empty(c["tokens"], width, dtype=dtype, device="cuda")
        s["offsets"] = torch.empty(c["experts"] + 1, dtype=torch.int32, device="cuda")
        s["packed"] = torch.empty(routes, dtype=torch.int32, device="cuda")
        s["inverse"] = torch.empty(routes, dtype=torch.int32, device="cuda")
        # counts of up to 1,024 experts for every 64 routes: more than a sort asks for
        s["scratch"] = torch.empty(8 * (c["experts"] + 1) * (2 + routes // 64), dtype=torch.uint8, device="cuda")
        return s
    s["offsets"], s["packed"], s["inverse"] = _sorted(ids, c["experts"])
    s["dy"] = _normal(seed, 23, c["tokens"], width).to(dtype)
    s["d_packed"] = _normal(seed, 24, routes, width).to(dtype)
    s["d_rows"] = torch.zeros(routes, width, dtype=dtype, device="cuda")
    s["d_weights"] = torch.empty(c["tokens"], c["top_k"], dtype=torch.float32, device="cuda")
    s["dx"] = torch.empty(c["tokens"], width, dtype=dtype, device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------

@functools.lru_cache(None)
def _pairs():
    """fp32 [256][2]: the two magnitudes with their signs of a byte of codes."""
    values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device="cuda")
    byte = torch.arange(256, device="cuda")
    return torch.stack((values[byte & 15], values[byte >> 4]), 1)


def _decode(codes, scales, columns):
    """fp32 [..., columns] of encoded rows."""
    v = _pairs()[codes.int()].flatten(-2).unflatten(-1, (-1, BLOCK))
    scale = scales.int()
    # 2^(byte - 127): byte 0 is the largest subnormal power of two, 255 is no number
    factor = torch.where(scale > 0, scale << 23, 1 << 22).view(torch.float32)
    factor = torch.where(scale == 255, float("nan"), factor)
    return (v * factor.unsqueeze(-1)).flatten(-2)[..., :columns]


def _plain_quantize(s):
    c = s["case"]
    codes, scales = _encode(s["x"].float())
    return {"codes": codes, "scales": scales, "values": _decode(codes, scales, c["columns"]).to(DTYPES[c["dtype"]])}


def _plain_product(s):
    c = s["case"]
    return (_decode(*s["a"], c["k"]) @ _decode(*s["b"], c["k"]).T).to(DTYPES[c["out"]])


def _plain_experts(s):
    c = s["case"]
    place = torch.arange(s["packed"].numel(), device="cuda")
    offsets = s["offsets"].long()
    expert = torch.searchsorted(offsets, place, right=True) - 1
    live = place < offsets[-1]
    expert = torch.where(live, expert, 0)
    rows = _decode(*s["rows"], c["k"])
    if c["gather"]:
        rows = rows[s["packed"].long() // c["top_k"]]
    codes, scales = (w.view(c["experts"], c["n"], -1) for w in s["weights"])
    if rows.shape[0] < c["experts"]:  # few rows: each with its own copy of its expert
        out = (_decode(codes[expert], scales[expert], c["k"]) @ rows.unsqueeze(2)).squeeze(2)
    else:
        # every expert's rows side by side, as many places as the fullest has rows; one place more takes the dropped ones
        at = torch.where(live, expert * s["cap"] + place - offsets[expert], c["experts"] * s["cap"])
        beside = torch.zeros(c["experts"] * s["cap"] + 1, c["k"], device="cuda")
        beside[at] = rows
        weights = _decode(codes, scales, c["k"]).transpose(1, 2).contiguous()
        out = torch.bmm(beside[:-1].view(c["experts"], s["cap"], c["k"]), weights).flatten(0, 1)
        out = out[torch.where(live, at, 0)]
    if c["swiglu"]:
        gate, up = out.chunk(2, 1)
        out = gate / (1 + torch.exp(-gate)) * up
    return torch.where(live.unsqueeze(1), out, s["c"].float()).to(DTYPES[c["out"]])


def _back(rows, inverse, weights, tokens):
    """fp32 [tokens][width]: the sum over a token's routes of its rows times the weights, where it has them."""
    live = inverse >= 0
    taken = torch.where(live.unsqueeze(1), rows[inverse.clamp_min(0).long()].float(), 0.0)
    if weights is not None:
        taken = taken * torch.where(live, weights.reshape(-1), 0.0).unsqueeze(1)
    return taken.view(tokens, -1, rows.shape[1]).sum(1)


def _plain_route(s):
    c = s["case"]
    offsets, packed, inverse = _sorted(s["ids"], c["experts"])
    live = torch.arange(packed.numel(), device="cuda") < offsets[-1]
    rows = torch.where(live.unsqueeze(1), s["x"][packed.long() // c["top_k"]], s["packed_rows"])
    y = _back(s["expert_rows"], inverse, s["route_weights"], c["tokens"]).to(DTYPES[c["dtype"]])
    return {"offsets": offsets, "packed": packed, "inverse": inverse, "packed_rows": rows, "y": y}


def _plain_gradient(s):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    packed = s["packed"].long()
    live = torch.arange(packed.numel(), device="cuda") < s["offsets"][-1]
    d_rows = s["route_weights"].reshape(-1)[packed].unsqueeze(1) * s["dy"][packed // c["top_k"]].float()
    d_rows = torch.where(live.unsqueeze(1), d_rows, s["d_rows"].float()).to(dtype)
    taken = s["expert_rows"][s["inverse"].clamp_min(0).long()].float().view(c["tokens"], c["top_k"], -1)
    d_weights = (taken * s["dy"].float().unsqueeze(1)).sum(2)
    d_weights = torch.where(s["inverse"].view_as(d_weights) >= 0, d_weights, 0.0)
    dx = _back(s["d_packed"], s["inverse"], None, c["tokens"]).to(dtype)
    return {"d_rows": d_rows, "d_weights": d_weights, "dx": dx}


PLAIN = {"quantize": _plain_quantize, "product": _plain_product, "experts": _plain_experts, "route": _plain_route,
         "gradient": _plain_gradient}


# ---- the library's calls ------------------------------------------------------

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


def _dtype(q, name):
    return q.DTYPE_BF16 if name == "bf16" else q.DTYPE_F32


def _matrix(q, codes, scales, experts, rows, columns):
    return ctypes.byref(q.MxMatrix(codes.data_ptr(), scales.data_ptr(), experts, rows, columns))


def _out(c, buffer):
    """The fp32 and the bf16 output argument, one of them null."""
    return (buffer.data_ptr(), None) if c["out"] == "f32" else (None, buffer.data_ptr())


def _own_quantize(s):
    q, c, x = _q38m(), s["case"], s["x"]
    q.call("q38m_mx_quantize_v1", x.data_ptr(), _dtype(q, c["dtype"]), x.stride(0),
           _matrix(q, s["codes"], s["scales"], 1, c["rows"], c["columns"]), s["values"].data_ptr(), _stream(), 0)
    return {"codes": s["codes"], "scales": s["scales"], "values": s["values"]}


def _own_product(s):
    q, c = _q38m(), s["case"]
    q.call("q38m_mx_gemm_v1", _matrix(q, *s["a"], 1, c["m"], c["k"]), _matrix(q, *s["b"], 1, c["n"], c["k"]),
           *_out(c, s["c"]), c["n"], _stream(), 0)
    return s["c"]


def _own_experts(s):
    q, c = _q38m(), s["case"]
    q.call("q38m_mx_grouped_gemm_v1", _matrix(q, *s["weights"], c["experts"], c["n"], c["k"]),
           _matrix(q, *s["rows"], 1, s["rows"][0].shape[0], c["k"]), s["offsets"].data_ptr(),
           s["packed"].data_ptr() if c["gather"] else None, c["top_k"], s["packed"].numel(),
           q.MX_EPILOGUE_SWIGLU if c["swiglu"] else q.MX_EPILOGUE_NONE, *_out(c, s["c"]), _stream(), 0)
    return s["c"]


def _own_route(s):
    q, c, stream = _q38m(), s["case"], _stream()
    dtype = _dtype(q, c["dtype"])
    q.call("q38m_moe_sort_routes_v1", s["ids"].data_ptr(), c["tokens"], c["top_k"], c["experts"],
           s["offsets"].data_ptr(), s["packed"].data_ptr(), s["inverse"].data_ptr(), s["scratch"].data_ptr(),
           s["scratch"].numel(), stream, 0)
    q.call("q38m_moe_permute_rows_v1", s["x"].data_ptr(), dtype, s["inverse"].data_ptr(), c["tokens"], c["top_k"],
           c["width"], s["packed_rows"].data_ptr(), stream, 0)
    q.call("q38m_moe_unpermute_rows_v1", s["expert_rows"].data_ptr(), dtype, s["inverse"].data_ptr(),
           s["route_weights"].data_ptr(), c["tokens"], c["top_k"], c["width"], s["y"].data_ptr(), stream, 0)
    return {k: s[k] for k in ("offsets", "packed", "inverse", "packed_rows", "y")}


def _own_gradient(s):
    q, c, stream = _q38m(), s["case"], _stream()
    dtype = _dtype(q, c["dtype"])
    q.call("q38m_moe_unpermute_backward_v1", s["dy"].data_ptr(), s["expert_rows"].data_ptr(), dtype,
           s["inverse"].data_ptr(), s["route_weights"].data_ptr(), c["tokens"], c["top_k"], c["width"],
           s["d_rows"].data_ptr(), s["d_weights"].data_ptr(), stream, 0)
    q.call("q38m_moe_unpermute_rows_v1", s["d_packed"].data_ptr(), dtype, s["inverse"].data_ptr(), None, c["tokens"],
           c["top_k"], c["width"], s["dx"].data_ptr(), stream, 0)
    return {k: s[k] for k in ("d_rows", "d_weights", "dx")}


OWN = {"quantize": _own_quantize, "product": _own_product, "experts": _own_experts, "route": _own_route,
       "gradient": _own_gradient}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---- 64 bits ----------------------------------------------------------------

def _value(nibble):
    """float64 of 4-bit codes: sign, two bits of exponent (bias 1), one of mantissa."""
    sign = 1 - 2 * (nibble >> 3).double()
    exponent, mantissa = (nibble >> 1) & 3, (nibble & 1).double()
    return sign * torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2.0 ** (exponent - 1))


def _exact_rows(codes, scales, columns):
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    factor = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)
    return (_value(both) * torch.where(scales.repeat_interleave(BLOCK, -1) == 255, float("nan"), factor))[..., :columns]


def _exact_quantize(s):
    x = s["x"]
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device="cuda")
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 24) // x.shape[1])
    for r in range(0, x.shape[0], step):
        b = x[r:r + step].double()
        b = torch.nn.functional.pad(b, (0, -b.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
        top = b.abs().amax(-1, keepdim=True)
        # the power of two at or below the largest magnitude, held to that by comparison
        power = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -200))))
        power = torch.where(power > top, power / 2, power)
        power = torch.where(2 * power <= top, 2 * power, power)
        unit = (power / 4).clamp_min(2.0 ** -127)
        v = b.abs() / unit
        above = torch.searchsorted(grid, v).clamp_max(7)  # the first magnitude that is not smaller
        below = (above - 1).clamp_min(0)
        up, down = grid[above] - v, v - grid[below]
        nearest = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
        value = torch.where(b < 0, -unit, unit) * grid[torch.where(v >= 6, 7, nearest)]
        out[r:r + step] = value.flatten(1)[:, :x.shape[1]]
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "quantize":
        return {"codes": None, "scales": None, "values": _exact_quantize(s)}
    if c["kind"] == "product":
        a, b = _exact_rows(*s["a"], c["k"]), _exact_rows(*s["b"], c["k"])
        return torch.matmul(a, b.T.contiguous())
    if c["kind"] == "experts":
        out = s["c"].double()
        rows, at = _exact_rows(*s["rows"], c["k"]), s["offsets"].tolist()
        for e in range(c["experts"]):
            if at[e] == at[e + 1]:
                continue
            p = torch.arange(at[e], at[e + 1], device="cuda")
            w = slice(e * c["n"], (e + 1) * c["n"])
            weight = _exact_rows(s["weights"][0][w], s["weights"][1][w], c["k"])
            y = rows[s["packed"][p].long().div(c["top_k"], rounding_mode="floor") if c["gather"] else p] @ weight.T.contiguous()
            if c["swiglu"]:
                half = c["n"] // 2
                y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
            out[p] = y
        return out
    tokens, top_k = c["tokens"], c["top_k"]
    # the routes that have an expert, by expert and then by their own number
    ids = _ids(seed, c)[0].flatten().tolist()
    route = sorted((i for i, e in enumerate(ids) if 0 <= e < c["experts"]), key=ids.__getitem__)
    kept, route = len(route), torch.tensor(route, dtype=torch.long, device="cuda")
    token = route // top_k
    weight = s["route_weights"].reshape(-1)[route].double().unsqueeze(1)
    step = 1 << 15
    if c["kind"] == "route":
        rows = s["packed_rows"].double()
        y = torch.zeros(tokens, c["width"], dtype=torch.float64, device="cuda")
        for p in range(0, kept, step):
            q = slice(p, min(kept, p + step))
            rows[q] = s["x"][token[q]].double()
            y.index_add_(0, token[q], weight[q] * s["expert_rows"][q].double())
        return {"offsets": None, "packed": None, "inverse": None, "packed_rows": rows, "y": y}
    d_rows = s["d_rows"].double()
    d_weights = torch.zeros(tokens * top_k, dtype=torch.float64, device="cuda")
    dx = torch.zeros(tokens, c["width"], dtype=torch.float64, device="cuda")
    for p in range(0, kept, step):
        q = slice(p, min(kept, p + step))
        dy = s["dy"][token[q]].double()
        d_rows[q] = weight[q] * dy
        d_weights[route[q]] = (dy * s["expert_rows"][q].double()).sum(1)
        dx.index_add_(0, token[q], s["d_packed"][q].double())
    return {"d_rows": d_rows, "d_weights": d_weights.view(tokens, top_k), "dx": dx}
