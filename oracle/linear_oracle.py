"""Plain 64-bit forms of the bf16 products with epilogues and of their gradients,
on torch float64 tensors (any device)."""
import math

import torch

ACTIVATIONS = ("none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh")


def activation(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    s = torch.sigmoid(2 * _t(z) if name == "gelu_tanh" else z)
    return s if name == "sigmoid" else z * s


def _t(z):
    return math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)


def slope(name, z):
    """The derivative; of relu 0 at 0."""
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        s = torch.sigmoid(2 * _t(z))
        return s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s * (1 - s) if name == "sigmoid" else s * (1 + z * (1 - s))


def linear(x, w, bias=None, act="none", residual=None):
    """(y, pre)"""
    z = x @ w.T
    if bias is not None:
        z = z + bias
    y = activation(act, z)
    return (y if residual is None else y + residual), z


def swiglu(gate_up):
    gate, up = gate_up.chunk(2, -1)
    return gate * torch.sigmoid(gate) * up


def swiglu_backward(gate_up, dh):
    gate, up = gate_up.chunk(2, -1)
    return torch.cat((dh * up * slope("silu", gate), dh * activation("silu", gate)), -1)


def expert_rows(offsets, routes):
    """[(expert, first, end)] of the experts that have rows, from a list of offsets."""
    held = [min(o, routes) for o in offsets]
    return [(e, a, b) for e, (a, b) in enumerate(zip(held, held[1:])) if b > a]


def experts(rows, weights, offsets, routes, source=None):
    """[routes][n] products, NaN where no expert has the row; source: row of each place."""
    out = torch.full((routes, weights.shape[1]), float("nan"), dtype=rows.dtype, device=rows.device)
    for e, a, b in expert_rows(offsets, routes):
        out[a:b] = (rows[a:b] if source is None else rows[source[a:b]]) @ weights[e].T
    return out


def experts_backward_rows(dc, weights, offsets):
    out = torch.full((dc.shape[0], weights.shape[2]), float("nan"), dtype=dc.dtype, device=dc.device)
    for e, a, b in expert_rows(offsets, dc.shape[0]):
        out[a:b] = dc[a:b] @ weights[e]
    return out


def experts_backward_weights(dc, rows, offsets, count, source=None):
    out = torch.zeros(count, dc.shape[1], rows.shape[1], dtype=dc.dtype, device=dc.device)
    for e, a, b in expert_rows(offsets, dc.shape[0]):
        out[e] = dc[a:b].T @ (rows[a:b] if source is None else rows[source[a:b]])
    return out
