"""Plain 64-bit forms of the microscaled 4-bit rows, their products and the
sort of tokens by expert with the way back and its gradients: the tests'
oracle, written from the definitions in include/q38m.h with numpy alone.

  block   32 consecutive values of a row, largest magnitude m
  scale   byte s = max(floor(log2 m) - 2, -127) + 127, 0 for m = 0, 255 where a
          value of the block is not finite
  code    sign bit and the index of |x| 2^(127 - s) rounded half to even among
          {0, .5, 1, 1.5, 2, 3, 4, 6}, 7 above
"""
import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
DROPPED = 0xffffffff


def padded(columns):
    return -(-columns // 128) * 128


def quantize(x):
    """x [rows][columns] (any real type) -> codes uint8 [rows][padded / 2],
    scales uint8 [rows][padded / 32], values float64 [rows][columns]."""
    x = np.asarray(x, dtype=np.float64)
    rows, columns = x.shape
    full = np.zeros((rows, padded(columns)))
    full[:, :columns] = x
    blocks = full.reshape(rows, -1, 32)
    finite = np.isfinite(blocks).all(-1)
    clean = np.where(finite[..., None], blocks, 0.0)
    top = np.abs(clean).max(-1)
    # frexp: m = f 2^e with f in [.5, 1), so floor(log2 m) = e - 1
    exponent = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1, -1000)
    scale = np.where(finite, np.maximum(exponent - 2, -127) + 127, 255)
    unit = np.where(finite, np.ldexp(1.0, np.minimum(scale, 254) - 127), 1.0)
    v = np.abs(clean) / unit[..., None]
    # nearest of the eight magnitudes; the even index on a tie
    up = np.minimum(np.searchsorted(MAGNITUDES, v), 7)
    down = np.maximum(up - 1, 0)
    above, below = MAGNITUDES[up] - v, v - MAGNITUDES[down]
    index = np.where((above < below) | ((above == below) & (up % 2 == 0)), up, down)
    index = np.where(v >= 6, 7, index)
    code = (index | np.signbit(clean) * 8).astype(np.uint8).reshape(rows, -1)
    values = np.where(np.signbit(clean), -1.0, 1.0) * MAGNITUDES[index] * unit[..., None]
    values = np.where(finite[..., None], values, np.nan).reshape(rows, -1)[:, :columns]
    return code[:, 0::2] | code[:, 1::2] << 4, scale.astype(np.uint8), values


def decode(codes, scales, columns):
    """float64 [rows][columns] of encoded rows."""
    codes, scales = np.asarray(codes, np.uint8), np.asarray(scales, np.uint8)
    both = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
    value = np.where(both & 8, -1.0, 1.0) * MAGNITUDES[both & 7]
    factor = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (value * np.repeat(factor, 32, axis=1))[:, :columns]


def product(a, b):
    """(A B^T, |A| |B|^T) of float64 rows: the product and the sum of its
    terms' magnitudes, which bounds its rounding."""
    return a @ b.T, np.abs(a) @ np.abs(b).T


def swiglu(gate, up):
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up


def sort_routes(ids, experts):
    """offsets [experts + 1], packed [routes], inverse [routes] (uint32)."""
    flat = np.asarray(ids).reshape(-1)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    packed = np.argsort(key, kind="stable").astype(np.uint32)
    offsets = np.searchsorted(key[packed], np.arange(experts + 1)).astype(np.uint32)
    inverse = np.full(flat.size, DROPPED, dtype=np.uint32)
    kept = int(offsets[-1])
    inverse[packed[:kept]] = np.arange(kept, dtype=np.uint32)
    return offsets, packed, inverse


def unpermute(rows, inverse, weights, tokens):
    """(y, sum of the terms' magnitudes), float64 [tokens][width]; weights
    None: ones."""
    rows = np.asarray(rows, np.float64)
    inverse = np.asarray(inverse).reshape(tokens, -1)
    y = np.zeros((tokens, rows.shape[1]))
    size = np.zeros_like(y)
    for rank in range(inverse.shape[1]):
        at = inverse[:, rank]
        t = np.nonzero(at < inverse.size)[0]
        term = rows[at[t]]
        if weights is not None:
            term = term * np.asarray(weights, np.float64).reshape(tokens, -1)[t, rank, None]
        y[t] += term
        size[t] += np.abs(term)
    return y, size


def unpermute_backward(dy, rows, inverse, weights):
    """(d_rows, d_weights, sum of the magnitudes of d_weights' terms); d_rows
    is nan where no route writes."""
    dy, rows = np.asarray(dy, np.float64), np.asarray(rows, np.float64)
    tokens = dy.shape[0]
    inverse = np.asarray(inverse).reshape(tokens, -1)
    weights = np.asarray(weights, np.float64).reshape(tokens, -1)
    d_rows = np.full(rows.shape, np.nan)
    d_weights = np.zeros(weights.shape)
    size = np.zeros(weights.shape)
    for rank in range(inverse.shape[1]):
        at = inverse[:, rank]
        t = np.nonzero(at < inverse.size)[0]
        d_rows[at[t]] = weights[t, rank, None] * dy[t]
        d_weights[t, rank] = (dy[t] * rows[at[t]]).sum(1)
        size[t, rank] = np.abs(dy[t] * rows[at[t]]).sum(1)
    return d_rows, d_weights, size
