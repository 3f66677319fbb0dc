"""The microscaled products on every tile shape, with scales in 16-byte pieces
(K of 450: padded to 512) and without (K of 129 and 300), each with rows and
columns that end inside a tile and with several tiles a workgroup, against the
plain 64-bit form.  The comments name the shape that the rule on sizes takes;
test_gpu_mx.py derives the bounds."""
import ctypes

import numpy as np
import pytest

from conftest import load_oracle
from helpers import device, host, stream, torch
from test_gpu_mx_layer import decode_rows, random_rows, spread
from test_gpu_mx import Encoded, check_product, close, encoded, product_bound, run_experts, want_experts, widen

load_oracle()
import mx_oracle as mx  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [
    (5, 17313, 129), (4, 16493, 450),                # 16 x 128
    (21, 17444, 129), (17, 17190, 450),              # 32 x 128
    (4149, 40, 129), (4402, 50, 450),                # 64 x 64
    (8290, 72, 129), (8340, 66, 450),                # 128 x 128
    (385, 25762, 450), (4000, 7900, 500)])          # 256 x 256: padded K of 512 and more alone
def test_product(q38m, m, n, k):
    print(f"product {m} x {n} x {k}", flush=True)
    rng = np.random.default_rng(m + n + k)
    check_product(q38m, Encoded(q38m, *encoded(rng, m, k), k), Encoded(q38m, *encoded(rng, n, k), k), k,
                  "bf16" if m % 2 else "f32", spare=3)


@pytest.mark.parametrize("swiglu,routes,experts,n,k", [
    (False, 8, 3, 34, 450), (True, 8, 3, 34, 450),               # 16 x 64
    (False, 200, 130, 66, 129), (False, 162, 130, 72, 450),      # 16 x 128
    (True, 149, 130, 66, 129), (True, 130, 130, 66, 500),
    (False, 3318, 130, 67, 129), (False, 3400, 130, 69, 450),    # 32 x 128
    (True, 3684, 130, 70, 129), (True, 3198, 130, 68, 450),
    (False, 4072, 7, 33, 300), (False, 4143, 3, 40, 450),        # 64 x 64
    (True, 4264, 3, 38, 129), (True, 4305, 3, 34, 450),
    (False, 13187, 130, 33, 129), (False, 17201, 12, 42, 450),   # 128 x 128
    (True, 16290, 7, 34, 129), (True, 12821, 130, 34, 450),
    (False, 594, 3, 16417, 450), (False, 15000, 5, 2048, 500),   # 256 x 256
    (True, 469, 3, 18958, 450), (True, 15000, 5, 2048, 500)])
def test_experts(q38m, swiglu, routes, experts, n, k):
    """Routes in part without an expert, experts without rows, gathered rows and rows in place."""
    print(f"experts {routes} of {experts}, {n} x {k} swiglu {swiglu}", flush=True)
    rng = np.random.default_rng(routes + n)
    ids = rng.integers(0, experts, size=(routes, 1)).astype(np.int32)
    ids[rng.random(ids.shape) < 0.03] = -1
    ids[ids == 1] = 2
    offsets, packed, _ = mx.sort_routes(ids, experts)
    kept = int(offsets[-1])
    w = Encoded(q38m, *encoded(rng, experts * n, k, 122, 126), k, experts)
    rows = Encoded(q38m, *encoded(rng, routes, k, 122, 126), k)
    for gather, dtype in ((True, "bf16"), (False, "f32")):
        words, got = run_experts(q38m, w, rows, device(offsets), device(packed) if gather else None, 1, routes,
                                 swiglu, dtype)
        want, bound = want_experts(w.values, rows.values, offsets, packed, 1 if gather else 0, experts, k, swiglu)
        assert (words[kept:] == 0x4a4a).all(), "a dropped route's row was written"
        close(got[:kept], want[:kept], bound[:kept], dtype, (routes, experts, n, k, gather))


@pytest.mark.parametrize("m,n,k", [(5, 70, 1024), (300, 530, 512), (4000, 4000, 512)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_least_alignment(q38m, m, n, k, dtype):
    """Scales 4 bytes and C one element behind a 16-byte boundary, rows of C an odd stride apart."""
    t = torch()
    print(f"alignment {m} x {n} x {k} {dtype}", flush=True)
    rng = np.random.default_rng(m)
    sides = []
    for rows in (m, n):
        codes, scales = encoded(rng, rows, k)
        on_device, shifted = device(codes), t.zeros(scales.size + 4, dtype=t.uint8, device="cuda")
        shifted[4:] = device(scales).reshape(-1)
        sides.append((q38m.MxMatrix(on_device.data_ptr(), shifted.data_ptr() + 4, 1, rows, k), on_device, shifted,
                      mx.decode(codes, scales, k)))
    stride = n + 1 + n % 2
    out = t.full((1 + m * stride + 8,), 0x4a4a, dtype=t.int16 if dtype == "bf16" else t.int32, device="cuda")
    c = out.data_ptr() + out.element_size()
    q38m.call("q38m_mx_gemm_v1", ctypes.byref(sides[0][0]), ctypes.byref(sides[1][0]),
              *((None, c) if dtype == "bf16" else (c, None)), stride, stream(), 0)
    t.cuda.synchronize()
    words = host(out, np.uint16 if dtype == "bf16" else np.uint32)
    assert words[0] == 0x4a4a and (words[1 + m * stride:] == 0x4a4a).all()
    words = words[1:1 + m * stride].reshape(m, stride)
    assert (words[:, n:] == 0x4a4a).all()
    words = np.ascontiguousarray(words[:, :n])
    got = widen(words) if dtype == "bf16" else words.view(np.float32).astype(np.float64)
    want, size = mx.product(sides[0][3], sides[1][3])
    close(got, want, product_bound(k, size), dtype, (m, n, k))


@pytest.mark.parametrize("swiglu,routes,experts,n,k,kind", [
    (False, 1396, 1024, 186, 4096, "even"), (True, 1100, 1024, 132, 4096, "even"),           # 16 x 64
    (False, 600, 512, 1100, 2048, "even"), (True, 600, 512, 1100, 2048, "even"),             # 16 x 128
    (False, 4000, 512, 1100, 2048, "skewed"), (True, 4000, 512, 1100, 2048, "skewed"),
    (False, 9000, 512, 1100, 2048, "skewed"), (True, 9000, 512, 1100, 2048, "skewed"),       # 32 x 128
    (True, 530, 40, 3594, 4096, "skewed")])
def test_weights_past_the_caches(q38m, swiglu, routes, experts, n, k, kind):
    """Weights of more than 256 MB: experts of one row tile and of several, compared at rows and
    columns spread over the whole."""
    t = torch()
    print(f"past the caches {routes} of {experts}, {n} x {k} {kind} swiglu {swiglu}", flush=True)
    rng = np.random.default_rng(routes + n)
    ids = rng.integers(0, experts, size=(routes, 1)).astype(np.int32)
    if kind == "skewed":
        ids[rng.random(ids.shape) < 0.3] //= 64
    offsets, packed, _ = mx.sort_routes(ids, experts)
    w, rows = (random_rows(q38m, e, m, k, 122, 124) for e, m in ((experts, n), (1, routes)))
    columns = n // 2 if swiglu else n
    at, order = device(offsets), device(packed)
    c = t.empty(routes, columns, dtype=t.float32, device="cuda")
    q38m.call("q38m_mx_grouped_gemm_v1", ctypes.byref(w.desc), ctypes.byref(rows.desc), at.data_ptr(),
              order.data_ptr(), 1, routes, q38m.MX_EPILOGUE_SWIGLU if swiglu else q38m.MX_EPILOGUE_NONE,
              c.data_ptr(), None, stream(), 0)
    places, some = spread(routes, 60), spread(columns, 50)
    got = c[t.as_tensor(places, device="cuda")][:, t.as_tensor(some, device="cuda")].cpu().numpy().astype(np.float64)
    a = decode_rows(rows, packed[places].astype(np.int64), k)
    picked = np.concatenate((some, columns + some)) if swiglu else some
    for i, p in enumerate(places):
        expert = int(ids[packed[p], 0])
        want, bound = want_experts(decode_rows(w, expert * n + picked, k), a[i:i + 1], np.array([0, 1]),
                                   np.zeros(1, np.int64), 0, 1, k, swiglu)
        close(got[i:i + 1], want, bound, "f32", (p, expert))
