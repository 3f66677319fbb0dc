"""Argument checks of the microscaled products and the sorted-token entry
points that need no GPU: sizes, and every refusal before a device is
touched."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

P = 0x100000  # a 16-byte aligned address that no refused call reads


def matrix(q38m, experts=1, rows=4, columns=256, codes=P, scales=P, reserved=0):
    return q38m.MxMatrix(codes, scales, experts, rows, columns, reserved)


def refused(q38m, name, *args):
    with pytest.raises(q38m.InvalidArgument):
        q38m.call(name, *args)


def test_row_sizes(q38m):
    lib = q38m.lib()
    for columns, row, scale in ((1, 64, 4), (128, 64, 4), (129, 128, 8), (2048, 1024, 64)):
        assert lib.q38m_mx_row_bytes(columns) == row
        assert lib.q38m_mx_scale_bytes(columns) == scale
    assert ctypes.sizeof(q38m.MxMatrix) == 32


def test_quantize_refusals(q38m):
    def call(x=P, dtype=q38m.DTYPE_BF16, stride=256, rounded=None, **m):
        refused(q38m, "q38m_mx_quantize_v1", x, dtype, stride,
                ctypes.byref(matrix(q38m, **m)), rounded, None, 0)

    call(x=None)
    call(x=P + 1)
    call(dtype=q38m.DTYPE_F32, x=P + 2)
    call(dtype=0)
    call(dtype=3)
    call(stride=255)
    call(rounded=P + 1)
    call(codes=None)
    call(scales=None)
    call(codes=P + 8)
    call(scales=P + 2)
    call(experts=0)
    call(rows=0)
    call(columns=0)
    call(columns=(1 << 24) + 1, stride=1 << 30)
    call(rows=(1 << 23) + 1)
    call(experts=1 << 12, rows=1 << 12)
    call(reserved=1)
    refused(q38m, "q38m_mx_quantize_v1", P, q38m.DTYPE_BF16, 256, None, None, None, 0)


def test_product_refusals(q38m):
    def call(a=None, b=None, f32=P, bf16=None, stride=4):
        refused(q38m, "q38m_mx_gemm_v1", ctypes.byref(a or matrix(q38m)),
                ctypes.byref(b or matrix(q38m)), f32, bf16, stride, None, 0)

    call(a=matrix(q38m, columns=128))
    call(a=matrix(q38m, experts=2))
    call(b=matrix(q38m, experts=2))
    call(f32=None)
    call(bf16=P)
    call(f32=P + 2)
    call(f32=None, bf16=P + 1)
    call(stride=3)
    call(a=matrix(q38m, rows=0xffffffff), b=matrix(q38m, rows=0xffffffff), stride=1 << 32)
    refused(q38m, "q38m_mx_gemm_v1", None, ctypes.byref(matrix(q38m)), P, None, 4, None, 0)


def test_grouped_refusals(q38m):
    def call(w=None, rows=None, offsets=P, packed=P, top_k=2, routes=8, epilogue=0, f32=P,
             bf16=None):
        refused(q38m, "q38m_mx_grouped_gemm_v1", ctypes.byref(w or matrix(q38m, experts=3)),
                ctypes.byref(rows or matrix(q38m)), offsets, packed, top_k, routes, epilogue,
                f32, bf16, None, 0)

    call(offsets=None)
    call(top_k=0)
    call(routes=0)
    call(routes=1 << 24)
    call(packed=None, routes=8)  # four rows for eight routes
    call(epilogue=2)
    call(w=matrix(q38m, experts=3, rows=5), epilogue=q38m.MX_EPILOGUE_SWIGLU)
    call(w=matrix(q38m, experts=1025))
    call(rows=matrix(q38m, experts=2))
    call(rows=matrix(q38m, columns=384))
    call(f32=None)
    call(bf16=P)
    call(f32=P + 1)
    call(offsets=P + 2)
    call(packed=P + 1)
    # gathered rows, or one expert's, of 4 GB and more
    call(w=matrix(q38m, experts=3, columns=2048), rows=matrix(q38m, rows=1 << 22, columns=2048))
    call(w=matrix(q38m, experts=3, rows=1 << 22, columns=2048), rows=matrix(q38m, columns=2048),
         epilogue=q38m.MX_EPILOGUE_SWIGLU)


def test_sort_refusals(q38m):
    size = q38m.lib().q38m_moe_sort_scratch_bytes
    assert size(1, 10, 512) == 0
    assert size(0, 10, 512) == 0 and size(4, 10, 0) == 0 and size(4, 10, 1025) == 0
    assert size(32768, 10, 512) > 0 and size(1 << 20, 16, 512) == 0  # 2^24 routes: refused

    def call(ids=P, tokens=32768, top_k=10, experts=512, offsets=P, packed=P, inverse=P,
             scratch=P, nbytes=1 << 30):
        refused(q38m, "q38m_moe_sort_routes_v1", ids, tokens, top_k, experts, offsets, packed,
                inverse, scratch, nbytes, None, 0)

    call(ids=None)
    call(offsets=None)
    call(packed=None)
    call(inverse=None)
    call(tokens=0)
    call(top_k=0)
    call(tokens=1 << 20, top_k=16)
    call(tokens=1 << 31, top_k=1 << 31)
    call(experts=0)
    call(experts=1025)
    call(scratch=None)
    call(scratch=P + 2)
    call(ids=P + 2)
    call(offsets=P + 1)
    call(packed=P + 2)
    call(inverse=P + 3)
    call(nbytes=size(32768, 10, 512) - 1)


def test_row_refusals(q38m):
    bf16, f32 = q38m.DTYPE_BF16, q38m.DTYPE_F32
    for bad in (dict(x=None), dict(x=P + 1), dict(x=P + 2, dtype=f32), dict(inverse=None),
                dict(inverse=P + 2), dict(rows=None), dict(rows=P + 1), dict(dtype=7), dict(tokens=0), dict(top_k=0),
                dict(tokens=1 << 24, top_k=1), dict(width=0), dict(width=(1 << 24) + 1)):
        a = dict(x=P, dtype=bf16, inverse=P, tokens=4, top_k=2, width=8, rows=P)
        a.update(bad)
        refused(q38m, "q38m_moe_permute_rows_v1", a["x"], a["dtype"], a["inverse"], a["tokens"],
                a["top_k"], a["width"], a["rows"], None, 0)
        refused(q38m, "q38m_moe_unpermute_rows_v1", a["x"], a["dtype"], a["inverse"], P,
                a["tokens"], a["top_k"], a["width"], a["rows"], None, 0)
        refused(q38m, "q38m_moe_unpermute_backward_v1", a["x"], P, a["dtype"], a["inverse"], P,
                a["tokens"], a["top_k"], a["width"], a["rows"] or P + 1, P, None, 0)
    refused(q38m, "q38m_moe_unpermute_rows_v1", P, bf16, P, P + 2, 4, 2, 8, P, None, 0)

    def backward(rows=P, weights=P, d_rows=P, d_weights=P):
        refused(q38m, "q38m_moe_unpermute_backward_v1", P, rows, bf16, P, weights, 4, 2, 8,
                d_rows, d_weights, None, 0)

    backward(weights=None)
    backward(weights=P + 2)
    backward(d_rows=None, d_weights=None)
    backward(rows=None)
    backward(rows=P + 1)
    backward(d_weights=P + 2)


def test_python_refusals(q38m):
    """What the conveniences would otherwise pass on as something else: other types, columns
    apart, unequal experts, host memory."""
    import torch as t

    x = t.zeros(6, 64, dtype=t.bfloat16)
    for bad in ((x.half(),), (x.double(),), (x.int(),), (x[0],), (x.T,), (x[:, ::2],), (x, 4),
                (x, 0), (x, 1, x.float()), (x, 1, x[:3]), (x, 1, x.T.contiguous().T), (x,)):
        with pytest.raises(q38m.InvalidArgument):
            q38m.mx_quantize(*bad)
    routes = q38m.SortedRoutes(6, 4, 8, device="cpu")
    ids = t.zeros(6, 4, dtype=t.int32)
    for bad in (ids.long(), ids.short(), ids[:5], ids.T.contiguous().T, ids.reshape(4, 6), ids):
        with pytest.raises(q38m.InvalidArgument):
            routes.sort(bad)


def test_cpp_layer_of_the_guide(q38m, tmp_path):
    """The guide's layer in C++ compiles against the wrapper, links, and throws what the entry
    points refuse."""
    guide = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    begin = guide.index("```cpp\n", guide.index("## 7. Microscaled experts")) + len("```cpp\n")
    source = tmp_path / "layer.cpp"
    source.write_text(guide[begin:guide.index("```\n", begin)] + r"""
#include <cstdio>
#include <stdexcept>
template <typename F>
void refused(F f) {
    try {
        f();
    } catch (const std::invalid_argument&) {
        return;
    }
    std::printf("accepted\n");
}
int main() {
    MxLayer l{};
    refused([&] { run_mx_layer(l, nullptr, nullptr, nullptr, nullptr, nullptr, 0); });
    refused([&] { q38m::mx_quantize(&l, q38m::DtypeV1::kF32, 0, l.x_rows, nullptr, nullptr, 0); });
    refused([&] { q38m::mx_gemm(l.x_rows, l.h_rows, nullptr, nullptr, 0, nullptr, 0); });
    refused([&] { q38m::moe_permute_rows(&l, q38m::DtypeV1::kBf16, nullptr, 1, 1, 8, &l, nullptr, 0); });
    refused([&] {
        q38m::moe_unpermute_backward(&l, &l, q38m::DtypeV1::kBf16, nullptr, nullptr, 1, 1, 8, &l, nullptr,
                                     nullptr, 0);
    });
    std::printf("ok\n");
}
""")
    package = os.path.dirname(q38m.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(source),
                    "-o", str(tmp_path / "layer"), "-L", package, "-lq38m", f"-Wl,-rpath,{package}",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True)
    out = subprocess.run([str(tmp_path / "layer")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr
