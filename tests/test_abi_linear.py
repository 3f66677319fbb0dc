"""Argument checks of the bf16 products with epilogues and gradients that need no
GPU: sizes, and every refusal before a device is touched."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

P = 0x100000  # a 16-byte aligned address that no refused call reads


def refused(q38m, name, *args):
    with pytest.raises(q38m.InvalidArgument):
        q38m.call(name, *args)


def maker(q38m):
    def tensor(rows=4, columns=8, dtype="bf16", data=P, stride=None, experts=1):
        return q38m.Tensor(data, columns if stride is None else stride,
                           {"bf16": q38m.DTYPE_BF16, "f32": q38m.DTYPE_F32}.get(dtype, dtype), experts, rows, columns)
    return tensor


def ref(t):
    return None if t is None else ctypes.byref(t)


def bad_tensors(q38m, rows, columns, dtype="bf16", **more):
    """Descriptors that no call takes in the place of a good one."""
    t = maker(q38m)
    size = 2 if dtype == "bf16" else 4
    return [t(rows, columns, dtype, data=None, **more), t(rows, columns, dtype, data=P + size // 2, **more),
            t(rows, columns, 0, **more), t(rows, columns, 3, **more), t(0, columns, dtype, **more),
            t(rows, 0, dtype, **more), t(rows, (1 << 24) + 1, dtype, **more), t((1 << 28) + 1, columns, dtype, **more),
            t(rows, columns, dtype, stride=columns - 1, **more), t(rows, columns, dtype, stride=(1 << 40) + 1, **more),
            t(rows + 1, columns, dtype, **more), t(rows, columns + 1, dtype, **more)]


def test_struct_and_scratch_sizes(q38m):
    assert ctypes.sizeof(q38m.Tensor) == 32
    size = q38m.lib().q38m_linear_scratch_bytes
    assert size(0, 8, 8) == size(8, 0, 8) == size(8, 8, 0) == 0
    assert size((1 << 28) + 1, 8, 8) == size(8, (1 << 24) + 1, 8) == size(8, 8, (1 << 24) + 1) == 0
    assert size(4, 8, 8) == 0  # one tile, one stage
    assert size(509, 2048, 8192) > 0
    for m, n, k in ((1, 8192, 2048), (61, 2048, 8192), (8192, 8192, 8192), (1 << 28, 1, 1), (1 << 20, 1 << 20, 64)):
        assert size(m, n, k) <= 1 << 34


def test_linear_refusals(q38m):
    t = maker(q38m)

    def call(x=t(4, 16), w=t(8, 16), bias=None, act=0, residual=None, y=t(4, 8), pre=None, scratch=P, nbytes=1 << 30):
        refused(q38m, "q38m_linear_v1", ref(x), ref(w), ref(bias), act, ref(residual), ref(y), ref(pre), scratch,
                nbytes, None, 0)

    for bad in [None, t(4, 16, "f32"), t(4, 17), t(2, 16, experts=2)] + bad_tensors(q38m, 4, 16)[:-2]:
        call(x=bad)
    for bad in [None, t(8, 16, "f32"), t(8, 15), t(4, 16, experts=2), t((1 << 24) + 1, 16)] + bad_tensors(q38m, 8, 16):
        call(w=bad)
    for bad in [None, t(4, 7), t(2, 8, experts=2)] + bad_tensors(q38m, 4, 8) + bad_tensors(q38m, 4, 8, "f32"):
        call(y=bad)
        if bad is not None:
            call(residual=bad)
            call(pre=bad)
    for bad in (t(1, 7), t(2, 8), t(1, 8, data=None), t(1, 8, data=P + 1), t(1, 8, "f32", data=P + 2), t(1, 8, 9)):
        call(bias=bad)
    call(act=6)
    call(residual=t(4, 8, "f32", data=P), y=t(4, 8))          # in place, another type
    call(residual=t(4, 8, stride=16), y=t(4, 8))              # in place, another stride
    # many inputs for few outputs: cut along K
    long = dict(x=t(509, 8192), w=t(2048, 8192), y=t(509, 2048))
    call(**long, scratch=None)
    call(**long, scratch=P + 8)
    call(**long, nbytes=0)
    call(x=t(1 << 28, 1 << 10), w=t(1 << 24, 1 << 10), y=t(1 << 28, 1 << 24))  # 2^31 tiles and more
    call(x=t(1 << 28, 1), w=t(256, 1), y=t(1 << 28, 256))  # odd rows: 2^24 tiles of 64 x 64


def test_input_gradient_refusals(q38m):
    t = maker(q38m)

    def call(dz=t(4, 8), w=t(8, 16), pre=None, act=0, residual=None, dx=t(4, 16), scratch=P, nbytes=1 << 30):
        refused(q38m, "q38m_linear_backward_input_v1", ref(dz), ref(w), ref(pre), act, ref(residual), ref(dx), scratch,
                nbytes, None, 0)

    for bad in [None, t(4, 8, "f32"), t(4, 7)] + bad_tensors(q38m, 4, 8)[:-2]:
        call(dz=bad)
    for bad in [None, t(8, 16, "f32")] + bad_tensors(q38m, 8, 16):
        call(w=bad)
    for bad in [None] + bad_tensors(q38m, 4, 16, "f32"):
        call(dx=bad)
        if bad is not None:
            call(pre=bad, act=2)
            call(residual=bad)
    call(act=2)  # an activation, and nothing that it was taken of
    call(act=6, pre=t(4, 16))
    call(residual=t(4, 16, "f32"), dx=t(4, 16))
    call(dz=t(1, 16384), w=t(16384, 64), dx=t(1, 64), scratch=None)


def test_weight_gradient_refusals(q38m):
    t = maker(q38m)

    def call(dz=t(4, 8), x=t(4, 16), residual=None, dw=t(8, 16), db=t(1, 8, "f32"), scratch=P, nbytes=1 << 30):
        refused(q38m, "q38m_linear_backward_weight_v1", ref(dz), ref(x), ref(residual), ref(dw), ref(db), scratch,
                nbytes, None, 0)

    for bad in [None, t(4, 8, "f32")] + bad_tensors(q38m, 4, 8):
        call(dz=bad)
    for bad in [None, t(4, 16, "f32")] + bad_tensors(q38m, 4, 16):
        call(x=bad)
    for bad in bad_tensors(q38m, 8, 16, "f32"):
        call(dw=bad)
        call(residual=bad)
    for bad in (t(1, 7), t(2, 8), t(1, 8, data=None), t(1, 8, "f32", data=P + 2)):
        call(db=bad)
    call(dw=None, db=None)
    call(dw=None, residual=t(8, 16))
    call(residual=t(8, 16, "f32"), dw=t(8, 16))
    many = dict(dz=t(16384, 8), x=t(16384, 16))
    call(**many, scratch=None)
    call(**many, dw=None, scratch=None)
    call(**many, dw=None, nbytes=8)


def test_activation_gradient_refusals(q38m):
    t = maker(q38m)

    def call(dy=t(4, 8), pre=t(4, 8), act=2, dz=t(4, 8)):
        refused(q38m, "q38m_linear_backward_activation_v1", ref(dy), ref(pre), act, ref(dz), None, 0)

    for bad in [None, t(2, 8, experts=2)] + bad_tensors(q38m, 4, 8):
        call(dy=bad)
        call(pre=bad)
        call(dz=bad)
    call(act=6)


def sorted_refusals(q38m, call, rows, routes):
    t = maker(q38m)
    call(offsets=None)
    call(offsets=P + 2)
    call(**rows(t(routes - 1, 16)))  # rows as they lie: one for each route
    call(**rows(t(routes // 2, 16, experts=2)))


def test_expert_product_refusals(q38m):
    t = maker(q38m)

    def call(w=t(8, 16, experts=3), rows=t(10, 16), offsets=P, packed=None, top_k=1, epilogue=0, c=t(10, 8), pre=None):
        refused(q38m, "q38m_moe_expert_gemm_v1", ref(w), ref(rows), offsets, packed, top_k, epilogue, ref(c), ref(pre),
                None, 0)

    sorted_refusals(q38m, call, lambda r: {"rows": r}, 10)
    for bad in [None, t(8, 16, "f32", experts=3), t(8, 15, experts=3), t(8, 16, experts=0), t(8, 16, experts=1025),
                t((1 << 24) + 1, 16, experts=3)]:
        call(w=bad)
    for bad in [None, t(10, 16, "f32"), t(10, 15)]:
        call(rows=bad)
    for bad in [None, t(10, 9), t(10, 4), t(5, 8, experts=2)] + bad_tensors(q38m, 10, 8)[:10]:
        call(c=bad)
    call(packed=P + 2)
    call(packed=P, top_k=0)
    call(epilogue=2)
    call(pre=t(10, 8))                                  # nothing to keep without the fold
    call(epilogue=1, c=t(10, 8))                        # eight rows: four gate, four up
    call(epilogue=1, c=t(10, 4), pre=t(10, 4))
    call(epilogue=1, w=t(7, 16, experts=3), c=t(10, 3))
    call(packed=P, c=t(1 << 24, 8))                     # 2^24 routes
    refused(q38m, "q38m_moe_expert_gemm_v1", None, None, None, None, 1, 0, None, None, None, 0)


def test_expert_row_gradient_refusals(q38m):
    t = maker(q38m)

    def call(w=t(8, 16, experts=3), dc=t(10, 8), offsets=P, pre=None, d=t(10, 16)):
        refused(q38m, "q38m_moe_expert_backward_rows_v1", ref(w), ref(dc), offsets, ref(pre), ref(d), None, 0)

    call(offsets=None)
    call(offsets=P + 1)
    for bad in [None, t(8, 16, "f32", experts=3), t(9, 16, experts=3), t(8, 16, experts=1025)]:
        call(w=bad)
    for bad in [None, t(10, 8, "f32"), t(10, 9), t(5, 8, experts=2)]:
        call(dc=bad)
    for bad in [None, t(10, 17), t(9, 16), t(10, 32)]:
        call(d=bad)
    call(pre=t(10, 32))                      # both halves' gradients want two halves
    call(pre=t(10, 16), d=t(10, 32))
    call(pre=t(10, 32), d=t(10, 16))
    call(dc=t(1 << 24, 8), d=t(1 << 24, 16))


def test_expert_weight_gradient_refusals(q38m):
    t = maker(q38m)

    def call(dc=t(10, 8), rows=t(10, 16), offsets=P, packed=None, top_k=1, residual=None, d=t(8, 16, experts=3)):
        refused(q38m, "q38m_moe_expert_backward_weights_v1", ref(dc), ref(rows), offsets, packed, top_k, ref(residual),
                ref(d), None, 0)

    sorted_refusals(q38m, call, lambda r: {"rows": r}, 10)
    for bad in [None, t(10, 8, "f32"), t(10, 9), t(5, 8, experts=2)]:
        call(dc=bad)
    for bad in [None, t(10, 16, "f32"), t(10, 17)]:
        call(rows=bad)
    for bad in [None, t(8, 17, experts=3), t(9, 16, experts=3), t(8, 16, experts=1025), t(8, 16, experts=0)]:
        call(d=bad)
    for bad in [t(8, 16), t(8, 16, experts=2), t(8, 17, experts=3), t(8, 16, "f32", experts=3)]:
        call(residual=bad)  # the last: in place, of another type
    call(packed=P, top_k=0)
    call(packed=P + 1)


def test_describe_refusals(q38m):
    """What the convenience would otherwise pass on as something else."""
    import torch as t

    x = t.zeros(6, 64, dtype=t.bfloat16)
    for bad in ((x.half(),), (x.double(),), (x.int(),), (x,), (x.view(2, 3, 2, 32),), (x[:0],)):
        with pytest.raises(q38m.InvalidArgument):
            q38m.describe(*bad)


def test_cpp_layer_of_the_guide(q38m, tmp_path):
    """The guide's training step in C++ compiles against the wrapper, links, and throws what the
    entry points refuse."""
    guide = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    begin = guide.index("```cpp\n", guide.index("## 8. bf16 experts")) + len("```cpp\n")
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
    TrainedExperts l{};
    refused([&] { forward(l, nullptr, nullptr, nullptr, 0); });
    refused([&] { backward(l, nullptr, nullptr, nullptr, nullptr, nullptr, 0); });
    q38m::TensorV1 t{};
    refused([&] { q38m::linear(t, t, nullptr, q38m::ActivationV1::kGelu, nullptr, t, nullptr, nullptr, 0, nullptr, 0); });
    refused([&] {
        q38m::linear_backward_input(t, t, nullptr, q38m::ActivationV1::kNone, nullptr, t, nullptr, 0, nullptr, 0);
    });
    refused([&] { q38m::linear_backward_weight(t, &t, nullptr, &t, nullptr, nullptr, 0, nullptr, 0); });
    refused([&] { q38m::linear_backward_activation(t, t, q38m::ActivationV1::kSilu, t, nullptr, 0); });
    std::printf("ok\n");
}
""")
    package = os.path.dirname(q38m.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(source),
                    "-o", str(tmp_path / "layer"), "-L", package, "-lq38m", f"-Wl,-rpath,{package}",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True)
    out = subprocess.run([str(tmp_path / "layer")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr
