"""The list of the experts' row tiles reads their offsets 16 bytes at a time, so it takes
words of 16 bytes alone: an array of 32-bit numbers, which LDS may hold at any four
bytes, does not compile."""
import os
import subprocess

import pytest

from conftest import PACKAGE_DIR, ROOT

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

SOURCE = """
#include <type_traits>
#include "q38m_product.h"
using namespace q38m;
static_assert(std::is_constructible_v<TileList<16>, %s, uint32_t, uint32_t>);
static_assert(alignof(v4i) == 16);
"""


@pytest.mark.parametrize("pointer,taken", [("const v4i*", True), ("v4i*", True), ("const uint32_t*", False),
                                           ("uint32_t*", False), ("const int32_t*", False)])
def test_offsets_are_words_of_16_bytes(pointer, taken, tmp_path):
    source = tmp_path / "list.hip"
    source.write_text(SOURCE % pointer)
    out = subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-device-only", "-std=c++17", "-fsyntax-only",
                          "-Wno-unused-function", "-I", os.path.join(PACKAGE_DIR, "csrc"), "-I",
                          os.path.join(ROOT, "include"), str(source)], capture_output=True, text=True)
    assert (out.returncode == 0) == taken, out.stderr
    assert taken or "static assertion failed" in out.stderr, out.stderr
