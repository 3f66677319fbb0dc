"""The built libraries' device code keeps the waits that gfx950 leaves to the
program.  The compiler inserts them for its own instructions; it does not look
into inline assembly, where the products' loads to LDS are."""
import os
import re

import pytest

import device_code as dc
from conftest import PACKAGE_DIR

LISTING = """
0000000000000100 <kernel>:
\tv_readfirstlane_b32 s4, v0        // 000000000100: 7E080500
\tv_readfirstlane_b32 s5, v1        // 000000000104: 7E0A0501
\ts_mov_b32 m0, s9                  // 000000000108: BEFC0009
\ts_nop {0}                         // 00000000010C: BF800000
\tglobal_load_lds_dwordx4 v3, s[4:5] // 000000000110: DDF48000 00040003
\ts_cbranch_scc1 65531               // 000000000118: BF85FFFB <kernel+0x8>
\ts_endpgm                          // 00000000011C: BF810000
"""


def scalar_m0(i):
    return {"m0"} if i.name.startswith("s_") and i.operands[0] == "m0" else set()


def lds_load(i):
    return {"m0"} if "_lds_" in i.name and i.name.startswith(("global", "buffer")) else set()


@pytest.mark.parametrize("nop,soon", [(0, ["s4", "s5"]), (2, ["s5"]), (3, [])])
def test_the_check_counts(nop, soon):
    """Wait states between the reads of lanes and the load: 1 + (nop + 1), one more for s4."""
    found = dc.too_soon(dc.parse(LISTING.format(nop)), dc.memory_reads, dc.vector_writes, 5)
    assert sorted(w.operands[0] for w, _ in found) == soon


def test_the_check_follows_branches():
    """The branch back to 0x108 leaves a write at 0x114 three wait states in front of the load."""
    text = LISTING.format(0).replace("\ts_cbranch", "\tv_readlane_b32 s4, v9, 0 // 000000000114: D289\n\ts_cbranch")
    found = dc.too_soon(dc.parse(text), dc.memory_reads, dc.vector_writes, 5)
    assert 0x114 in {w.address for w, _ in found}


@pytest.fixture(scope="module", params=["product", "checked"])
def objects(q38m, request, tmp_path_factory):
    library = q38m.LIB_PATH if request.param == "product" else q38m.CHECKED_LIB_PATH
    found = dc.code_objects(library, tmp_path_factory.mktemp("code"))
    assert len(found) >= 11  # one for each source
    return [(o, dc.disassemble(o)) for o in found]


def test_scalar_operands_of_memory_instructions_have_settled(objects):
    """A scalar register that a vector instruction writes is read by a vector memory instruction
    no earlier than five wait states later, m0 by a load to LDS one after a scalar write: the
    hardware does not hold these back."""
    loads = 0
    for _, code in objects:
        loads += sum(bool(lds_load(i)) for i in code)
        for reads, writes, states in ((dc.memory_reads, dc.vector_writes, 5), (lds_load, scalar_m0, 1)):
            found = dc.too_soon(code, reads, writes, states)
            assert not found, [(w.kernel, hex(w.address), w.name, w.operands, hex(r.address), r.name, r.operands)
                               for w, r in found[:3]] + [len(found)]
    assert loads > 500  # the listing shows them


def test_m0_belongs_to_the_loads(objects):
    """Every load to LDS has its own write of m0 right in front, and nothing else reads m0: no
    value that the compiler keeps there is lost."""
    for _, code in objects:
        for k, i in enumerate(code):
            if lds_load(i):
                setting = next(p for p in reversed(code[:k]) if p.name != "s_nop")
                assert scalar_m0(setting), (i.kernel, hex(i.address))
            else:
                reads = i.operands[1:] if scalar_m0(i) else i.operands
                assert not any("m0" in dc.scalar_registers(o) for o in reads), (i.kernel, hex(i.address), i.name)


def assembly_statements():
    """(file, statement) of every inline assembly."""
    folder = os.path.join(PACKAGE_DIR, "csrc")
    for name in sorted(os.listdir(folder)):
        text = open(os.path.join(folder, name)).read()
        for start in (m.start() for m in re.finditer(r"\basm\b(?: volatile)?\(", text)):
            depth, end = 0, text.index("(", start)
            while True:
                depth += {"(": 1, ")": -1}.get(text[end], 0)
                end += 1
                if depth == 0:
                    break
            yield name, text[start:end]


@pytest.mark.parametrize("writes,register,least", [("s_mov_b32 m0", "m0", 2), ("s_bcnt1_i32", "scc", 3)])
def test_inline_assembly_names_what_it_writes(writes, register, least):
    """m0 and the scalar condition bit are among the clobbers of every statement that sets them."""
    found = [(name, text) for name, text in assembly_statements() if writes in text]
    assert len(found) >= least
    for name, text in found:
        assert f'"{register}"' in text, (name, text)


def test_product_kernels_keep_their_registers(objects):
    """No microscaled kernel keeps a vector register in memory: 256 x 256 tiles have none to
    spare, and a compiler that spills there would put memory into the innermost loop."""
    kernels = {name: r for path, _ in objects for name, r in dc.resources(path).items() if "mx_" in name}
    assert len([name for name in kernels if "mx_tile_kernel" in name]) >= 36
    for name, r in kernels.items():
        assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (name, r)
