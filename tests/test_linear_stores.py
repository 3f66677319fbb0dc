"""Which of the bf16 products' kernels go past the caches: those of whole lines of dense rows
come in two forms, and the one for rows that stay has no load and no store that does."""
import os
import re
import subprocess

import device_code as dc

DENSE_ROWS = re.compile(r"linear_tile_kernelINS_11LinearShapeILj32E\w*?LinearOrderE[01]ELb0ELNS_10LinearFoldE[01]ELb([01])E")


def test_rows_that_stay_use_the_caches(q38m, tmp_path):
    seen = {"0": 0, "1": 0}
    for path in dc.code_objects(q38m.LIB_PATH, tmp_path):
        names = [n for n in dc.resources(path) if DENSE_ROWS.search(n)]
        if not names:
            continue
        listing = subprocess.run([os.path.join(dc.LLVM, "llvm-objdump"), "-d", "--mcpu=gfx950",
                                  "--disassemble-symbols=" + ",".join(names), path], check=True, capture_output=True,
                                 text=True).stdout
        code = dc.parse(listing)
        for name in names:
            past = DENSE_ROWS.search(name).group(1)
            wide = [i for i in code if i.kernel == name and re.match(r"global_(load|store)_dwordx4", i.name)]
            streamed = [i for i in wide if any(re.search(r"\bnt\b", o) for o in i.operands)]
            assert wide and bool(streamed) == (past == "1"), (name, len(wide), len(streamed))
            seen[past] += 1
    assert seen == {"0": 8, "1": 8}  # two tile shapes, two orders, with a residual and without
