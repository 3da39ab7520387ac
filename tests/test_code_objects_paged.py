"""The gfx950 code of the paged cache's kernels in the built library: the loop of paged_tiles_kernel's first pass touches no scratch
memory (its second pass, which shares the kernel's registers and hardly ever runs, does), the other kernels nowhere."""
import os
import re
import subprocess

import pytest

from test_code_objects import LIB, LLVM, basic_blocks, code_objects


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(LIB) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("needs the built library and llvm-objdump")
    out = {}
    for i, co in enumerate(code_objects(LIB)):
        if b"paged_" not in co:
            continue
        path = tmp_path_factory.mktemp("co") / f"{i}.elf"
        path.write_bytes(co)
        dump = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", "--demangle", str(path)],
                              capture_output=True, text=True, check=True).stdout
        name = None
        for l in dump.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:$", l)
            if m:
                found = re.search(r"paged_[a-z]+_kernel<[^>]*>", m[1])
                name = found[0] if found else None
                if name:
                    out[name] = []
            elif name:
                out[name].append(l)
    return out


def test_no_scratch_in_the_first_pass_of_the_tiles(kernels):
    """Its loop is the first of the blocks with the most MFMAs: a phase of O += P V and S = K Q^T."""
    tiles = {n: lines for n, lines in kernels.items() if n.startswith("paged_tiles")}
    assert len(tiles) == 4, sorted(tiles)
    for name, lines in tiles.items():
        blocks = list(basic_blocks(lines))
        mfmas = [sum("v_mfma" in x for x in b) for b in blocks]
        assert max(mfmas) == (64 if "128" in name else 32), (name, max(mfmas))
        main = blocks[mfmas.index(max(mfmas))]
        assert not [x for x in main if x.startswith("scratch_")], name


def test_no_scratch_in_the_others(kernels):
    others = {n: lines for n, lines in kernels.items() if not n.startswith("paged_tiles")}
    assert sum(n.startswith("paged_rows") for n in others) == 6 and sum(n.startswith("paged_join") for n in others) == 4
    assert sum(n.startswith("paged_append") for n in others) == 16 and sum(n.startswith("paged_read") for n in others) == 8
    for name, lines in others.items():
        assert not [l for l in lines if re.match(r"\s+scratch_", l)], name
