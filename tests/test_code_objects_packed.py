"""The gfx950 code of the packed sequences' kernels in the built library: no scratch memory in the loops (a reload there waits for the
tiles on their way too) but those of the attention's second pass, which hardly ever runs; none at all in the small kernels."""
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
        if b"packed_" not in co and b"rope_tokens" not in co:
            continue
        path = tmp_path_factory.mktemp("co") / f"{i}.elf"
        path.write_bytes(co)
        dump = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", "--demangle", str(path)],
                              capture_output=True, text=True, check=True).stdout
        name = None
        for l in dump.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:$", l)
            if m:
                found = re.search(r"(?:packed_[a-z]+|rope_tokens)_kernel<[^>]*>", m[1])
                name = found[0] if found else None
                if name:
                    out[name] = []
            elif name:
                out[name].append(l)
    return out


def mfmas(block):
    return sum("v_mfma" in x for x in block)


def test_no_scratch_in_the_loops(kernels):
    for d in (64, 128):
        blocks = list(basic_blocks(kernels[f"packed_attn_kernel<{d}>"]))
        most = max(map(mfmas, blocks))
        assert most == d // 2, most                 # a phase: O += P V and S = K Q^T
        main = next(b for b in blocks if mfmas(b) == most)
        assert not [x for x in main if x.startswith("scratch_")]
        blocks = list(basic_blocks(kernels[f"packed_back_kernel<{d}>"]))
        assert sum(map(mfmas, blocks)) == d // 2 + 3 * d // 4   # four products over 32 rows and 32 keys, three over 32 rows and 64 keys
        for b in blocks:
            assert not (mfmas(b) and [x for x in b if x.startswith("scratch_")])


def test_no_scratch_in_the_others(kernels):
    others = {n: lines for n, lines in kernels.items() if not n.startswith(("packed_attn", "packed_back"))}
    assert sum(n.startswith("rope_tokens") for n in others) == 8 and sum(n.startswith("packed_stats") for n in others) == 16
    assert sum(n.startswith("packed_join") for n in others) == 2 and sum(n.startswith("packed_sum") for n in others) == 2
    for name, lines in others.items():
        assert not [l for l in lines if re.match(r"\s+scratch_", l)], name
