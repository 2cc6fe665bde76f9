"""A fault that the compiler has made in kernels that need all registers: behind a branch that lanes take differently, copies between vector and accumulation
registers (or memory of spilled ones) in front of the instruction that lets all lanes go on.  They are then made for some lanes only, and what the others had is
lost.  The kernels of the built library are looked through for it (no GPU needed)."""
import collections
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from rai_amd._lib import LIB_PATH

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin") or shutil.which("llvm-objdump")
LABEL, KERNEL = re.compile(r"^(?:[0-9a-f]+ )?<(L\d+)>:$"), re.compile(r"^[0-9a-f]+ <(\S+)>:$")
LEAVES = re.compile(r"s_(cbranch|branch|endpgm|setpc|swappc)|s_\w+_b64 exec|s_\w+saveexec")
MOVES = re.compile(r"v_accvgpr_|scratch_|v_mov_b(32|64)_e32 v\S+, v")


def misplaced(assembly):
    """Kernel -> blocks that copy registers, and do nothing else with vectors, ahead of the restore of the mask of lanes that they begin with."""
    found, kernel, label, vectors = collections.defaultdict(list), None, None, []
    for line in assembly.splitlines():
        m = LABEL.match(line)
        if m:
            label, vectors = m[1], []
            continue
        m = KERNEL.match(line)
        if m:
            kernel, label = m[1], None
            continue
        op = line.split("//")[0].strip()
        if label is None or not op:
            continue
        if op.startswith("s_or_b64 exec, exec,"):
            if any(v.startswith(("v_accvgpr_", "scratch_")) for v in vectors) and all(MOVES.match(v) for v in vectors):
                found[kernel].append((label, vectors))
            label = None
        elif LEAVES.match(op):
            label = None
        elif re.match(r"(v_|scratch_|buffer_|global_|flat_|ds_)", op) and not op.startswith("v_writelane"):
            vectors.append(op)
    return dict(found)


def test_the_search_finds_what_it_is_for():
    bad = """
0000000000001000 <kernel_a>:
\ts_and_saveexec_b64 s[8:9], s[66:67]
\ts_cbranch_execz L3
\tglobal_load_dword v2, v[156:157], off
<L3>:
\tv_accvgpr_write_b32 a84, v184
\ts_mov_b64 s[52:53], s[44:45]
\ts_or_b64 exec, exec, s[8:9]
\tv_add_u32_e32 v1, s69, v1
"""
    assert list(misplaced(bad)) == ["kernel_a"]
    right = bad.replace("\tv_accvgpr_write_b32 a84, v184\n", "").replace("\tv_add_u32", "\tv_accvgpr_write_b32 a84, v184\n\tv_add_u32")
    assert misplaced(right) == {}
    assert misplaced(bad.replace("\ts_mov_b64 s[52:53], s[44:45]", "\tv_mul_f32_e32 v3, v4, v5")) == {}   # the body of the other branch


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
@pytest.mark.skipif(not LIB_PATH.exists(), reason="library not built")
def test_no_kernel_copies_registers_for_some_lanes_only(tmp_path):
    lib = tmp_path / LIB_PATH.name
    shutil.copyfile(LIB_PATH, lib)
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    parts = sorted(p for p in Path(tmp_path).iterdir() if p.name.endswith("gfx950"))
    assert parts
    found, kernels = {}, 0
    for p in parts:
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--symbolize-operands", str(p)], check=True, capture_output=True, text=True).stdout
        kernels += text.count("s_endpgm")
        found.update(misplaced(text))
    assert kernels > 100 and found == {}
