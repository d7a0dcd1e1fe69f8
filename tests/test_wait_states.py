"""The copies from memory to LDS that the prompt kernel writes out: the compiler does not see into such a
block, so the block itself has to keep the gfx950's distances.  A vector instruction that writes a scalar
register (a read of one lane) needs five wait states before a memory instruction reads that register as its
address, a write of M0 one before a load to LDS.  Read from the built library's own code (no device)."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

LIB = os.path.join(ROOT, "rust-mlx_amd", "libmx355.so")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def too_near(code):
    """(loads to LDS seen, those whose address or M0 was written too near before them)."""
    seen, bad, before, kernel = 0, [], [], ""
    for line in code.splitlines():
        name = re.match(r"[0-9a-f]+ <(.+)>:", line)
        if name:
            kernel, before = name.group(1), []
            continue
        ins = line.split("//")[0].strip()
        if not ins:
            continue
        if re.match(r"global_load_lds|buffer_load.* lds", ins):
            seen += 1
            regs = set()
            for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", ins):
                regs |= set(range(int(a), int(b) + 1))
            wait = 0
            for past in reversed(before):
                lane = re.match(r"v_read(?:first)?lane_b32 (?:s(\d+)|(m0))", past)
                if lane and wait < 5 and (lane.group(2) or int(lane.group(1)) in regs):
                    bad.append((kernel[:60], past, ins, wait))
                if wait < 1 and re.match(r"s_\w+ m0,", past):
                    bad.append((kernel[:60], past, ins, wait))
                nop = re.match(r"s_nop (\d+)", past)
                wait += int(nop.group(1)) + 1 if nop else 1
                if wait >= 5:
                    break
        before = before[-6:] + [ins]
    return seen, bad


def test_the_check_itself():
    near = "0 <k>:\n v_readfirstlane_b32 s6, v2\n s_mov_b32 m0, s1\n s_nop {}\n global_load_lds_dwordx4 v1, s[6:7]\n"
    assert too_near(near.format(0))[1] and not too_near(near.format(3))[1]
    assert too_near("0 <k>:\n s_mov_b32 m0, s1\n global_load_lds_dwordx4 v[2:3], off\n")[1]
    assert too_near(near.format(3))[0] == 1


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_copies_to_lds_keep_their_distances(mx, tmp_path):
    os.symlink(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    seen, bad = 0, []
    for part in sorted(os.listdir(tmp_path)):
        if not part.endswith("gfx950") or b"prefill_kernelI" not in (tmp_path / part).read_bytes():
            continue
        code = subprocess.run([OBJDUMP, "-d", part], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        n, some = too_near(code)
        seen, bad = seen + n, bad + some
    assert seen >= 24  # the prompt kernels copy that way
    assert not bad, bad[:4]
