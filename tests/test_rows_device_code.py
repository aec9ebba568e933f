"""What the compiler makes of the operators on rows, on the CPU (hipcc compiles for gfx950 without a GPU)."""
import os
import re
import subprocess

import pytest

from ugache_amd import build

# scalar instructions that leave a condition (a comparison's, or whether the result is zero) and those that leave a carry
CONDITION = re.compile(r"s_(cmp|cmpk|bitcmp|and|or|xor|andn2|orn2|nand|nor|not|bfe|lshl|lshr|ashr|bcnt|min|max|abs|quadmask|wqm)")
CARRY = re.compile(r"s_(add|addc|sub|subb|addk)_")


@pytest.fixture(scope="module", params=["ugk_expert.hip", "ugk_take_rows.hip", "ugk_grad_norm.hip"])
def assembly(request):
    cmd = [build.hipcc_path()] + build.HIPCC_FLAGS + ["--cuda-device-only", "-S", "-I", build.INCLUDE, "-I", build.CSRC,
                                                      os.path.join(build.CSRC, request.param), "-o", "-"]
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert proc.returncode == 0, proc.stderr[-3000:]
    return proc.stdout


def test_a_select_follows_a_comparison(assembly):
    """the compiler has made a minimum of 64-bit scalars, whose comparison a branch used as well, into a select on the carry of an
    earlier addition: lanes then read behind a tensor's end"""
    kernel, last, seen = "", "", 0
    for line in assembly.splitlines():
        label = re.match(r"(_Z\w+):", line)
        if label:
            kernel, last = label.group(1), ""
        if not line.startswith("\t") or not line.split():
            continue
        op = line.split()[0]
        if op.startswith("s_cselect"):
            seen += 1
            assert not CARRY.match(last), (kernel, last, line.strip())
        elif CONDITION.match(op) or CARRY.match(op):
            last = op
    assert seen > 0


def test_no_packed_fp32_and_no_memory_for_spilled_registers(assembly):
    assert not re.search(r"v_pk_(add|mul|fma)_f32", assembly)
    assert set(re.findall(r"; ScratchSize: (\d+)", assembly)) == {"0"}
