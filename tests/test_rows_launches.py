"""Which kernels the operators on rows launch, on the CPU: tests/sanitizer/launch_order.cc lists the launches of a call of the
built kernel library instead of performing them."""
import os
import subprocess

import pytest

from ugache_amd import build

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitizer")
MB = 1 << 20


@pytest.fixture(scope="module")
def launches():
    proc = subprocess.run(["make", "-C", HERE, "_build/launch_order"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout[-4000:]
    if not os.path.exists(build.HIP_LIB):
        build.build_hip()

    def run(call, *numbers, **environment):
        """-> (kernel, template arguments) of the launches"""
        out = subprocess.run([os.path.join(HERE, "_build", "launch_order"), build.HIP_LIB, call, *map(str, numbers)], check=True,
                             stdout=subprocess.PIPE, text=True, env={**os.environ, **environment}).stdout
        return [tuple(line.split()[:2]) for line in out.splitlines() if not line.startswith("words ")]

    return run


# 1,024 fp32 elements a row; the output, and with clipping what is read and written, against 256 MiB
@pytest.mark.parametrize("call,sizes,past", [("dispatch", (100, 1024), False), ("dispatch", (128 * 256, 1024), False),
                                             ("dispatch", (128 * 256 + 1, 1024), True), ("take", (5, 1024), False), ("take", (65_536, 1024), False),
                                             ("take", (65_537, 1024), True), ("clip", (1000,), False), ("clip", (32 * MB,), False),
                                             ("clip", (32 * MB + 1,), True)])
def test_what_lookups_are_told_of_their_outputs_is_nothing_to_the_operators(launches, call, sizes, past):
    """size decides whether stores go past the caches, not the hint that a lookup has left on the thread nor its variable"""
    done = launches(call, 0, *sizes)
    assert ("true" in done[-1][1]) == past, done
    for hint in (1, 2):
        assert launches(call, hint, *sizes) == done
    for forced in "01":
        assert launches(call, 0, *sizes, UGK_GATHER_NT_STORE=forced) == done
