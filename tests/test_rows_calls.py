"""CPU tests of the calls of the operators on rows (collcache.torch) that are turned down, or answered, before any GPU is asked."""
import os
import re
import shutil
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ugache_amd"))

import collcache.torch as co  # noqa: E402
import torch.autograd.forward_ad as forward_ad  # noqa: E402
from ugache_amd import build  # noqa: E402

ORDER = co.ExpertOrder(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(5, dtype=torch.int32))


# ---- forward mode ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("call", [
    lambda d: co.coll_torch_expert_dispatch(d(4, 8), ORDER),
    lambda d: co.coll_torch_expert_dispatch_grad(d(8, 8), ORDER),
    lambda d: co.coll_torch_expert_combine(d(8, 8), ORDER),
    lambda d: co.coll_torch_expert_combine_grad(d(4, 8), torch.zeros(8, 8), ORDER),
    lambda d: co.coll_torch_take_rows(d(4, 8), torch.zeros(3, dtype=torch.int64)),
    lambda d: co.coll_torch_take_rows(d(4, 8)[1:], torch.zeros(3, dtype=torch.int64)),
    lambda d: co.coll_torch_take_rows_grad(d(3, 8), torch.zeros(3, dtype=torch.int64), 4),
    lambda d: co.coll_torch_grad_norm([d(3)]),
    lambda d: co.coll_torch_grad_norm(d(3)),
    lambda d: co.coll_torch_clip_grad_norm([d(3)], 1.0),
])
def test_a_tangent_is_refused_and_not_lost(call):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            call(lambda *shape: forward_ad.make_dual(torch.zeros(*shape), torch.ones(*shape)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):  # which forward mode does not mind
            call(lambda *shape: forward_ad.make_dual(torch.zeros(*shape), torch.ones(*shape)))
        with pytest.raises(TypeError, match="GPU"):  # tensors without one are taken as ever, here as far as a CPU's go
            call(torch.zeros)


def test_what_has_no_tangent_of_its_own_is_taken():
    """the primal of a dual tensor, and a detached tensor in a Function that brings its own forward mode, as far as a CPU's go"""
    class Own(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            with pytest.raises(TypeError, match="GPU"):
                co.coll_torch_grad_norm([x])
            return x.sum()

        @staticmethod
        def jvp(ctx, tangent):
            return tangent.sum()

    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(3), torch.ones(3))
        with pytest.raises(TypeError, match="GPU"):
            co.coll_torch_grad_norm([forward_ad.unpack_dual(dual).primal])
        assert forward_ad.unpack_dual(Own.apply(dual)).tangent == 3
    with pytest.raises(TypeError, match="GPU"):
        co.coll_torch_grad_norm([dual])


# ---- the package without the compiled module ------------------------------------------------------------------------

WITHOUT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import collcache.torch as co
import collcache.torch.serving as hps
assert co.__file__.startswith(sys.argv[1]) and callable(co.coll_torch_lookup_unique)
assert torch.equal(hps._at_positions(torch.arange(12.).view(4, 3), torch.tensor([2, 0], dtype=torch.int32)), torch.arange(12.).view(4, 3)[[2, 0]])
for call in (lambda: co.coll_torch_expert_sort(torch.zeros(4, 2, dtype=torch.int64), 4), lambda: co.coll_torch_grad_norm([torch.zeros(3)]),
             lambda: co.coll_torch_take_rows(torch.zeros(4, 8, requires_grad=True), torch.zeros(3, dtype=torch.int64))):
    try:
        call()
    except ImportError as e:
        assert "rows_native" in str(e) and "ugache_amd.build" in str(e), e
    else:
        raise AssertionError("no ImportError")
print("went on")
"""


@pytest.mark.parametrize("module", ["absent", "not loadable"])
def test_the_package_without_the_compiled_module(tmp_path, module):
    """lookups need no rows_native: the package is imported without it, and the operators on rows say what they lack"""
    copy = tmp_path / "ugache_amd"
    shutil.copytree(os.path.join(ROOT, "ugache_amd"), copy, copy_function=os.symlink,
                    ignore=shutil.ignore_patterns("__pycache__", "_build", "csrc", "rows_native.*"))
    if module == "not loadable":
        (copy / "collcache" / "torch" / os.path.basename(build.native_rows_path())).write_bytes(b"")
    done = subprocess.run([sys.executable, "-c", WITHOUT, str(copy)], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "went on" in done.stdout, done.stderr[-2000:]


FOREIGN = """
import importlib.util, sys
import torch
spec = importlib.util.spec_from_file_location("rows_native", sys.argv[1])
module = importlib.util.module_from_spec(spec)
spec.loader.exec_module(module)
print("loaded")
"""


@pytest.mark.parametrize("off,loads", [(0, True), (-1, False), (1, False)])
def test_the_compiled_module_and_the_kernel_library_are_of_one_build(tmp_path, off, loads):
    """beside a library of another ABI, whose calls take other arguments, the module is not loaded"""
    native = build.native_rows_path()
    called = [line.split()[-1] for line in subprocess.run(["nm", "-D", "--undefined-only", native], check=True, stdout=subprocess.PIPE,
                                                          text=True).stdout.splitlines() if line.split()[-1].startswith("ugk_")]
    version = int(re.search(r"#define UGK_ABI_VERSION (\d+)", open(os.path.join(build.INCLUDE, "ugache_hip.h")).read()).group(1))
    (tmp_path / "stub.c").write_text("int ugk_abi_version(void) { return %d; }\n" % (version + off) + "".join(
        "int %s(void) { return 1; }\n" % name for name in called if name != "ugk_abi_version"))
    where = tmp_path / "ugache_amd" / "collcache" / "torch"
    where.mkdir(parents=True)
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "stub.c"), "-o", str(tmp_path / "ugache_amd" / "libugache_hip.so")], check=True)
    shutil.copy(native, where)
    done = subprocess.run([sys.executable, "-c", FOREIGN, str(where / os.path.basename(native))], cwd=tmp_path, capture_output=True, text=True,
                          timeout=300)
    if loads:
        assert done.returncode == 0 and "loaded" in done.stdout, done.stderr[-2000:]
    else:
        assert done.returncode != 0 and "ImportError: libugache_hip.so and rows_native come from different builds" in done.stderr
