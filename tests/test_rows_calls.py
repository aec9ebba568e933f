"""CPU tests of the calls of the operators on rows (collcache.torch) that are turned down, or answered, before any GPU is asked."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ugache_amd"))

import collcache.torch as co  # noqa: E402
import torch.autograd.forward_ad as forward_ad  # noqa: E402

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
