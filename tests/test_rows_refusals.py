"""CPU tests of what the operators on rows refuse (collcache.torch, ugk_expert_*, ugk_take_rows_*, ugk_grad_*): bad arguments are
turned down before anything reaches a GPU."""
import ctypes
import os
import sys

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ugache_amd"))

import collcache.torch as co  # noqa: E402
from ugache_amd import hip  # noqa: E402

P = 4096  # a pointer nobody follows
WS = 1 << 40


def tensors(*entries):
    return (hip.Tensor * len(entries))(*[hip.Tensor(*e, 0) for e in entries])


@pytest.mark.parametrize("name,args,message", [
    ("ugk_expert_sort_i64", (P, 8, 0, P, P, P, P, WS, None), "experts"),
    ("ugk_expert_sort_i64", (P, 8, 1025, P, P, P, P, WS, None), "1 to 1024"),
    ("ugk_expert_sort_i32", (P, 1 << 31, 8, P, P, P, P, WS, None), "31 bits"),
    ("ugk_expert_sort_i32", (None, 8, 8, P, P, P, P, WS, None), "null pointer"),
    ("ugk_expert_sort_i32", (P, 8, 8, P, P, None, P, WS, None), "null pointer"),
    ("ugk_expert_sort_i32", (P, 100_000, 8, P, P, P, P, 3, None), "workspace of 3 bytes"),
    ("ugk_expert_sort_i32", (P, 100_000, 8, P, P, P, None, WS, None), "workspace"),
    ("ugk_expert_dispatch", (P, 64, P, P, 4, 2, 64, 3, P, None), "element code 3"),
    ("ugk_expert_dispatch", (P, 64, P, P, 4, 0, 64, 4, P, None), "assignments"),
    ("ugk_expert_dispatch", (P, 64, P, P, 1 << 30, 2, 64, 4, P, None), "31 bits"),
    ("ugk_expert_dispatch", (P, 64, P, P, 4, 2, 0, 4, P, None), "rows of 0"),
    ("ugk_expert_dispatch", (P, 63, P, P, 4, 2, 64, 4, P, None), "stride of 63"),
    ("ugk_expert_dispatch", (P, 64, P, None, 4, 2, 64, 4, P, None), "null pointer"),
    ("ugk_expert_combine", (P, 8, 64, P, 4, 2, P, 5, 64, 4, P, None), "code 5 of the weights"),
    ("ugk_expert_combine", (P, 1 << 31, 64, P, 4, 2, P, 4, 64, 4, P, None), "31 bits"),
    ("ugk_expert_combine", (None, 8, 64, P, 4, 2, P, 4, 64, 4, P, None), "null pointer"),
    ("ugk_expert_combine", (P, 8, 1, P, 4, 2, P, 4, 64, 4, P, None), "stride of 1"),
    ("ugk_expert_combine_grad", (P, 64, P, 2, P, P, 4, 2, P, 4, 64, 4, P, P, None), "stride of 2"),
    ("ugk_expert_combine_grad", (P, 64, None, 64, P, P, 4, 2, P, 4, 64, 4, P, P, None), "null pointer"),
    ("ugk_expert_combine_grad", (P, 64, P, 64, P, P, 4, 2, P, 9, 64, 4, P, P, None), "code 9"),
    ("ugk_take_rows_i64", (P, 10, 64, P, 5, 64, 8, P, None), "element code 8"),
    ("ugk_take_rows_i64", (P, 10, 64, P, 5, 0, 4, P, None), "rows of 0"),
    ("ugk_take_rows_i32", (P, 10, 64, None, 5, 64, 4, P, None), "null pointer"),
    ("ugk_take_rows_i32", (None, 10, 64, P, 5, 64, 4, P, None), "null pointer"),
    ("ugk_take_rows_grad_i64", (P, 64, P, 1 << 31, 10, 64, 4, P, P, WS, None), "31 bits"),
    ("ugk_take_rows_grad_i64", (P, 64, P, 5, 1 << 31, 64, 4, P, P, WS, None), "31 bits"),
    ("ugk_take_rows_grad_i32", (P, 8, P, 5, 10, 64, 4, P, P, WS, None), "stride of 8"),
    ("ugk_take_rows_grad_i32", (P, 64, P, 5, 10, 64, 4, P, P, 16, None), "workspace of 16 bytes"),
    ("ugk_take_rows_grad_i32", (P, 64, P, 5, 10, 64, 4, None, P, WS, None), "null pointer"),
    ("ugk_take_rows_grad_i32", (P, 4096, P, 1 << 26, 1 << 20, 4096, 4, P, P, WS, None), "more than one launch takes"),
    ("ugk_take_rows_i32", (P, 10, 4096, P, 1 << 26, 4096, 4, P, None), "more than one launch takes"),
    ("ugk_expert_dispatch", (P, 4096, P, P, 1 << 26, 2, 4096, 4, P, None), "more than one launch takes"),
    ("ugk_expert_combine", (P, 1 << 27, 4096, P, 1 << 26, 2, P, 4, 4096, 4, P, None), "more than one launch takes"),
    ("ugk_expert_combine_grad", (P, 4096, P, 4096, P, P, 1 << 26, 2, P, 4, 4096, 4, P, P, None), "more than one launch takes"),
    ("ugk_grad_norm", (tensors((P, None, 8, 3)), 1, P, WS, P, None), "element code 3 of tensor 0"),
    ("ugk_grad_norm", (tensors((P, None, 8, 4), (None, None, 8, 4)), 2, P, WS, P, None), "null data of tensor 1"),
    ("ugk_grad_norm", (tensors((P, None, 8, 4)), 1, P, 8, P, None), "workspace of 8 bytes"),
    ("ugk_grad_norm", (tensors((P, None, 8, 4)), 1, P, WS, None, None), "null output"),
    ("ugk_grad_norm", (None, 1, P, WS, P, None), "null list"),
    ("ugk_grad_clip", (tensors((P, None, 8, 4)), 1, -1.0, P, WS, P, None), "limit of -1"),
    ("ugk_grad_clip", (tensors((P, None, 8, 4)), 1, float("nan"), P, WS, P, None), "limit of"),
])
def test_the_kernel_layer_refuses(name, args, message):
    args = [ctypes.addressof(a) if isinstance(a, ctypes.Array) else a for a in args]
    with pytest.raises(hip.UgkError, match=message):
        hip.call(name, *args)


ORDER = co.ExpertOrder(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(5, dtype=torch.int32))


@pytest.mark.parametrize("call", [
    lambda: co.coll_torch_expert_sort(torch.zeros(4, 2, dtype=torch.int64), 4),
    lambda: co.coll_torch_expert_sort([1, 2], 4),
    lambda: co.coll_torch_expert_dispatch(torch.zeros(4, 8), ORDER),
    lambda: co.coll_torch_expert_dispatch_grad(torch.zeros(8, 8), ORDER),
    lambda: co.coll_torch_expert_combine(torch.zeros(8, 8), ORDER),
    lambda: co.coll_torch_expert_combine_grad(torch.zeros(4, 8), torch.zeros(8, 8), ORDER),
    lambda: co.coll_torch_take_rows(torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)),
    lambda: co.coll_torch_take_rows_grad(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 4),
    lambda: co.coll_torch_grad_norm([torch.zeros(3)]),
    lambda: co.coll_torch_clip_grad_norm([torch.zeros(3)], 1.0),
    lambda: co.coll_torch_clip_grad_norm([torch.zeros(3, dtype=torch.float64)], 1.0),
])
def test_tensors_that_are_not_on_a_gpu(call):
    with pytest.raises(TypeError, match="GPU"):
        call()


@pytest.mark.parametrize("call,message", [
    (lambda: co.coll_torch_clip_grad_norm([torch.zeros(3)], -1.0), "max_norm"),
    (lambda: co.coll_torch_clip_grad_norm([torch.zeros(3)], float("nan")), "max_norm"),
    (lambda: co.coll_torch_grad_norm([]), "no gradients"),
    (lambda: co.coll_torch_grad_norm([None]), "no gradients"),
    (lambda: co.coll_torch_clip_grad_norm([torch.zeros(3)], 1.0, out=[]), "0 outputs"),
])
def test_values_that_make_no_sense(call, message):
    with pytest.raises(ValueError, match=message):
        call()
