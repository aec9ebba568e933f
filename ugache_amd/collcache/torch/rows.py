"""Rows that a router sends to experts and back, rows that are trained, and the norm over their gradients (extensions:
the reference looks rows up and trains none).

Torch operators over the kernels of include/ugache_hip.h: GPU tensors of float32, float16 or bfloat16 in and out, enqueued
on torch's current stream of the tensors' device like any torch op, no host wait, no atomics in a sum: the same
inputs give the same bits.  Every call takes its memory from torch, so calls on several streams and calls recorded into
HIP graphs share nothing.  Bad arguments raise TypeError or ValueError before anything is enqueued; sizes beyond what one launch
takes, and a launch that fails, raise RuntimeError.  Rows whose elements are not neighbours (a transposed table) are copied first.

The operators that are called differentiable below record their gradient (torch.autograd, reverse mode) where an input asks
for one; the gradients are entry points of their own as well, for programs that call backward passes themselves, and record
nothing, like the norm and the clipping.  There is no forward mode: a tensor with a tangent (torch.autograd.forward_ad) raises
NotImplementedError.  The calls themselves are compiled (collcache.torch.rows_native); where that module is not built, or built
for another torch, they raise ImportError and the lookups go on without them.
"""
import collections

import torch
from torch.autograd.function import once_differentiable


class _Missing:
    """in the place of the compiled module: every call of it raises why it could not be loaded"""

    def __init__(self, why):
        self._why = why

    def __getattr__(self, name):
        raise ImportError("the operators on rows need collcache.torch.rows_native (python -m ugache_amd.build): %s" % self._why)


try:
    from . import rows_native as _native
except ImportError as _error:
    _native = _Missing(_error)

AVAILABLE = not isinstance(_native, _Missing)
MAX_EXPERTS = 1024

ExpertOrder = collections.namedtuple("ExpertOrder", ["slot", "src", "offsets"])
ExpertOrder.__doc__ = """The assignments of a batch in order of their experts (coll_torch_expert_sort), int32 GPU tensors:
slot     the position of every assignment, -1 where it has no expert; shaped like the expert ids
src      the assignment at every position, -1 behind the last live one: token src[p] // top_k is at position p
offsets  [num_experts + 1]: expert e has the positions offsets[e] .. offsets[e + 1]; offsets[-1] live ones in all"""

_grad_enabled = torch.is_grad_enabled


def _asks(t):
    return isinstance(t, torch.Tensor) and t.requires_grad


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slot, offsets):
        ctx.save_for_backward(slot, offsets)
        ctx.shape = x.shape
        return _native.dispatch(x, slot, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _native.dispatch_grad(grad, *ctx.saved_tensors).view(ctx.shape), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slot, offsets):
        # each gradient reads the other's values; those that no gradient reads may change, or go
        for_rows, for_weights = ctx.needs_input_grad[:2]
        ctx.save_for_backward(rows if for_weights else None, weights if for_rows else None, slot, offsets)
        ctx.shape = rows.shape
        ctx.unread = None if for_rows or weights is None else weights.detach()  # its shape and type
        return _native.combine(rows, slot, offsets, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, slot, offsets = ctx.saved_tensors
        for_rows, for_weights = ctx.needs_input_grad[:2]
        grad_rows, grad_weights = _native.combine_grad(grad, rows, slot, offsets, ctx.unread if weights is None else weights, for_weights)
        return grad_rows.view(ctx.shape) if for_rows else None, grad_weights, None, None


class _TakeRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index):
        ctx.save_for_backward(index)
        ctx.num_rows = table.size(0)
        return _native.take_rows(table, index)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _native.take_rows_grad(grad, ctx.saved_tensors[0], ctx.num_rows), None


# ---- experts --------------------------------------------------------------------------------------------------------


def coll_torch_expert_sort(expert_ids, num_experts):
    """the assignments of a batch in order of their experts -> ExpertOrder.  expert_ids: GPU int32 / int64 [tokens, top_k]
    or [tokens]; an id outside [0, num_experts) is an assignment that goes nowhere (padding, or an expert of another GPU).
    Within an expert assignments keep their order.  num_experts: 1 to 1024."""
    return ExpertOrder(*_native.expert_sort(expert_ids, num_experts))


def coll_torch_expert_dispatch(x, order):
    """every token's row at the positions of its assignments: a new [tokens * top_k, dim] tensor, rows[order.slot[t, k]] =
    x[t]; the rows of expert e are rows[order.offsets[e] : order.offsets[e + 1]], and those behind order.offsets[-1] are zero.
    x: [tokens, dim], or any leading shape of that many rows.  Differentiable in x."""
    if _grad_enabled() and _asks(x):
        return _Dispatch.apply(x, order.slot, order.offsets)
    return _native.dispatch(x, order.slot, order.offsets)


def coll_torch_expert_dispatch_grad(grad_rows, order):
    """the gradient of coll_torch_expert_dispatch: a new [tokens, dim] tensor, the rows of a token's positions added up in
    fp32; grad_rows: [tokens * top_k, dim]"""
    return _native.dispatch_grad(grad_rows, order.slot, order.offsets)


def coll_torch_expert_combine(rows, order, weights=None):
    """what came back from the experts, added up per token: a new [tokens, dim] tensor, out[t] = sum over k of weights[t, k] *
    rows[order.slot[t, k]] in fp32; assignments without an expert add nothing, a token without any gives a zero row.
    rows: [tokens * top_k, dim]; weights: float32, float16 or bfloat16, [tokens, top_k] (or any leading shape of
    that many tokens) or [tokens * top_k], or None for ones.  Differentiable in rows and weights."""
    if _grad_enabled() and (_asks(rows) or _asks(weights)):
        return _Combine.apply(rows, weights, order.slot, order.offsets)
    return _native.combine(rows, order.slot, order.offsets, weights)


def coll_torch_expert_combine_grad(grad_out, rows, order, weights=None):
    """the gradients of coll_torch_expert_combine: (grad_rows, grad_weights) with grad_rows[order.slot[t, k]] = weights[t, k] *
    grad_out[t], zero behind order.offsets[-1], and grad_weights[t, k] = <rows[order.slot[t, k]], grad_out[t]> of the type of
    the weights, zero where an assignment has no expert (None where there are no weights)"""
    return _native.combine_grad(grad_out, rows, order.slot, order.offsets, weights, True)


# ---- rows that are trained ------------------------------------------------------------------------------------------


def coll_torch_take_rows(table, index):
    """rows by index: a new [*index.shape, dim] tensor, out[i] = table[index[i]], bit for bit; an index outside [0, rows) is
    padding and gives a zero row.  table: [rows, dim] (a token embedding, or the distinct rows of coll_torch_lookup_unique
    with its inverse as index); index: GPU int32 / int64.  Differentiable in table."""
    if _grad_enabled() and _asks(table):
        return _TakeRows.apply(table, index)
    return _native.take_rows(table, index)


def coll_torch_take_rows_grad(grad, index, num_rows):
    """the gradient of coll_torch_take_rows, or of any lookup of rows by key: a new [num_rows, dim] tensor whose row r is the
    sum of grad[i] over all i with index[i] == r, added in fp32 in an order that the index alone fixes; rows nobody named
    are zero.  grad: [*index.shape, dim], or one of the two a list in the order of the other.  With the distinct keys and the
    inverse of coll_torch_lookup_unique: the gradient of the distinct rows."""
    return _native.take_rows_grad(grad, index, num_rows)


# ---- the norm over gradients ----------------------------------------------------------------------------------------


def coll_torch_grad_norm(grads):
    """the l2 norm over all elements of all tensors: a float32 GPU scalar.  Squares and sums are held in 64 bits, so neither
    large nor tiny gradients leave the range.  grads: a tensor, or a sequence or an iterator of them; entries that are None are
    left out."""
    return _native.grad_norm(grads, None, None)


def coll_torch_clip_grad_norm(grads, max_norm, out=None):
    """scale the gradients so that their norm is at most max_norm: every element times min(1, max_norm / (norm + 1e-6)), rounded
    once; returns the norm before that, a float32 GPU scalar.  In place, or into the tensors of `out` (the gradients then
    stay).  Without a host wait: a norm that is not finite shows in the result (no number: every element none; infinite: the
    finite elements zero); max_norm infinite: nothing is scaled.  What is written is written once and is no other gradient's
    memory: ValueError.  Gradients of equal keys have to be summed before
    (coll_torch_take_rows_grad): the norm of the parts is not the norm of the sum."""
    return _native.grad_norm(grads, float(max_norm), out)
