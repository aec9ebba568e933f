"""Rows that a router sends to experts and back, rows that are trained, and the norm over their gradients (extensions:
the reference looks rows up and trains none).

Torch operators over the kernels of include/ugache_hip.h: GPU tensors of float32, float16 or bfloat16 in and out, enqueued
on torch's current stream of the tensors' device like any torch op, no host wait, no atomics in a sum: the same
inputs give the same bits.  Every call takes its memory from torch, so calls on several streams and calls recorded into
HIP graphs share nothing.  What cannot be computed raises TypeError or ValueError before anything is enqueued; a failing
launch raises RuntimeError.

The operators that have a gradient record it (torch.autograd) where an input asks for one; the gradients are entry points of
their own as well, for programs that call backward passes themselves.
"""
import array
import collections
import importlib.util
import os

import torch
from torch.autograd.function import once_differentiable

from ..common import _PKG_DIR

_spec = importlib.util.spec_from_file_location("collcache.torch._hip", os.path.join(_PKG_DIR, "hip.py"))
_hip = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_hip)
_L = _hip.lib()

# element codes of the kernels: the size for fp32 and fp16, UGK_ELEM_BF16 for bfloat16
_ELEM = {torch.float32: 4, torch.float16: 2, torch.bfloat16: _hip.ELEM_BF16}
_INT = (torch.int32, torch.int64)
MAX_EXPERTS = 1024

ExpertOrder = collections.namedtuple("ExpertOrder", ["slot", "src", "offsets"])
ExpertOrder.__doc__ = """The assignments of a batch in order of their experts (coll_torch_expert_sort), int32 GPU tensors:
slot     the position of every assignment, -1 where it has no expert; shaped like the expert ids
src      the assignment at every position, -1 behind the last live one: token src[p] // top_k is at position p
offsets  [num_experts + 1]: expert e has the positions offsets[e] .. offsets[e + 1]; offsets[-1] live ones in all"""

_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(fn, dev, *args):
    """fn(*args, stream) on GPU `dev` and torch's current stream there"""
    if dev == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        raise _hip.UgkError(_L.ugk_last_error().decode())


def _check(what, t, dtypes, dev=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes:
        raise TypeError("%s must be a GPU tensor of %s" % (what, ", ".join(str(d)[6:] for d in dtypes)))
    if dev is not None and t.get_device() != dev:
        raise ValueError("%s must be on the GPU of the other tensors" % what)


def _matrix(t):
    """(t as rows, elements from one row to the next); a copy only where rows are not runs of elements in ascending order"""
    if t.dim() != 2:
        t = t.reshape(-1, t.size(-1))
    if (t.size(1) > 1 and t.stride(1) != 1) or (t.size(0) > 1 and t.stride(0) < t.size(1)):
        t = t.contiguous()
    return t, (t.stride(0) if t.size(0) > 1 else t.size(1))


def _check_order(order, dev):
    slot, offsets = order.slot, order.offsets
    _check("order.slot", slot, (torch.int32,), dev)
    _check("order.offsets", offsets, (torch.int32,), dev)
    if slot.dim() not in (1, 2) or (slot.dim() == 2 and slot.size(1) < 1) or offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("order must be what coll_torch_expert_sort returned")
    slot, offsets = slot.contiguous(), offsets.contiguous()
    live = offsets.data_ptr() + 4 * (offsets.numel() - 1)
    return slot, offsets, live, slot.size(0), (slot.size(1) if slot.dim() == 2 else 1)


def _check_rows(what, t, dev=None):
    _check(what, t, _ELEM, dev)
    if t.dim() < 1 or t.size(-1) < 1:
        raise ValueError("%s must be rows of at least one element" % what)


# ---- experts --------------------------------------------------------------------------------------------------------


def coll_torch_expert_sort(expert_ids, num_experts):
    """the assignments of a batch in order of their experts -> ExpertOrder.  expert_ids: GPU int32 / int64 [tokens, top_k]
    or [tokens]; an id outside [0, num_experts) is an assignment that goes nowhere (padding, or an expert of another GPU).
    Within an expert assignments keep their order.  num_experts: 1 to 1024."""
    _check("expert_ids", expert_ids, _INT)
    num_experts = int(num_experts)
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError("num_experts must be 1 to %d, got %d" % (MAX_EXPERTS, num_experts))
    if expert_ids.dim() not in (1, 2) or (expert_ids.dim() == 2 and expert_ids.size(1) < 1):
        raise ValueError("expert_ids must be [tokens, top_k] or [tokens]")
    ids = expert_ids.contiguous()
    n, where = ids.numel(), ids.device
    if n >= 1 << 31:
        raise ValueError("%d assignments are more than positions of 31 bits name" % n)
    slot = torch.empty(ids.shape, dtype=torch.int32, device=where)
    src = torch.empty(n, dtype=torch.int32, device=where)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=where)
    nbytes = _L.ugk_expert_sort_workspace_bytes(n, num_experts)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=where) if nbytes else None
    _launch(_L.ugk_expert_sort_i64 if ids.dtype == torch.int64 else _L.ugk_expert_sort_i32, ids.get_device(), ids.data_ptr(), n,
            num_experts, slot.data_ptr(), src.data_ptr(), offsets.data_ptr(), workspace.data_ptr() if nbytes else None, nbytes)
    return ExpertOrder(slot, src, offsets)


def _dispatch(x, order):
    dev = x.get_device()
    slot, _, live, tokens, top = _check_order(order, dev)
    x, stride = _matrix(x)
    if x.size(0) != tokens:
        raise ValueError("%d rows, but the order is of %d tokens" % (x.size(0), tokens))
    rows = torch.empty(tokens * top, x.size(1), dtype=x.dtype, device=x.device)
    _launch(_L.ugk_expert_dispatch, dev, x.data_ptr(), stride, slot.data_ptr(), live, tokens, top, x.size(1), _ELEM[x.dtype],
            rows.data_ptr())
    return rows


def _combine(rows, order, weights):
    dev = rows.get_device()
    slot, _, _, tokens, top = _check_order(order, dev)
    rows, stride = _matrix(rows)
    if rows.size(0) != slot.numel():
        raise ValueError("%d rows, but the order is of %d assignments" % (rows.size(0), slot.numel()))
    weights = _check_weights(weights, slot, dev)
    out = torch.empty(tokens, rows.size(1), dtype=rows.dtype, device=rows.device)
    _launch(_L.ugk_expert_combine, dev, rows.data_ptr(), rows.size(0), stride, slot.data_ptr(), tokens, top,
            None if weights is None else weights.data_ptr(), 4 if weights is None else _ELEM[weights.dtype], rows.size(1),
            _ELEM[rows.dtype], out.data_ptr())
    return out


def _check_weights(weights, slot, dev):
    if weights is None:
        return None
    _check("weights", weights, _ELEM, dev)
    if weights.numel() != slot.numel():
        raise ValueError("%d weights for %d assignments" % (weights.numel(), slot.numel()))
    return weights.contiguous()


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slot, src, offsets):
        ctx.save_for_backward(slot, src, offsets)
        ctx.shape = x.shape
        return _dispatch(x, ExpertOrder(slot, src, offsets))

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _combine(grad, ExpertOrder(*ctx.saved_tensors), None).view(ctx.shape), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slot, src, offsets):
        ctx.save_for_backward(rows, weights, slot, src, offsets)
        return _combine(rows, ExpertOrder(slot, src, offsets), weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, slot, src, offsets = ctx.saved_tensors
        order = ExpertOrder(slot, src, offsets)
        grad_rows, grad_weights = _combine_grad(grad, rows, order, weights, ctx.needs_input_grad[1])
        return grad_rows.view(rows.shape), grad_weights, None, None, None


def coll_torch_expert_dispatch(x, order):
    """every token's row at the positions of its assignments: a new [tokens * top_k, dim] tensor, rows[order.slot[t, k]] =
    x[t]; the rows of expert e are rows[order.offsets[e] : order.offsets[e + 1]], and those behind order.offsets[-1] are zero.
    x: [tokens, dim], or any leading shape of that many rows.  Differentiable in x."""
    _check_rows("x", x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dispatch.apply(x, *order)
    return _dispatch(x, order)


def coll_torch_expert_dispatch_grad(grad_rows, order):
    """the gradient of coll_torch_expert_dispatch: a new [tokens, dim] tensor, the rows of a token's positions added up in
    fp32; grad_rows: [tokens * top_k, dim]"""
    _check_rows("grad_rows", grad_rows)
    return _combine(grad_rows, order, None)


def coll_torch_expert_combine(rows, order, weights=None):
    """what came back from the experts, added up per token: a new [tokens, dim] tensor, out[t] = sum over k of weights[t, k] *
    rows[order.slot[t, k]] in fp32; assignments without an expert add nothing, a token without any gives a zero row.
    rows: [tokens * top_k, dim]; weights: float32, float16 or bfloat16, one per assignment, or None for ones.
    Differentiable in rows and weights."""
    _check_rows("rows", rows)
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(rows, weights, *order)
    return _combine(rows, order, weights)


def _combine_grad(grad, rows, order, weights, weights_too):
    dev = grad.get_device()
    slot, _, live, tokens, top = _check_order(order, dev)
    grad, grad_stride = _matrix(grad)
    rows, stride = _matrix(rows)
    if grad.size(0) != tokens or rows.size(0) != slot.numel() or grad.size(1) != rows.size(1) or grad.dtype != rows.dtype:
        raise ValueError("grad_out %s of %s and rows %s of %s are not those of %d tokens with %d assignments each" % (
            tuple(grad.shape), grad.dtype, tuple(rows.shape), rows.dtype, tokens, top))
    w = _check_weights(weights, slot, dev)
    grad_rows = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
    grad_w = None if w is None or not weights_too else torch.empty(weights.shape, dtype=w.dtype, device=w.device)
    _launch(_L.ugk_expert_combine_grad, dev, grad.data_ptr(), grad_stride, rows.data_ptr(), stride, slot.data_ptr(), live, tokens,
            top, None if w is None else w.data_ptr(), 4 if w is None else _ELEM[w.dtype], rows.size(1), _ELEM[rows.dtype],
            grad_rows.data_ptr(), None if grad_w is None else grad_w.data_ptr())
    return grad_rows, grad_w


def coll_torch_expert_combine_grad(grad_out, rows, order, weights=None):
    """the gradients of coll_torch_expert_combine: (grad_rows, grad_weights) with grad_rows[order.slot[t, k]] = weights[t, k] *
    grad_out[t], zero behind order.offsets[-1], and grad_weights[t, k] = <rows[order.slot[t, k]], grad_out[t]> of the type of
    the weights, zero where an assignment has no expert (None where there are no weights)"""
    _check_rows("grad_out", grad_out)
    _check_rows("rows", rows, grad_out.get_device())
    return _combine_grad(grad_out, rows, order, weights, True)


# ---- rows that are trained ------------------------------------------------------------------------------------------


def _take_rows(table, index):
    dev = table.get_device()
    t, stride = _matrix(table)
    flat = index.reshape(-1).contiguous()
    out = torch.empty(*index.shape, t.size(1), dtype=t.dtype, device=t.device)
    _launch(_L.ugk_take_rows_i64 if flat.dtype == torch.int64 else _L.ugk_take_rows_i32, dev, t.data_ptr(), t.size(0), stride,
            flat.data_ptr(), flat.numel(), t.size(1), _ELEM[t.dtype], out.data_ptr())
    return out


class _TakeRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index):
        ctx.save_for_backward(index)
        ctx.num_rows = table.size(0)
        return _take_rows(table, index)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return coll_torch_take_rows_grad(grad, ctx.saved_tensors[0], ctx.num_rows), None


def coll_torch_take_rows(table, index):
    """rows by index: a new [*index.shape, dim] tensor, out[i] = table[index[i]], bit for bit; an index outside [0, rows) is
    padding and gives a zero row.  table: [rows, dim] (a token embedding, or the distinct rows of coll_torch_lookup_unique
    with its inverse as index); index: GPU int32 / int64.  Differentiable in table."""
    _check_rows("table", table)
    if table.dim() != 2:
        raise ValueError("table must be [rows, dim]")
    _check("index", index, _INT, table.get_device())
    if torch.is_grad_enabled() and table.requires_grad:
        return _TakeRows.apply(table, index)
    return _take_rows(table, index)


def coll_torch_take_rows_grad(grad, index, num_rows):
    """the gradient of coll_torch_take_rows, or of any lookup of rows by key: a new [num_rows, dim] tensor whose row r is the
    sum of grad[i] over all i with index[i] == r, added in fp32 in an order that the index alone fixes; rows nobody named
    are zero.  grad: [*index.shape, dim].  With the distinct keys and the inverse of coll_torch_lookup_unique: the gradient of
    the distinct rows."""
    _check_rows("grad", grad)
    dev = grad.get_device()
    _check("index", index, _INT, dev)
    num_rows = int(num_rows)
    g, stride = _matrix(grad)
    flat = index.reshape(-1).contiguous()
    n = flat.numel()
    if g.size(0) != n:
        raise ValueError("%d rows for %d indices" % (g.size(0), n))
    if not 0 <= num_rows < 1 << 31 or n >= 1 << 31:
        raise ValueError("%d indices into %d rows: both must be below 2^31" % (n, num_rows))
    out = torch.empty(num_rows, g.size(1), dtype=g.dtype, device=g.device)
    nbytes = _L.ugk_take_rows_grad_workspace_bytes(n, num_rows, g.size(1))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=g.device)
    _launch(_L.ugk_take_rows_grad_i64 if flat.dtype == torch.int64 else _L.ugk_take_rows_grad_i32, dev, g.data_ptr(), stride,
            flat.data_ptr(), n, num_rows, g.size(1), _ELEM[g.dtype], out.data_ptr(), workspace.data_ptr(), nbytes)
    return out


# ---- the norm over gradients ----------------------------------------------------------------------------------------


def _dense(t):
    """whether t's elements are one run of memory, in whatever order of its dimensions"""
    expect = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.size()) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _norm_call(grads, max_norm, out):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(grads):
            raise ValueError("%d outputs for %d gradients" % (len(out), len(grads)))
        out = [o for o, g in zip(out, grads) if g is not None]
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("no gradients")
    in_place = max_norm is not None and out is None
    dev = grads[0].get_device()
    listed, kept = [], []
    for i, g in enumerate(grads):
        code = _ELEM.get(g.dtype)
        if code is None or not g.is_cuda or g.layout != torch.strided:
            raise TypeError("gradients must be dense GPU tensors of float32, float16 or bfloat16")
        if g.get_device() != dev:
            raise ValueError("the gradients must be on one GPU")
        if not g.is_contiguous() and not (out is None and g.numel() and _dense(g)):
            if in_place and g.numel():
                raise ValueError("a gradient of strides %s cannot be scaled in place: its elements are no run of memory"
                                 % (tuple(g.stride()),))
            g = g.contiguous()
            kept.append(g)
        at = g.data_ptr()
        to = at
        if out is not None:
            o = out[i]
            if o.dtype != g.dtype or o.shape != g.shape or o.get_device() != dev or not o.is_contiguous():
                raise ValueError("an output must be contiguous and of its gradient's shape, type and GPU")
            to = o.data_ptr()
        listed += (at, to, g.numel(), code)
    if max_norm is not None:
        places = [p for p, n in zip(listed[1::4], listed[2::4]) if n]
        if len(set(places)) != len(places):
            raise ValueError("two gradients are written to the same place")
    table = array.array("Q", listed)
    address, n = table.buffer_info()[0], len(grads)
    nbytes = _L.ugk_grad_norm_workspace_bytes(address, n)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=norm.device)
    if max_norm is None:
        _launch(_L.ugk_grad_norm, dev, address, n, workspace.data_ptr(), nbytes, norm.data_ptr())
    else:
        _launch(_L.ugk_grad_clip, dev, address, n, max_norm, workspace.data_ptr(), nbytes, norm.data_ptr())
    return norm


def coll_torch_grad_norm(grads):
    """the l2 norm over all elements of all tensors: a float32 GPU scalar.  Squares and sums are held in 64 bits, so neither
    large nor tiny gradients leave the range.  Entries that are None are left out."""
    with torch.no_grad():
        return _norm_call(grads, None, None)


def coll_torch_clip_grad_norm(grads, max_norm, out=None):
    """scale the gradients so that their norm is at most max_norm: every element times min(1, max_norm / (norm + 1e-6)), rounded
    once; returns the norm before that, a float32 GPU scalar.  In place, or into the tensors of `out` (the gradients then
    stay).  Without a host wait: a norm that is not finite shows in the result (no number: every element none; infinite: the
    finite elements zero).  No two gradients may share memory.  Gradients of equal keys have to be summed before
    (coll_torch_take_rows_grad): the norm of the parts is not the norm of the sum."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must be at least 0, got %r" % (max_norm,))
    with torch.no_grad():
        return _norm_call(grads, max_norm, out)
