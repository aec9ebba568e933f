"""GPU tests of calls of the operators on rows (collcache.torch) that a program can make beside the ordinary ones: forward-mode
tensors, shapes that pair rows with other entries, tensors changed or let go between a forward and a backward pass, rows that
very many entries name.

Small whole numbers are summed exactly in float32 as long as no partial sum passes 2^24: results are then equal bit for bit
whatever the order, and one entry lost or counted twice shows."""
import json
import os
import shutil
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ugache_amd"))

if torch.cuda.is_available():
    import collcache.torch as co
    import torch.autograd.forward_ad as forward_ad


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def whole(g, *shape, dtype=torch.float32):
    return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


def order_of(g, tokens, top, experts):
    ids = torch.topk(torch.rand(tokens, experts, device="cuda", generator=g), top, dim=1).indices
    return co.coll_torch_expert_sort(ids, experts)


# ---- forward mode ---------------------------------------------------------------------------------------------------


def test_a_tangent_is_refused_and_not_lost():
    g = gen(1)
    order = order_of(g, 10, 2, 4)
    x, rows, w, table = randn(g, 10, 8), randn(g, 20, 8), torch.rand(10, 2, device="cuda", generator=g), randn(g, 30, 8)
    index = torch.randint(0, 30, (12,), device="cuda", generator=g)
    out = [torch.empty_like(x)]
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: co.coll_torch_expert_dispatch(dual(x), order), lambda: co.coll_torch_expert_combine(dual(rows), order, w),
                     lambda: co.coll_torch_expert_combine(rows, order, dual(w)), lambda: co.coll_torch_take_rows(dual(table), index),
                     lambda: co.coll_torch_expert_dispatch(dual(x.clone().requires_grad_()), order),
                     lambda: co.coll_torch_take_rows(dual(table.clone().requires_grad_()), index),
                     lambda: co.coll_torch_expert_dispatch_grad(dual(rows), order), lambda: co.coll_torch_take_rows_grad(dual(x), index[:10], 30),
                     lambda: co.coll_torch_expert_combine_grad(x, dual(rows), order, w), lambda: co.coll_torch_grad_norm([x, dual(rows)]),
                     lambda: co.coll_torch_clip_grad_norm([dual(x)], 1.0, out=out), lambda: co.coll_torch_clip_grad_norm([x], 1.0, out=[dual(out[0])])):
            with pytest.raises(NotImplementedError):
                call()
        # tensors without a tangent are nothing to forward mode
        assert torch.equal(co.coll_torch_take_rows(table, index), table[index])
        assert torch.equal(co.coll_torch_take_rows(forward_ad.unpack_dual(dual(table)).primal, index), table[index])
    assert torch.equal(co.coll_torch_take_rows(table, index), table[index])


def test_a_function_with_a_forward_mode_of_its_own():
    """the operator is linear: a program can give it its tangent"""
    class Take(torch.autograd.Function):
        @staticmethod
        def forward(ctx, table, index):
            ctx.index = index
            return co.coll_torch_take_rows(table, index)

        @staticmethod
        def jvp(ctx, tangent, _):
            return co.coll_torch_take_rows(tangent, ctx.index)

    g = gen(2)
    table, tangent, index = randn(g, 30, 8), randn(g, 30, 8), torch.randint(0, 30, (12,), device="cuda", generator=g)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(Take.apply(forward_ad.make_dual(table, tangent), index))
        assert torch.equal(got.primal, table[index]) and torch.equal(got.tangent, tangent[index])


# ---- the package without the compiled module ------------------------------------------------------------------------

LAYER = """
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np, torch
import collcache.torch as co
import collcache.torch.serving as hps
from collcache.torch import rows
assert co.__file__.startswith(sys.argv[1])
assert hps.Config(ps_config_file=sys.argv[2]) == "OK"
g = torch.Generator().manual_seed(3)
hps.record_hotness(torch.randint(0, 2000, (5000,), generator=g).cuda())
assert hps.Init(ps_config_file=sys.argv[2], global_batch_size=256) == "OK"
ids = torch.randint(0, 2000, (300, 4), generator=g)
at = torch.stack([torch.arange(300).repeat_interleave(4), torch.arange(4).repeat(300)])
sp = torch.sparse_coo_tensor(at, ids.reshape(-1), (300, 4)).cuda()
want = torch.from_numpy(np.fromfile(sys.argv[3], dtype=np.float32)).view(2000, 16)[ids]
for in_library in (False, True):
    layer = hps.SparseLookupLayer(model_name="dlrm", table_id=0, emb_vec_size=16, unique_in_library=in_library)
    assert torch.equal(layer(sp, combiner="sum").cpu(), want.sum(1))
print("operators" if rows.AVAILABLE else "none", flush=True)
hps.Shutdown()
"""


@pytest.mark.parametrize("module", ["there", "absent"])
def test_the_sparse_layer_without_the_compiled_module(tmp_path, module):
    package = os.path.join(ROOT, "ugache_amd")
    if module == "absent":
        package = str(tmp_path / "ugache_amd")
        shutil.copytree(os.path.join(ROOT, "ugache_amd"), package, copy_function=os.symlink,
                        ignore=shutil.ignore_patterns("__pycache__", "_build", "csrc", "rows_native.*"))
    model = tmp_path / "dlrm_sparse.model"
    model.mkdir()
    np.arange(2000, dtype=np.int64).tofile(model / "key")
    np.random.default_rng(1).integers(-9, 10, (2000, 16)).astype(np.float32).tofile(model / "emb_vector")
    path = tmp_path / "ps_config.json"
    path.write_text(json.dumps({"iteration_per_epoch": 50, "epoch": 1, "coll_cache_enable_refresh": False, "models": [{
        "model": "dlrm", "sparse_files": [str(model)], "gpucacheper": 0.3, "max_batch_size": 4096, "deployed_device_list": [0],
        "maxnum_catfeature_query_per_table_per_sample": [26], "embedding_vecsize_per_table": [16], "max_vocabulary_size": [2000]}]}))
    done = subprocess.run([sys.executable, "-c", LAYER, package, str(path), str(model / "emb_vector")], cwd=tmp_path, capture_output=True,
                          text=True, timeout=100)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.split()[-1] == ("operators" if module == "there" else "none")


# ---- shapes that say which entry belongs to which ---------------------------------------------------------------------


def test_weights_in_another_order_are_refused():
    g = gen(4)
    tokens, top = 12, 3
    order = order_of(g, tokens, top, 5)
    rows, w = randn(g, tokens * top, 8), torch.rand(tokens, top, device="cuda", generator=g)
    grad = randn(g, tokens, 8)
    want = co.coll_torch_expert_combine(rows, order, w)
    want_grad = co.coll_torch_expert_combine_grad(grad, rows, order, w)[1]
    for shape in ((tokens * top,), (4, 3, top), (tokens, top, 1), (1, tokens, top), (tokens * top, 1)):
        assert torch.equal(co.coll_torch_expert_combine(rows, order, w.view(shape)), want)
        got = co.coll_torch_expert_combine_grad(grad, rows, order, w.view(shape))[1]
        assert got.shape == shape and torch.equal(got, want_grad.view(shape))
    for bad in (w.t(), w.t().contiguous(), w.view(6, 6), w.t().unsqueeze(0), w.view(4, 3, top).transpose(1, 2).reshape(4, 9)):
        for call in (lambda: co.coll_torch_expert_combine(rows, order, bad), lambda: co.coll_torch_expert_combine_grad(grad, rows, order, bad),
                     lambda: co.coll_torch_expert_combine(rows, order, bad.detach().requires_grad_())):
            with pytest.raises(ValueError, match="top_k"):
                call()
    # one expert a token, and one token: there is only one order
    single = co.coll_torch_expert_sort(torch.arange(12, device="cuda") % 5, 5)
    for shape in ((12,), (12, 1), (3, 4), (1, 12)):
        assert torch.equal(co.coll_torch_expert_combine(rows[:12], single, w.reshape(-1)[:12].view(shape)),
                           co.coll_torch_expert_combine(rows[:12], single, w.reshape(-1)[:12]))
    alone = co.coll_torch_expert_sort(torch.arange(3, device="cuda").view(1, 3), 5)
    for shape in ((3,), (1, 3), (3, 1)):
        assert torch.equal(co.coll_torch_expert_combine(rows[:3], alone, w[0].view(shape)), co.coll_torch_expert_combine(rows[:3], alone, w[:1]))
    none = co.coll_torch_expert_sort(torch.empty(0, 4, dtype=torch.int64, device="cuda"), 9)
    assert co.coll_torch_expert_combine(rows[:0], none, torch.empty(4, 0, device="cuda")).shape == (0, 8)


def test_a_gradient_in_another_order_than_its_index_is_refused():
    g = gen(5)
    index, grad = torch.randint(0, 9, (4, 6), device="cuda", generator=g), whole(g, 4, 6, 8)
    want = torch.zeros(9, 8, device="cuda").index_add_(0, index.reshape(-1), grad.view(24, 8))
    for i, d in ((index, grad), (index.view(24), grad), (index, grad.view(24, 8)), (index.view(2, 2, 6), grad.view(2, 2, 6, 8)),
                 (index.unsqueeze(-1), grad), (index, grad.unsqueeze(0)), (index.view(1, 24), grad)):
        assert torch.equal(co.coll_torch_take_rows_grad(d, i, 9), want)
    for i, d in ((index.t(), grad), (index.t().contiguous(), grad), (index, grad.transpose(0, 1)), (index.view(2, 12), grad),
                 (index.view(2, 2, 6), grad)):
        with pytest.raises(ValueError, match="index.shape"):
            co.coll_torch_take_rows_grad(d, i, 9)
    one = co.coll_torch_take_rows_grad(grad[0, 0], index[0, 0], 9)
    assert torch.equal(one[index[0, 0]], grad[0, 0]) and int(one.any(1).sum()) == int(grad[0, 0].any())
    assert not co.coll_torch_take_rows_grad(grad[:0], index.t()[:, :0], 9).any()


# ---- between a forward and a backward pass ----------------------------------------------------------------------------


@pytest.mark.parametrize("asks", ["rows, no weights", "rows", "weights", "both"])
def test_what_no_gradient_reads_may_change_before_the_backward_pass(asks):
    """the gradient of the rows reads the weights, that of the weights the rows, and neither its own"""
    g = gen(6)
    tokens, top, dim = 40, 3, 20
    order = order_of(g, tokens, top, 8)
    leaf, w = whole(g, tokens * top, dim), whole(g, tokens, top)
    grad = whole(g, tokens, dim)
    want_rows, want_w = co.coll_torch_expert_combine_grad(grad, leaf + 1, order, w)
    if asks == "rows, no weights":
        want_rows = co.coll_torch_expert_combine_grad(grad, leaf + 1, order)[0]
    for changed in ("nothing", "rows", "weights"):
        r = leaf.clone().requires_grad_(asks != "weights")
        v = None if asks == "rows, no weights" else w.clone().requires_grad_(asks != "rows")
        rows, weights = r + 1, None if v is None else v + 0  # made, not leaves: they may be changed in place
        out = co.coll_torch_expert_combine(rows, order, weights)
        with torch.no_grad():
            if changed == "rows":
                rows.mul_(5)
            elif changed == "weights" and weights is not None:
                weights.mul_(5)
        if (changed == "rows" and asks in ("weights", "both")) or (changed == "weights" and asks in ("rows", "both")):
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.backward(grad)
            continue
        out.backward(grad)
        assert r.grad is None if asks == "weights" else torch.equal(r.grad, want_rows)
        if v is not None:
            assert v.grad is None if asks == "rows" else torch.equal(v.grad, want_w)


@pytest.mark.parametrize("weighted", [False, True])
def test_rows_that_no_gradient_reads_are_let_go(weighted):
    g = gen(7)
    order = order_of(g, 1000, 4, 8)
    leaf = randn(g, 4000, 1024).requires_grad_()
    w = torch.rand(1000, 4, device="cuda", generator=g) if weighted else None
    out = co.coll_torch_expert_combine(leaf + 1, order, w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    rows = leaf + 1
    held = torch.cuda.memory_allocated() - before
    assert held >= 4000 * 1024 * 4
    again = co.coll_torch_expert_combine(rows, order, w)
    del rows
    assert torch.cuda.memory_allocated() - before < held  # the output is a quarter of the rows
    assert torch.equal(torch.autograd.grad(out.sum(), leaf)[0], torch.autograd.grad(again.sum(), leaf)[0])


def test_gradients_asked_for_one_at_a_time():
    g = gen(8)
    order = order_of(g, 50, 2, 8)
    rows, w = whole(g, 100, 12).requires_grad_(), whole(g, 50, 2).requires_grad_()
    grad = whole(g, 50, 12)
    want = co.coll_torch_expert_combine_grad(grad, rows.detach(), order, w.detach())
    for k, leaf in enumerate((rows, w)):
        assert torch.equal(torch.autograd.grad(co.coll_torch_expert_combine(rows, order, w), leaf, grad)[0], want[k])
    out = co.coll_torch_expert_combine(rows.view(50, 2, 12), order, w.half())
    out.backward(grad)
    assert torch.equal(rows.grad, want[0]) and torch.equal(w.grad, want[1])
    none = torch.empty(0, 4, dtype=torch.int64, device="cuda")
    nobody = torch.empty(0, 12, device="cuda").requires_grad_()
    co.coll_torch_expert_combine(nobody, co.coll_torch_expert_sort(none, 8)).sum().backward()
    assert nobody.grad.shape == (0, 12)


def test_rows_are_left_out_only_where_nothing_reads_them():
    g = gen(9)
    order = order_of(g, 10, 2, 4)
    for weights in (None, torch.rand(10, 2, device="cuda", generator=g)):
        with pytest.raises(TypeError, match="rows"):
            co.coll_torch_expert_combine_grad(randn(g, 10, 8), None, order, weights)


# ---- rows that very many entries name ---------------------------------------------------------------------------------

# n entries over rows, each of `hot` rows named by its share of `share` of them.  Where rows are found by their position (rows > n,
# or few short rows) and by themselves; more than 16 parts of a row, and of several rows in one workgroup; rows of one element, of
# less than a chunk, and of more than 32 chunks, which are joined column by column
HOT = [(30_000, 1, 24, 1, 1.0), (20_000, 2, 200, 2, 1.0), (700_000, 5, 12, 5, 1.0), (700_000, 5, 1, 2, 0.9), (120_000, 30_000, 48, 1, 0.999),
       (120_000, 30_000, 48, 7, 0.7), (120_000, 300_000, 48, 1, 0.999), (120_000, 300_000, 3, 3, 0.8), (60_000, 70_000, 257, 1, 0.99),
       (60_000, 20_000, 257, 3, 0.9), (60_000, 9000, 1030, 1, 0.95), (40_000, 50_000, 1030, 5, 0.5), (400_000, 3000, 9, 40, 0.95),
       (1_200_000, 1_000_000, 4, 2, 0.6), (1_200_000, 2_000_000, 4, 300, 0.9), (4097, 5000, 300, 1, 1.0), (4000, 8000, 300, 1, 1.0)]


def sums_of_whole(grad, index, rows):
    """[rows, dim] float64: differences of running sums over the entries in order of their rows, exact in whole numbers"""
    order = torch.sort(index).indices
    upto = torch.cat([torch.zeros(1, grad.size(1), dtype=torch.float64, device="cuda"), torch.cumsum(grad.double()[order], 0)])
    ends = torch.cumsum(torch.bincount(index, minlength=rows), 0)
    return upto[ends] - torch.cat([upto[:1], upto[ends[:-1]]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,rows,dim,hot,share", HOT)
def test_no_entry_of_a_row_that_many_name_is_lost(n, rows, dim, hot, share, dtype):
    """whole numbers of at most 3 and fewer than 2^22 entries: every partial sum is exact in float32, so the result is the exact
    sum rounded once, whatever the order"""
    g = gen(n + rows + dim)
    index = torch.randint(0, rows, (n,), device="cuda", generator=g)
    named = torch.randperm(rows, device="cuda", generator=g)[torch.randint(0, hot, (n,), device="cuda", generator=g)]
    index = torch.where(torch.rand(n, device="cuda", generator=g) < share, named, index)
    grad = whole(g, n, dim, dtype=dtype)
    assert torch.equal(co.coll_torch_take_rows_grad(grad, index, rows), sums_of_whole(grad, index, rows).to(dtype))
    runs = torch.sort(index).values  # the same in order, so that the row's entries are neighbours before they are sorted too
    assert torch.equal(co.coll_torch_take_rows_grad(grad, runs.int(), rows), sums_of_whole(grad, runs, rows).to(dtype))


# ---- products and squares, none lost -----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 7, 8, 9, 255, 257, 511, 1001, 1025, 2047, 2049, 4099, 17_001])
def test_no_product_of_a_long_row_is_lost(dim, dtype):
    """dots of whole numbers of at most 3: every partial sum is below 2^24 and exact, also where chunks of a row overlap"""
    g = gen(dim)
    tokens, top = 19, 5
    order = order_of(g, tokens, top, 8)
    rows, grad, w = whole(g, tokens * top, dim, dtype=dtype), whole(g, tokens, dim, dtype=dtype), whole(g, tokens, top)
    grad_rows, grad_w = co.coll_torch_expert_combine_grad(grad, rows, order, w)
    at = rows[order.slot.long()].double()
    assert torch.equal(grad_w.double(), (at * grad.double().unsqueeze(1)).sum(-1))
    assert torch.equal(grad_rows[order.slot.long()].double(), grad.double().unsqueeze(1) * w.double().unsqueeze(-1))
    assert torch.equal(co.coll_torch_expert_combine(rows, order, w).double(), (at * w.double().unsqueeze(-1)).sum(1))


@pytest.mark.parametrize("sizes", [(1, 8191, 8192, 8193, 16_385), (100_000_003, 60_000_001, 5)])
def test_no_square_is_lost(sizes):
    """tensors of zeros with threes at their ends, at the ends of the pieces that are summed, and anywhere: a norm is the root of
    nine times their number, rounded once"""
    g = gen(len(sizes))
    grads = [torch.zeros(n, device="cuda", dtype=torch.bfloat16 if k % 2 == 0 else torch.float32) for k, n in enumerate(sizes)]
    for turn in range(6):
        count = 0
        for t in grads:
            n, piece = t.numel(), 32_768 // t.element_size()
            at = torch.randint(0, n, (3,), device="cuda", generator=g)
            if turn < 3:
                k = int(torch.randint(0, n // piece + 1, (1,), device="cuda", generator=g))
                at = torch.tensor([0, n - 1, k * piece - 1, k * piece, n // 8 * 8 - 1], device="cuda").clamp(0, n - 1)
            t.zero_()[at] = 3
            count += torch.unique(at).numel()
        norm = torch.tensor(9.0 * count, dtype=torch.float64).sqrt().float()
        assert torch.equal(co.coll_torch_grad_norm(grads).cpu(), norm)
        out = [torch.empty_like(t) for t in grads]
        assert torch.equal(co.coll_torch_clip_grad_norm(grads, 1e9, out=out).cpu(), norm)
        assert all(torch.equal(a, b) for a, b in zip(out, grads))
