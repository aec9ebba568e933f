"""GPU tests of the operators on rows (collcache.torch: expert sort, dispatch, combine, rows taken by index, the norm over
gradients and clipping) against plain implementations in 64 bits.

Tolerances, in front of every run: a rounding to a type of unit round-off u (float32 2^-24, float16 2^-11, bfloat16 2^-8) is off
by at most u relative to the value, for float16 at most 2^-25 absolute among its subnormals; a sum of n terms in float32 is off by
at most n * 2^-24 * sum |term| whatever its order, and a fused multiply-add adds one rounding.  Moved rows, positions and
counts are equal bit for bit."""
import os
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

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def close(got, want, terms, count, extra=1):
    """got: rounded once to its type; want, terms (sum of the absolute values of its terms): float64; count: additions in
    float32, extra: further roundings to float32 of a value or of every term"""
    assert got.shape == want.shape
    u = U[got.dtype]
    bound = u * want.abs() + (1 + u) * (count + extra) * F32 * terms + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def random_ids(g, tokens, top, experts, masked=0.0, dtype=torch.int64):
    if top <= experts:
        ids = torch.topk(torch.rand(max(tokens, 1), experts, device="cuda", generator=g), top, dim=1).indices[:tokens]
    else:
        ids = torch.randint(0, experts, (tokens, top), device="cuda", generator=g)
    if masked:
        ids = torch.where(torch.rand(tokens, top, device="cuda", generator=g) < masked, -1, ids)
    return ids.to(dtype)


def sorted_by_hand(ids, experts):
    flat = ids.reshape(-1).cpu().numpy().astype(np.int64)
    live = np.nonzero((flat >= 0) & (flat < experts))[0]
    src = np.full(flat.size, -1, np.int32)
    src[: live.size] = live[np.argsort(flat[live], kind="stable")]
    slot = np.full(flat.size, -1, np.int32)
    slot[src[: live.size]] = np.arange(live.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=experts))]).astype(np.int32)
    return slot.reshape(ids.shape), src, offsets


def check_order(order, ids, experts):
    slot, src, offsets = sorted_by_hand(ids, experts)
    assert order.slot.dtype == order.src.dtype == order.offsets.dtype == torch.int32
    assert np.array_equal(order.offsets.cpu().numpy(), offsets)
    assert np.array_equal(order.slot.cpu().numpy(), slot)
    assert np.array_equal(order.src.cpu().numpy(), src)


# ---- sort -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,top,experts", [
    (1, 1, 1), (1, 8, 256), (2, 1, 2), (7, 3, 10), (63, 1, 64), (64, 1, 63), (65, 2, 1024), (511, 8, 128), (512, 8, 128), (513, 8, 128),
    (2048, 1, 5), (2049, 2, 33), (4096, 1, 1), (5000, 6, 60), (8191, 1, 1000), (20_011, 10, 1024), (131_072, 8, 128), (300_007, 1, 1)])
@pytest.mark.parametrize("masked", [0.0, 0.3])
def test_sort(tokens, top, experts, masked):
    dtype = torch.int32 if (tokens + top) % 2 else torch.int64
    ids = random_ids(gen(tokens + experts), tokens, top, experts, masked, dtype)
    check_order(co.coll_torch_expert_sort(ids, experts), ids, experts)


@pytest.mark.parametrize("tokens,top,experts", [
    (1024, 1, 7), (1025, 1, 7), (2048, 1, 1024), (2049, 1, 64), (4095, 1, 64), (4096, 1, 2), (4097, 1, 64), (32_768, 1, 640), (32_769, 1, 1),
    (32_769, 1, 1024), (150_001, 2, 1023), (70_000, 8, 1000), (700_000, 3, 40), (110_001, 10, 513)])
def test_sort_where_its_shape_changes(tokens, top, experts):
    g = gen(tokens)
    ids = (torch.rand(tokens, top, device="cuda", generator=g) ** 2 * (experts + 1)).long() - 1  # skewed, some nowhere
    check_order(co.coll_torch_expert_sort(ids, experts), ids, experts)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [40, 6000])
def test_sort_ids_out_of_range_go_nowhere(dtype, tokens):
    far = torch.iinfo(dtype)
    ids = torch.randint(0, 16, (tokens, 4), device="cuda", generator=gen(1)).to(dtype)
    ids[::3, 1] = far.max
    ids[::4, 2] = far.min
    ids[1::5, 0] = 16
    if dtype == torch.int64:
        ids[::7, 3] = 1 << 32  # the low half names an expert
    check_order(co.coll_torch_expert_sort(ids, 16), ids, 16)


@pytest.mark.parametrize("tokens", [1, 100, 10_000])
def test_sort_of_one_expert_of_none_and_of_all_alike(tokens):
    nobody = torch.full((tokens, 2), -1, dtype=torch.int64, device="cuda")
    check_order(co.coll_torch_expert_sort(nobody, 7), nobody, 7)
    alike = torch.full((tokens, 2), 6, dtype=torch.int64, device="cuda")
    check_order(co.coll_torch_expert_sort(alike, 7), alike, 7)
    flat = torch.arange(tokens, device="cuda") % 3
    check_order(co.coll_torch_expert_sort(flat, 3), flat, 3)


def test_sort_of_no_tokens():
    order = co.coll_torch_expert_sort(torch.empty(0, 4, dtype=torch.int64, device="cuda"), 9)
    assert order.slot.shape == (0, 4) and order.src.shape == (0,)
    assert torch.equal(order.offsets.cpu(), torch.zeros(10, dtype=torch.int32))


def test_sort_of_strided_ids():
    ids = random_ids(gen(3), 999, 8, 40)
    for view in (ids.t().contiguous().t(), ids[::2], ids[:, ::3], ids[:, 1:2].expand(-1, 4)):
        check_order(co.coll_torch_expert_sort(view, 40), view, 40)


# ---- dispatch and combine -------------------------------------------------------------------------------------------

SHAPES = [  # tokens, top, experts, dim
    (1, 1, 1, 1), (1, 8, 16, 2048), (3, 2, 4, 3), (5, 8, 8, 7), (7, 1, 3, 8), (9, 3, 5, 9), (33, 4, 9, 64), (50, 11, 20, 130),
    (20, 5, 6, 255), (20, 6, 6, 257), (129, 2, 8, 1001), (40, 3, 10, 2048), (17, 8, 64, 4099), (300, 4, 60, 512), (11, 2, 4, 17_001)]


def plain_there(x, slot, n):
    """[n, dim] float64 from x [tokens, dim], zero where no slot points"""
    rows = torch.zeros(n, x.size(1), dtype=torch.float64, device="cuda")
    t, k = torch.nonzero(slot >= 0, as_tuple=True)
    rows[slot[t, k].long()] = x.double()[t]
    return rows


def plain_back(rows, slot, w=None):
    """(sum, sum of absolute terms) float64 [tokens, dim]"""
    total = torch.zeros(slot.size(0), rows.size(1), dtype=torch.float64, device="cuda")
    terms = torch.zeros_like(total)
    for k in range(slot.size(1)):
        t = torch.nonzero(slot[:, k] >= 0).reshape(-1)
        part = rows.double()[slot[t, k].long()]
        if w is not None:
            part = part * w.double()[t, k].unsqueeze(1)
        total[t] += part
        terms[t] += part.abs()
    return total, terms


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [0.0, 0.4])
@pytest.mark.parametrize("tokens,top,experts,dim", SHAPES)
def test_dispatch_and_its_gradient(tokens, top, experts, dim, masked, dtype):
    g = gen(tokens * 7 + dim)
    order = co.coll_torch_expert_sort(random_ids(g, tokens, top, experts, masked), experts)
    x = randn(g, tokens, dim, dtype=dtype)
    rows = co.coll_torch_expert_dispatch(x, order)
    assert rows.dtype == dtype and torch.equal(rows.double(), plain_there(x, order.slot, tokens * top))
    grad = randn(g, tokens * top, dim, dtype=dtype)
    grad[int(order.offsets[-1]):] = float("nan")  # behind the last live row there is nobody's gradient
    want, terms = plain_back(grad, order.slot)
    close(co.coll_torch_expert_dispatch_grad(grad, order), want, terms, top)


@pytest.mark.parametrize("wtype", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,top,experts,dim", SHAPES)
def test_combine_and_its_gradients(tokens, top, experts, dim, dtype, wtype):
    g = gen(tokens * 5 + dim)
    order = co.coll_torch_expert_sort(random_ids(g, tokens, top, experts, 0.3 if dim % 2 else 0.0), experts)
    live, slot = int(order.offsets[-1]), order.slot
    rows = randn(g, tokens * top, dim, dtype=dtype)
    rows[live:] = float("nan")
    w = None if wtype is None else torch.rand(tokens, top, device="cuda", generator=g).to(wtype)
    want, terms = plain_back(rows, slot, w)
    close(co.coll_torch_expert_combine(rows, order, w), want, terms, top)
    grad = randn(g, tokens, dim, dtype=dtype)
    grad_rows, grad_w = co.coll_torch_expert_combine_grad(grad, rows, order, w)
    spread = plain_there(grad, slot, tokens * top)
    if w is None:
        assert grad_w is None and torch.equal(grad_rows.double(), spread)
        return
    scale = torch.zeros(tokens * top, dtype=torch.float64, device="cuda")
    t, k = torch.nonzero(slot >= 0, as_tuple=True)
    scale[slot[t, k].long()] = w.double()[t, k]
    want = spread * scale.unsqueeze(1)
    close(grad_rows, want, want.abs(), 0)
    assert not grad_rows[live:].any()
    products = torch.zeros(tokens, top, dim, dtype=torch.float64, device="cuda")
    products[t, k] = rows.double()[slot[t, k].long()] * grad.double()[t]
    assert grad_w.dtype == wtype
    close(grad_w, products.sum(-1), products.abs().sum(-1), dim)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_strides_and_odd_addresses(dtype):
    g = gen(11)
    tokens, top, experts, dim = 37, 3, 8, 77
    order = co.coll_torch_expert_sort(random_ids(g, tokens, top, experts, 0.2), experts)
    wide = randn(g, tokens, 2 * dim + 3, dtype=dtype)
    for x in (wide[:, 1:1 + dim], wide[:, 3:3 + dim], wide[:, 1:1 + 2 * dim:2], wide[:1, :dim].expand(tokens, dim)):
        assert torch.equal(co.coll_torch_expert_dispatch(x, order).double(), plain_there(x, order.slot, tokens * top))
    deep = randn(g, tokens * top, dim + 9, dtype=dtype)
    w = torch.rand(tokens, 2 * top, device="cuda", generator=g)[:, ::2]
    for rows in (deep[:, 2:2 + dim], deep[:, 5:5 + dim]):
        want, terms = plain_back(rows, order.slot, w)
        close(co.coll_torch_expert_combine(rows, order, w), want, terms, top)
        a = co.coll_torch_expert_combine_grad(wide[:, 1:1 + dim], rows, order, w)
        b = co.coll_torch_expert_combine_grad(wide[:, 1:1 + dim].contiguous(), rows.contiguous(), order, w.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_three_dimensional_tokens_and_one_expert_per_token():
    g = gen(12)
    ids = torch.randint(0, 6, (24,), device="cuda", generator=g)
    order = co.coll_torch_expert_sort(ids, 6)
    x = randn(g, 4, 6, 48, dtype=torch.bfloat16)
    rows = co.coll_torch_expert_dispatch(x, order)
    assert rows.shape == (24, 48)
    assert torch.equal(co.coll_torch_expert_combine(rows, order), x.reshape(24, 48))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nans_stay_with_their_tokens(dtype):
    g = gen(13)
    ids = random_ids(g, 64, 2, 8)
    ids[10] = -1
    order = co.coll_torch_expert_sort(ids, 8)
    x = randn(g, 64, 40, dtype=dtype)
    x[3] = float("inf")
    x[5, 7] = float("nan")
    x[10] = float("nan")  # goes nowhere
    rows = co.coll_torch_expert_dispatch(x, order)
    assert int(torch.isnan(rows).sum()) == 2 and int(torch.isinf(rows).sum()) == 80
    back = co.coll_torch_expert_combine(rows, order)
    assert bool(torch.isinf(back[3]).all()) and torch.isnan(back).nonzero().tolist() == [[5, 7]]
    assert not back[10].any()


def test_what_does_not_fit_is_refused():
    ids = torch.zeros(6, 2, dtype=torch.int64, device="cuda")
    order = co.coll_torch_expert_sort(ids, 4)
    x, rows, w = torch.zeros(6, 8, device="cuda"), torch.zeros(12, 8, device="cuda"), torch.zeros(6, 2, device="cuda")
    for call in (lambda: co.coll_torch_expert_sort(ids, 0), lambda: co.coll_torch_expert_sort(ids, 1025),
                 lambda: co.coll_torch_expert_sort(ids.view(3, 2, 2), 4), lambda: co.coll_torch_expert_sort(ids[:, :0], 4),
                 lambda: co.coll_torch_expert_dispatch(x[:5], order), lambda: co.coll_torch_expert_dispatch(x[:, :0], order),
                 lambda: co.coll_torch_expert_dispatch_grad(rows[:11], order), lambda: co.coll_torch_expert_combine(rows[:11], order, w),
                 lambda: co.coll_torch_expert_combine(rows, order, w[:5]),
                 lambda: co.coll_torch_expert_combine_grad(x[:, :7], rows, order, w),
                 lambda: co.coll_torch_expert_combine_grad(x.half(), rows, order, w),
                 lambda: co.coll_torch_expert_combine(rows, co.ExpertOrder(order.slot, order.src, order.offsets[:1]), w),
                 lambda: co.coll_torch_take_rows(x.view(2, 3, 8), ids), lambda: co.coll_torch_take_rows_grad(x, ids, 5),
                 lambda: co.coll_torch_take_rows_grad(rows, ids, -1), lambda: co.coll_torch_take_rows_grad(rows, ids, 1 << 31),
                 lambda: co.coll_torch_clip_grad_norm([x, x], 1.0), lambda: co.coll_torch_clip_grad_norm([x], 1.0, out=[x.half()]),
                 lambda: co.coll_torch_clip_grad_norm([x], 1.0, out=[x[:5]]),
                 lambda: co.coll_torch_clip_grad_norm([x, rows], 1.0, out=[x])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: co.coll_torch_expert_sort(ids.float(), 4), lambda: co.coll_torch_expert_dispatch(x.double(), order),
                 lambda: co.coll_torch_expert_combine(rows, order, w.long()), lambda: co.coll_torch_expert_combine(rows, order, w.cpu()),
                 lambda: co.coll_torch_expert_dispatch(x, co.ExpertOrder(order.slot.long(), order.src, order.offsets)),
                 lambda: co.coll_torch_take_rows(x, ids.float()), lambda: co.coll_torch_take_rows(x, ids.cpu()),
                 lambda: co.coll_torch_grad_norm([x.long()]), lambda: co.coll_torch_grad_norm([x, x.cpu()])):
        with pytest.raises(TypeError):
            call()


def test_rows_of_no_tokens():
    order = co.coll_torch_expert_sort(torch.empty(0, 4, dtype=torch.int64, device="cuda"), 9)
    x = torch.empty(0, 16, device="cuda")
    rows = co.coll_torch_expert_dispatch(x, order)
    assert rows.shape == (0, 16)
    assert co.coll_torch_expert_combine(rows, order, torch.empty(0, 4, device="cuda")).shape == (0, 16)
    assert co.coll_torch_expert_dispatch_grad(rows, order).shape == (0, 16)
    grad_rows, grad_w = co.coll_torch_expert_combine_grad(x, rows, order, torch.empty(0, 4, device="cuda"))
    assert grad_rows.shape == (0, 16) and grad_w.shape == (0, 4)


# ---- rows taken by index --------------------------------------------------------------------------------------------


def plain_row_sums(grad, index, rows):
    total = torch.zeros(rows, grad.size(1), dtype=torch.float64, device="cuda")
    terms, count = torch.zeros_like(total), torch.zeros(rows, 1, dtype=torch.float64, device="cuda")
    kept = torch.nonzero((index >= 0) & (index < rows)).reshape(-1)
    named, g = index[kept].long(), grad.double()[kept]
    total.index_add_(0, named, g)
    terms.index_add_(0, named, g.abs())
    count.index_add_(0, named, torch.ones_like(g[:, :1]))
    return total, terms, count


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 1000, 8), (5, 3, 16), (64, 64, 9), (100, 1023, 33), (1000, 1024, 128), (1000, 1025, 1),
                                        (4096, 5, 64), (4097, 70_000, 40), (30_000, 1, 24), (20_000, 2, 200), (50_000, 1_100_000, 4),
                                        (9000, 900, 1001), (3000, 40, 2048)])
def test_take_rows_and_their_gradient(n, rows, dim, dtype):
    g = gen(n + rows)
    itype = torch.int32 if n % 2 else torch.int64
    index = (torch.rand(n, device="cuda", generator=g) ** 3 * rows).long().clamp(max=rows - 1)
    if n > 4:
        index[::9] = -1
        index[1::11] = rows
    index = index.to(itype)
    table = randn(g, rows, dim, dtype=dtype)
    there = ((index >= 0) & (index < rows)).unsqueeze(1)
    want = torch.where(there, table[index.long().clamp(0, rows - 1)], torch.zeros((), dtype=dtype, device="cuda"))
    assert torch.equal(co.coll_torch_take_rows(table, index), want)
    grad = randn(g, n, dim, dtype=dtype)
    got = co.coll_torch_take_rows_grad(grad, index, rows)
    total, terms, count = plain_row_sums(grad, index, rows)
    close(got, total, terms, count)
    assert torch.equal(got, co.coll_torch_take_rows_grad(grad, index, rows))  # no two runs differ


@pytest.mark.parametrize("n,rows,dim", [
    (1024, 900, 5), (1024, 1025, 5), (1025, 5000, 3), (2048, 2048, 9), (2049, 70_001, 7), (4096, 31, 11), (4096, 100_000, 5), (4097, 4098, 5),
    (32_768, 32_768, 3), (32_769, 32_768, 5), (32_769, 200_000, 3), (33_000, 33_001, 130), (20_000, 20_000, 257), (140_000, 1000, 33),
    (140_000, 300_001, 7), (400_000, 2_000_000, 1), (700_000, 5, 12), (1_200_000, 1_100_000, 2)])
@pytest.mark.parametrize("spread", [1, 4])
def test_row_gradients_where_the_way_changes(n, rows, dim, spread):
    g = gen(n + rows + spread)
    index = (torch.rand(n, device="cuda", generator=g) ** spread * (rows + 2)).long() - 1  # -1 and rows among them
    grad = randn(g, n, dim, dtype=torch.float16 if n % 2 else torch.float32)
    got = co.coll_torch_take_rows_grad(grad, index, rows)
    total, terms, count = plain_row_sums(grad, index, rows)
    close(got, total, terms, count)
    assert torch.equal(got, co.coll_torch_take_rows_grad(grad, index.int(), rows))


@pytest.mark.parametrize("n", [50, 5000, 60_000])
@pytest.mark.parametrize("rows", [40, 100_000])
def test_row_gradients_in_runs_of_every_length(n, rows):
    """rows named 0, 1, 2, ... times, so that runs of equal indices begin and end everywhere in the pieces they are summed in"""
    times = torch.arange(n)
    index = torch.repeat_interleave(torch.arange(n), times % 101)[:n] % rows
    index = index[torch.randperm(n, generator=torch.Generator().manual_seed(n))].cuda()
    grad = whole(gen(n), n, 20)
    want = torch.zeros(rows, 20, dtype=torch.float64, device="cuda").index_add_(0, index, grad.double())
    assert torch.equal(co.coll_torch_take_rows_grad(grad, index, rows).double(), want)


def test_take_rows_moves_bits():
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (50, 30), device="cuda", generator=gen(1), dtype=torch.int64).to(torch.int32)
    index = torch.randint(0, 50, (7, 11), device="cuda", generator=gen(2))
    for dtype in DTYPES:
        table = bits.view(dtype)
        got = co.coll_torch_take_rows(table, index)
        assert got.shape == (7, 11, table.size(1))
        assert torch.equal(got.view(torch.int32).reshape(77, 30), bits[index.reshape(-1)])


def test_take_rows_of_empty_things():
    table = torch.ones(5, 8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert co.coll_torch_take_rows(table, none).shape == (0, 8)
    for rows in (0, 1, 5, 100_000):
        got = co.coll_torch_take_rows_grad(torch.empty(0, 8, device="cuda"), none, rows)
        assert got.shape == (rows, 8) and not got.any()
    nowhere = torch.full((6,), -1, dtype=torch.int64, device="cuda")
    assert not co.coll_torch_take_rows(table[:0], nowhere).any()
    assert not co.coll_torch_take_rows_grad(torch.full((6, 8), float("nan"), device="cuda"), nowhere, 9).any()
    assert co.coll_torch_take_rows_grad(torch.ones(6, 8, device="cuda"), nowhere, 0).shape == (0, 8)


@pytest.mark.parametrize("share", [0.5, 0.999])
def test_a_row_that_most_entries_name(share):
    g = gen(5)
    n, rows, dim = 120_000, 30_000, 48
    index = torch.randint(0, rows, (n,), device="cuda", generator=g)
    index[torch.rand(n, device="cuda", generator=g) < share] = 12_345
    grad = randn(g, n, dim)
    total, terms, count = plain_row_sums(grad, index, rows)
    close(co.coll_torch_take_rows_grad(grad, index, rows), total, terms, count)


def test_gradient_at_strides():
    g = gen(6)
    index = torch.randint(0, 20, (3, 50), device="cuda", generator=g)
    wide = randn(g, 3, 50, 61, dtype=torch.bfloat16)
    got = co.coll_torch_take_rows_grad(wide[..., 5:42], index, 20)
    assert torch.equal(got, co.coll_torch_take_rows_grad(wide[..., 5:42].contiguous(), index, 20))
    one = torch.ones((), device="cuda").expand(3, 50, 16)
    counts = torch.bincount(index.reshape(-1), minlength=20).float().unsqueeze(1).expand(20, 16)
    assert torch.equal(co.coll_torch_take_rows_grad(one, index, 20), counts)


# ---- gradients by autograd, against differences ---------------------------------------------------------------------


def whole(g, *shape, dtype=torch.float32):
    """small whole numbers: their products and sums are exact in float32, and differences of them too"""
    return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("masked", [0.0, 0.5])
def test_gradients_are_those_of_differences(masked):
    """the operators are linear in each argument: (f(x + d) - f(x)) . g is <gradient, d>, exactly in whole numbers"""
    g = gen(21)
    tokens, top, experts, dim = 45, 3, 6, 19
    order = co.coll_torch_expert_sort(random_ids(g, tokens, top, experts, masked), experts)

    def check(f, *args):
        args = [a.requires_grad_() for a in args]
        out = f(*args)
        weight = whole(g, *out.shape)
        grads = torch.autograd.grad(out, args, weight)
        for i, a in enumerate(args):
            d = whole(g, *a.shape)
            with torch.no_grad():
                moved = f(*[b + d if j == i else b for j, b in enumerate(args)])
            assert torch.equal(((moved - out).double() * weight.double()).sum(), (grads[i].double() * d.double()).sum())

    check(lambda x: co.coll_torch_expert_dispatch(x, order), whole(g, tokens, dim))
    check(lambda r: co.coll_torch_expert_combine(r, order), whole(g, tokens * top, dim))
    check(lambda r, w: co.coll_torch_expert_combine(r, order, w), whole(g, tokens * top, dim), whole(g, tokens, top))
    index = torch.randint(-2, 9, (6, 20), device="cuda", generator=g)
    check(lambda t: co.coll_torch_take_rows(t, index), whole(g, 8, dim))


def test_gradients_of_inputs_that_do_not_ask():
    g = gen(22)
    order = co.coll_torch_expert_sort(random_ids(g, 10, 2, 4), 4)
    rows, w = randn(g, 20, 8), torch.rand(10, 2, device="cuda", generator=g, requires_grad=True)
    assert not co.coll_torch_expert_combine(rows, order, w.detach()).requires_grad
    out = co.coll_torch_expert_combine(rows, order, w)
    out.sum().backward()
    assert w.grad.shape == w.shape and rows.grad is None
    with torch.no_grad():
        assert not co.coll_torch_expert_combine(rows, order, w).requires_grad
    r = rows.clone().requires_grad_()
    co.coll_torch_expert_combine(r, order, w.detach()).sum().backward()
    assert r.grad.shape == rows.shape


# ---- the norm over gradients ----------------------------------------------------------------------------------------


def plain_norm(grads):
    return float(np.sqrt(sum(float((t.double() ** 2).sum()) for t in grads)))


def check_norm(got, grads):
    want = plain_norm(grads)
    # one rounding to float32; the 64-bit sums of both sides are off by far less
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - want) <= (F32 * 1.001) * want, (float(got), want)


def check_clipped(got, grads, max_norm):
    norm = plain_norm(grads)
    factor = min(1.0, max_norm / (norm + 1e-6))
    for a, b in zip(got, grads):
        assert a.dtype == b.dtype and a.shape == b.shape
        want = b.double() * factor
        # the factor and the product are rounded to float32, the result to its type
        off = (a.double() - want).abs()
        assert bool((off <= want.abs() * (U[a.dtype] + 2.01 * F32 * (1 + U[a.dtype])) + TINY[a.dtype]).all())


LISTS = {
    "one": [(1, torch.float32)],
    "three types": [(1000, torch.float32), (77, torch.float16), (40_001, torch.bfloat16)],
    "pieces": [(8191, torch.float32), (8192, torch.float32), (8193, torch.float32), (16_385, torch.bfloat16), (100_003, torch.float16)],
    "empty among them": [(0, torch.float32), (5, torch.bfloat16), (0, torch.float16), (3, torch.float32)],
    "many": [(1 + 37 * i % 501, DTYPES[i % 3]) for i in range(700)],
    "large": [(3_000_017, torch.bfloat16), (1_000_003, torch.float32), (1, torch.float16)],
}


@pytest.mark.parametrize("name", sorted(LISTS))
def test_norm_and_clipping(name):
    g = gen(31)
    grads = [randn(g, n, dtype=d) for n, d in LISTS[name]]
    check_norm(co.coll_torch_grad_norm(grads), grads)
    norm = plain_norm(grads)
    for max_norm in (0.5 * norm, 2 * norm, 0.0):
        out = [torch.full_like(t, float("nan")) for t in grads]
        kept = [t.clone() for t in grads]
        check_norm(co.coll_torch_clip_grad_norm(grads, max_norm, out=out), grads)
        check_clipped(out, grads, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(kept, grads))
        again = [t.clone() for t in grads]
        co.coll_torch_clip_grad_norm(again, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(again, out))
        if max_norm > norm + 1e-3:
            assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_norm_of_more_than_the_memory_side_cache_holds():
    g = gen(35)
    grads = [randn(g, 100_000_003, dtype=torch.bfloat16), randn(g, 60_000_001), randn(g, 5)]
    out = [torch.empty_like(t) for t in grads]
    check_norm(co.coll_torch_clip_grad_norm(grads, 3.0, out=out), grads)
    check_clipped(out, grads, 3.0)
    before = [t.clone() for t in grads]
    co.coll_torch_clip_grad_norm(grads, 3.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))
    check_clipped(grads, before, 3.0)


@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_norm_at_odd_addresses(shift):
    g = gen(32)
    for dtype in DTYPES:
        buffer = randn(g, 50_000, dtype=dtype)
        before = buffer.clone()
        part = buffer[shift:shift + 33_333]
        check_norm(co.coll_torch_grad_norm([part]), [part])
        co.coll_torch_clip_grad_norm([part], 1.0)
        check_clipped([part], [before[shift:shift + 33_333]], 1.0)
        assert torch.equal(buffer[:shift], before[:shift]) and torch.equal(buffer[shift + 33_333:], before[shift + 33_333:])


def test_norm_of_large_and_tiny_gradients():
    for value in (1e30, 3e-30, 1.17e-38):
        grads = [torch.full((1000,), value, device="cuda"), torch.full((24,), -value, device="cuda", dtype=torch.bfloat16)]
        check_norm(co.coll_torch_grad_norm(grads), grads)
    big = [torch.full((1 << 20,), 3e38, device="cuda")]  # the norm is beyond float32, the sum of squares is not beyond 64 bits
    out = [torch.empty_like(big[0])]
    assert float(co.coll_torch_clip_grad_norm(big, 1.0, out=out)) == float("inf")
    check_clipped(out, big, 1.0)


def test_norm_that_is_not_finite():
    g = gen(33)
    grads = [randn(g, 100), randn(g, 300, dtype=torch.bfloat16)]
    grads[1][7] = float("inf")
    out = [torch.empty_like(t) for t in grads]
    assert float(co.coll_torch_clip_grad_norm(grads, 1.0, out=out)) == float("inf")
    assert not out[0].any() and torch.isnan(out[1]).nonzero().tolist() == [[7]] and int(out[1].nan_to_num().count_nonzero()) == 0
    grads[0][3] = float("nan")
    assert torch.isnan(co.coll_torch_clip_grad_norm(grads, 1.0, out=out))
    assert all(bool(torch.isnan(t).all()) for t in out)


def test_clipping_counts_as_a_change():
    """what autograd has saved of a tensor that is scaled in place, or written to, is stale"""
    x, to = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda")
    y = x * 2
    loss = (y * y).sum()
    co.coll_torch_clip_grad_norm([y.detach()], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = to._version
    co.coll_torch_clip_grad_norm([x.detach()], 1.0, out=[to])
    assert to._version > before


def test_gradients_from_a_generator():
    g = gen(35)
    grads = [randn(g, 50), randn(g, 7, 3, dtype=torch.bfloat16)]
    before = [t.clone() for t in grads]
    check_norm(co.coll_torch_grad_norm(t for t in grads), before)
    check_norm(co.coll_torch_clip_grad_norm((t for t in grads), 0.5), before)
    check_clipped(grads, before, 0.5)
    out = [torch.empty_like(t) for t in grads]
    co.coll_torch_clip_grad_norm((t for t in before), 0.25, out=(t for t in out))
    check_clipped(out, before, 0.25)


def test_gradients_that_share_memory_are_refused():
    g = gen(36)
    a, b = randn(g, 64), randn(g, 64)
    before = a.clone()
    free = torch.empty(256, device="cuda")
    for grads, out in [([a[:40], a[39:]], None), ([b, a[8:16], a], None),       # scaled in place, one inside another
                       ([a, b], [free[:64], free[63:127]]),                     # written to overlapping places
                       ([a, b], [b, free[:64]]), ([a[:32], a[32:]], [a[16:48], free[:32]]),  # another's, or its own shifted
                       ([a[:32]], [a[16:48]])]:
        with pytest.raises(ValueError, match="same place"):
            co.coll_torch_clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(a, before)
    # side by side, read twice, and into its own place
    whole = torch.cat([a, b])
    co.coll_torch_clip_grad_norm([a[:31], b, a[31:]], 0.5)
    check_clipped([torch.cat([a, b])], [whole], 0.5)
    co.coll_torch_clip_grad_norm([b, b], 0.25, out=[free[:64], free[64:128]])
    check_clipped([free[:128]], [torch.cat([b, b])], 0.25)
    before = [b.clone(), a.clone()]
    co.coll_torch_clip_grad_norm([b, a], 0.125, out=[b, free[:64]])
    check_clipped([b, free[:64]], before, 0.125)


def test_clipping_without_a_limit():
    g = gen(37)
    for bad in (None, float("inf"), float("nan")):
        grads = [randn(g, 90), randn(g, 30, dtype=torch.float16)]
        if bad is not None:
            grads[0][4] = bad
        before = [t.clone() for t in grads]
        out = [torch.empty_like(t) for t in grads]
        for to in (out, None):
            norm = co.coll_torch_clip_grad_norm(grads, float("inf"), out=to)
            assert bool(torch.isfinite(norm)) == (bad is None)
        for t, u, v in zip(grads, out, before):
            assert torch.equal(t.nan_to_num(7.0), v.nan_to_num(7.0)) and torch.equal(u.nan_to_num(7.0), v.nan_to_num(7.0))


def test_tensors_that_torch_holds_negated():
    g = gen(38)
    part = torch.complex(randn(g, 24, 1), randn(g, 24, 1)).conj().imag  # rows of one element, two apart, negated when read
    assert part.is_neg()
    index = torch.arange(24, device="cuda")
    assert torch.equal(co.coll_torch_take_rows(part, index), part.resolve_neg())
    one = part[:1, 0]
    out = [torch.empty(1, device="cuda")]
    co.coll_torch_clip_grad_norm([one], 1e9, out=out)
    assert torch.equal(out[0], one.resolve_neg())
    with pytest.raises(ValueError, match="in place"):
        co.coll_torch_clip_grad_norm([one], 1.0)


def test_norm_of_other_layouts():
    g = gen(34)
    a, b = randn(g, 40, 30), randn(g, 6, 5, 4, dtype=torch.float16)
    turned = [a.t(), b.permute(2, 0, 1)]
    check_norm(co.coll_torch_grad_norm(turned + [a[:, ::2], None]), turned + [a[:, ::2]])
    check_norm(co.coll_torch_grad_norm(a), [a])
    before = [t.clone() for t in turned]
    co.coll_torch_clip_grad_norm(turned, 0.5)
    check_clipped(turned, before, 0.5)
    with pytest.raises(ValueError, match="in place"):
        co.coll_torch_clip_grad_norm([a[:, ::2]], 1.0)
    out = torch.empty(30, 40, device="cuda")
    co.coll_torch_clip_grad_norm([a.t(), None], 0.25, out=[out, None])
    check_clipped([out], [a.t()], 0.25)


# ---- streams, graphs, sizes, a step as a whole ----------------------------------------------------------------------


def every_operator(x, ids, w, index, experts, rows):
    order = co.coll_torch_expert_sort(ids, experts)
    sent = co.coll_torch_expert_dispatch(x, order)
    back = co.coll_torch_expert_combine(sent, order, w)
    grad_rows, grad_w = co.coll_torch_expert_combine_grad(back, sent, order, w)
    grad_x = co.coll_torch_expert_dispatch_grad(grad_rows, order)
    taken = co.coll_torch_take_rows(x, index)
    grad_t = co.coll_torch_take_rows_grad(taken, index, rows)
    clipped = [torch.empty_like(grad_t), torch.empty_like(grad_x)]
    norm = co.coll_torch_clip_grad_norm([grad_t, grad_x], 1.0, out=clipped)
    return [order.slot, order.src, order.offsets, sent, back, grad_rows, grad_w, grad_x, taken, grad_t, norm] + clipped


def inputs_for(seed, tokens, top, experts, dim, dtype):
    g = gen(seed)
    return [randn(g, tokens, dim, dtype=dtype), random_ids(g, tokens, top, experts, 0.1), torch.rand(tokens, top, device="cuda", generator=g),
            torch.randint(-1, tokens, (3 * tokens,), device="cuda", generator=g)]


@pytest.mark.parametrize("tokens", [5, 700, 6000])
def test_operators_replayed_from_two_graphs_as_eager(tokens):
    """two graphs of the same calls, captured one after the other, replayed in turn on new inputs with eager calls between"""
    args = (6, 2, 8, 72, torch.bfloat16)
    held, graphs = [], []
    for k in range(2):
        static = inputs_for(100 + k, tokens, *args[1:])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            every_operator(*static, 8, tokens)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = every_operator(*static, 8, tokens)
        graphs.append(graph)
        held.append((static, outs))
    for turn in range(4):
        for k in (0, 1):
            static, outs = held[k]
            fresh = inputs_for(200 + 2 * turn + k, tokens, *args[1:])
            for to, t in zip(static, fresh):
                to.copy_(t)
            graphs[k].replay()
            eager = every_operator(*fresh, 8, tokens)
            torch.cuda.synchronize()
            for a, b in zip(outs, eager):
                assert torch.equal(a, b)


def test_a_backward_pass_replayed():
    """forward and backward through autograd in a graph, replayed on new inputs with eager steps between"""
    tokens, top, experts, dim = 300, 2, 8, 40
    g = gen(70)
    table = randn(g, 500, dim, dtype=torch.bfloat16)
    static = [torch.empty(tokens, dtype=torch.int64, device="cuda"), torch.empty(tokens, top, dtype=torch.int64, device="cuda"),
              torch.empty(tokens, top, device="cuda", requires_grad=True), torch.empty(tokens, dim, dtype=torch.bfloat16, device="cuda")]

    def fresh(seed):
        f = gen(seed)
        return [torch.randint(-1, 500, (tokens,), device="cuda", generator=f), random_ids(f, tokens, top, experts, 0.1),
                torch.rand(tokens, top, device="cuda", generator=f).requires_grad_(), randn(f, tokens, dim, dtype=torch.bfloat16)]

    def step(ids, chosen, w, grad):
        leaf = table.detach().requires_grad_()
        order = co.coll_torch_expert_sort(chosen, experts)
        rows = co.coll_torch_expert_dispatch(co.coll_torch_take_rows(leaf, ids), order)
        out = co.coll_torch_expert_combine(rows, order, w)
        return [out.detach()] + list(torch.autograd.grad(out, [leaf, w], grad))

    def fill(seed):
        with torch.no_grad():
            for to, t in zip(static, fresh(seed)):
                to.copy_(t)

    fill(71)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for seed in range(72, 76):
        fill(seed)
        graph.replay()
        eager = step(*fresh(seed))
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


def test_the_first_calls_of_a_process_captured():
    """the kernels are loaded with their first call: that may be one that is recorded"""
    code = """
import sys
import torch
sys.path.insert(0, "ugache_amd")
import collcache.torch as co
x = torch.randn(64, 32, device="cuda")
ids = torch.randint(0, 4, (64, 2), device="cuda")
index = torch.randint(0, 64, (100,), device="cuda")
def step():
    order = co.coll_torch_expert_sort(ids, 4)
    rows = co.coll_torch_expert_dispatch(x, order)
    out = co.coll_torch_expert_combine(rows, order)
    grad, _ = co.coll_torch_expert_combine_grad(out, rows, order)
    taken = co.coll_torch_take_rows_grad(co.coll_torch_take_rows(x, index), index, 64)
    clipped = torch.empty_like(taken)
    return [out, grad, taken, co.coll_torch_clip_grad_norm([taken], 1.0, out=[clipped]), clipped]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))
print("replayed", flush=True)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "replayed" in done.stdout, done.stderr[-2000:]


def test_operators_on_two_streams_at_once():
    cases = [inputs_for(40 + k, 3000, 4, 16, 96, torch.float16) for k in range(2)]
    want = [every_operator(*c, 16, 3000) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(every_operator(*cases[k], 16, 3000))
    torch.cuda.synchronize()
    for k in range(2):
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))


def test_rows_beyond_32_bits_of_elements():
    dim, rows = 2056, (1 << 31) // 2056 + 5000
    table = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    g = gen(50)
    last = randn(g, 4000, dim, dtype=torch.bfloat16)
    table[-4000:] = last
    index = torch.randint(rows - 4000, rows, (500,), device="cuda", generator=g)
    assert torch.equal(co.coll_torch_take_rows(table, index), last[index - (rows - 4000)])
    table[:-4000] = 0
    # the sums of a table that large, and the norm over it
    grad = randn(g, 500, dim, dtype=torch.bfloat16)
    got = co.coll_torch_take_rows_grad(grad, index, rows)
    total, terms, count = plain_row_sums(grad, index - (rows - 4000), 4000)
    close(got[-4000:], total, terms, count)
    assert not got[:1000].any() and not got[rows // 2:rows // 2 + 1000].any()
    check_norm(co.coll_torch_grad_norm([got]), [got[-4000:]])
    del got
    # every row once, as assignments of one token each
    order = co.coll_torch_expert_sort(torch.zeros(rows, dtype=torch.int32, device="cuda"), 1)
    sent = co.coll_torch_expert_dispatch(table, order)
    assert torch.equal(sent[-4000:], last)
    back = co.coll_torch_expert_combine(sent, order)
    assert torch.equal(back[-4000:], last) and not back[:1000].any()


def test_a_layer_of_experts_trained():
    """embedding -> router -> experts -> back -> loss, as a model would use the operators together, with the gradients of every
    parameter against the same layer computed densely in 64 bits"""
    g = gen(60)
    vocabulary, tokens, top, experts, dim = 50, 90, 2, 5, 24
    ids = torch.randint(0, vocabulary, (tokens,), device="cuda", generator=g)
    ids[::13] = -1  # padding
    names = ["table", "router", "expert"]
    start = {"table": randn(g, vocabulary, dim), "router": randn(g, dim, experts), "expert": randn(g, experts, dim, dim) * 0.2}
    p = {k: v.clone().requires_grad_() for k, v in start.items()}
    x = co.coll_torch_take_rows(p["table"], ids)
    w, chosen = torch.topk(torch.softmax(x @ p["router"], 1), top, dim=1)
    chosen = torch.where((ids >= 0).unsqueeze(1), chosen, -1)
    order = co.coll_torch_expert_sort(chosen, experts)
    rows = co.coll_torch_expert_dispatch(x, order)
    bounds = order.offsets.tolist()
    made = torch.cat([rows[bounds[e]:bounds[e + 1]] @ p["expert"][e] for e in range(experts)] + [rows[bounds[-1]:]])
    out = co.coll_torch_expert_combine(made, order, w)
    target = randn(g, tokens, dim)
    ((out - target) ** 2).sum().backward()

    q = {k: v.double().requires_grad_() for k, v in start.items()}
    keep = (ids >= 0).double().unsqueeze(1)
    xd = q["table"][ids.clamp(min=0)] * keep
    probs = torch.softmax(xd @ q["router"], 1)
    gate = torch.zeros_like(probs).scatter(1, chosen.clamp(min=0), 1.0) * keep * probs
    outd = sum(gate[:, e:e + 1] * (xd @ q["expert"][e]) for e in range(experts))
    ((outd - target.double()) ** 2).sum().backward()
    for k in names:
        # float32 throughout, a few hundred roundings behind one another: 2^-12 of the largest gradient
        assert float((p[k].grad.double() - q[k].grad).abs().max()) <= 2.0 ** -12 * float(q[k].grad.abs().max()), k
    grads = [p[k].grad for k in names]
    before = [t.clone() for t in grads]
    norm = co.coll_torch_clip_grad_norm(grads, 1.0)
    check_norm(norm, before)
    check_clipped(grads, before, 1.0)


def test_the_gradient_of_distinct_keys_looked_up():
    """the distinct keys of a batch from the cache, spread over its positions, and the gradients of the distinct rows"""
    n_item, dim = 5000, 32
    co.config({"cache_percentage": 0.3, "_cache_policy": co.kCollCacheAsymmLink, "num_device": 1, "num_global_step_per_epoch": 100,
               "num_epoch": 1, "num_total_item": n_item, "omp_thread_num": 4})
    try:
        co.coll_cache_record_init(0)
        keys = (torch.rand(3000, generator=torch.Generator().manual_seed(1)) ** 2 * n_item).long()
        co.coll_torch_record(0, keys)
        table = co.coll_torch_create_emb_shm(0, n_item, dim, torch.float32)
        table.copy_(torch.randn(n_item, dim, generator=torch.Generator().manual_seed(2)))
        co.coll_torch_init_t(0, 0, table, 0.3)
        rows, inverse = co.coll_torch_lookup_unique(0, keys.cuda())
        rows = rows.clone().requires_grad_()
        out = co.coll_torch_take_rows(rows, inverse)
        assert torch.equal(out.detach().cpu(), table[keys])
        grad = randn(gen(61), *out.shape)
        out.backward(grad)
        total, terms, count = plain_row_sums(grad, inverse, rows.size(0))
        close(rows.grad, total, terms, count)
        check_norm(co.coll_torch_grad_norm([rows.grad]), [rows.grad])
    finally:
        co.coll_torch_shutdown()
