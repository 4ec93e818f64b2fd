"""Searches of rows in 4 bits where the candidates are hard to tell: a count far
above the sequence's length, rows without a finite distance, and rows that
fp32 sums cannot order.

Expected neighbours come from sums in 64 bits; where rows lie close together,
of values with so few bits that the sums are exact there, so that ties are ties
and go to the lowest index.  Distances are rounded once to 32 bits: 2^-24
relative.
"""
import math

import pytest

from test_gpu_row_store import plain_search, randn, random_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def check_search(torch, got, values, index, q, k, metric):
    """The k nearest of `values`, whose positions are `index`; the rest is padding."""
    near, far = got
    want, distance, _ = plain_search(torch, values, q, k, metric)
    want = torch.where(want >= 0, index[want.clamp(min=0)] if len(index) else want, want)
    assert torch.equal(near, want)
    fine = want >= 0
    off = (far.double() - distance).abs()[fine]
    assert (off <= 2.0 ** -24 * 1.01 * distance.abs()[fine] + 2.0 ** -40).all()
    assert (far[~fine] == (math.inf if metric == 0 else -math.inf)).all()


# ------------------------------------------------- a count above the length
def long_store(torch, engine, n, room, page_rows, zeros, scale="float16"):
    """A sequence of n rows of 64 values in a store of `room` rows."""
    rows, values = random_rows(torch, engine, 100 + n, n, 64, 32, zeros, getattr(torch, scale), page_rows)
    total = -(-room // page_rows) + 5
    held, old = [], rows.pages
    for t in old.pools:
        p = torch.zeros(total, *t.shape[1:], dtype=t.dtype, device="cuda")
        p[:t.shape[0]] = t
        held.append(p)
    pages = engine.Pages.empty(held, 2, total)
    pages.table[1, :old.table.shape[1]] = old.table[1]
    pages.refs[:len(old.refs)] = old.refs
    pages.rows[1] = n
    held.insert(2, None) if not zeros else None
    return engine.Q4Rows(held[0], held[1], 64, 32, held[2], held[3], pages), values


@pytest.mark.parametrize("n", [1, 20, 128, 800])
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("page_rows", [48, 256])
def test_count_far_above_the_length(torch, engine, n, metric, page_rows):
    rows, values = long_store(torch, engine, n, 100000, page_rows, metric == 1)
    q = randn(torch, 6, 3, 64)
    index = torch.arange(n, device="cuda")
    for count in (900, 3200, 100000):
        for k in (1, 10, 256):
            check_search(torch, rows.search(q, k, metric=metric, seq=1, count=count), values[:count],
                         index[:count], q, k, metric)


@pytest.mark.parametrize("metric", [0, 1])
def test_few_groups_with_keys(torch, engine, metric):
    """Most rows' pages are missing, or most rows' scales are NaN."""
    n, page_rows = 20000, 64
    rows, values = random_rows(torch, engine, 31, n, 64, 32, True, torch.float16, page_rows)
    q = randn(torch, 6, 5, 64)
    gone = torch.ones(n // page_rows + 1, dtype=torch.bool, device="cuda")
    gone[[3, 100, 311]] = False
    rows.pages.table[1, :len(gone)][gone] = -1
    index = torch.arange(n, device="cuda")
    index = index[~gone[index // page_rows]]
    for k in (1, 10, 100, 256):
        check_search(torch, rows.search(q, k, metric=metric, seq=1, count=n), values[index], index, q, k, metric)
    rows, values = random_rows(torch, engine, 32, n, 64, 32, False, torch.float16)
    keep = torch.zeros(n, dtype=torch.bool, device="cuda")
    keep[torch.cat((torch.arange(17, 90), torch.tensor([5000]), torch.arange(19001, 19040)))] = True
    rows.scales[~keep] = float("nan")
    rows.norms[~keep] = float("nan")
    index = keep.nonzero().flatten()
    for k in (1, 10, 100, 256):
        check_search(torch, rows.search(q, k, metric=metric), values[index], index, q, k, metric)


def test_count_above_the_length_in_a_graph(torch, engine):
    """A captured search of a sequence whose length changes between replays."""
    rows, values = long_store(torch, engine, 800, 50000, 64, False)
    q = randn(torch, 6, 4, 64)
    rows.search(q, 20, seq=1, count=50000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rows.search(q, 20, seq=1, count=50000)
    for n in (800, 37, 0, 260):
        rows.pages.rows[1] = n
        graph.replay()
        check_search(torch, got, values[:n], torch.arange(n, device="cuda"), q, 20, 0)


# ------------------------------------------- distances that are no finite number
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("x", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 9001])
def test_queries_that_are_not_finite(torch, engine, metric, x, dim):
    """No row is at a finite distance from them; the queries beside them find theirs."""
    rows, values = random_rows(torch, engine, 41, 3000, dim, 32, True, torch.float16)
    q = randn(torch, 6, 5, dim).to(getattr(torch, x))
    q[1, 7], q[2, dim - 1], q[3, 0] = math.inf, -math.inf, math.nan
    near, far = rows.search(q, 30, metric=metric)
    index = torch.arange(3000, device="cuda")
    check_search(torch, (near[::4], far[::4]), values, index, q[::4], 30, metric)
    assert (near[1:4] == -1).all()
    assert (far[1:4] == (math.inf if metric == 0 else -math.inf)).all()


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_that_are_not_finite(torch, engine, metric, zeros):
    """Scales of both infinities among the rows, more of them than are looked for."""
    n = 5000
    rows, values = random_rows(torch, engine, 42, n, 96, 32, zeros, torch.float16)
    odd = torch.arange(n, device="cuda") % 3 != 1
    rows.scales[odd, 1] = math.inf
    rows.scales[::6, 1] = -math.inf
    rows.norms[odd] = math.inf
    index = (~odd).nonzero().flatten()
    q = randn(torch, 6, 4, 96)
    for k in (1, 40, 256):
        check_search(torch, rows.search(q, k, metric=metric), values[index], index, q, k, metric)


def test_distances_beyond_32_bits(torch, engine):
    """Products and squares that 64 bits hold and 32 do not: such rows are no
    neighbours either, and the others keep their order."""
    n = 4000
    rows, _ = random_rows(torch, engine, 43, n, 64, 32, False, torch.float16)
    rows.scales[:] = torch.where(torch.arange(n, device="cuda")[:, None] % 4 == 0, 0.5, 2.0).half()
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = torch.zeros(2, 64, device="cuda")
    q[0, 5], q[1, 40] = 1.5e38, -2.5e38
    q[:, 9] = 1e36
    most = torch.finfo(torch.float32).max
    for b in (0, 1):
        product = values @ q[b].double()
        index = (product.abs() <= most).nonzero().flatten()
        assert 500 < len(index) < 3500
        for k in (10, 256):
            check_search(torch, rows.search(q[b:b + 1], k, metric=1), values[index], index, q[b:b + 1], k, 1)
    # squares: every distance is too large, though |row|^2 - 2 q.row is not
    near, far = rows.search(torch.full((1, 64), 3e18, device="cuda"), 10)
    assert (near == -1).all() and torch.isinf(far).all()
    # some are not: |q|^2 = 2^128, and a value above 0 takes 2^105 or more off it
    rows, _ = random_rows(torch, engine, 44, n, 64, 32, False, torch.bfloat16)
    rows.scales[:] = 2.0 ** 40
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = torch.zeros(1, 64, device="cuda")
    q[0, 3] = 2.0 ** 64
    near, far = rows.search(q, 100)
    assert torch.isfinite(far).all() and (values[near[0], 3] > 0).all()
    keep = values[:, 3] > 0
    keep[keep.nonzero().flatten()[50:]] = False
    rows.scales[~keep & (values[:, 3] > 0)] = math.nan  # 50 rows are left at finite distances
    near, far = rows.search(q, 100)
    assert torch.equal(near[0, :50].sort().values, keep.nonzero().flatten())
    assert torch.isfinite(far[0, :50]).all() and (near[0, 50:] == -1).all() and torch.isinf(far[0, 50:]).all()


# --------------------------------------------- rows that fp32 sums cannot order
def close_rows(torch, engine, seed, n, small, scale, page_rows, with_norms=True):
    """Rows that share one group of values up to 128 and differ in the other, whose
    values are up to about `small`; every sum of their products is exact in 64 bits."""
    rows, _ = random_rows(torch, engine, seed, n, 256, 128, False, getattr(torch, scale), page_rows)
    order = torch.arange(n, device="cuda")
    if page_rows:
        order = rows.pages.table[1, order // page_rows].long() * page_rows + order % page_rows
    codes, scales, norms = (t.view(-1, *t.shape[2:]) if page_rows else t
                            for t in (rows.codes, rows.scales, rows.norms))
    codes[order, :64] = codes[order[0], :64].clone()
    scales[order, 0] = 16.0
    g = torch.Generator(device="cuda").manual_seed(seed)
    scales[order, 1] = (small / 8 * (1 + torch.randint(0, 64, (n,), device="cuda", generator=g) / 64)).to(scales.dtype)
    c = torch.stack((codes[order] & 15, codes[order] >> 4), -1).flatten(1).double() - 8
    values = c * scales[order].double().repeat_interleave(128, 1)
    norms[order] = values.square().sum(1).float()
    if not with_norms:
        rows = engine.Q4Rows(rows.codes, rows.scales, 256, 128, None, None, rows.pages)
    return rows, values


@pytest.mark.parametrize("n,k,batch,small,x,scale,page_rows", [
    (4000, 8, 4, 2.0 ** -8, "float32", "float16", 0),
    (4000, 8, 16, 2.0 ** -8, "float16", "bfloat16", 64),
    (4000, 100, 1, 2.0 ** -5, "float16", "float16", 0),
    (4000, 1, 3, 2.0 ** -8, "bfloat16", "float16", 48),
    (70000, 10, 5, 2.0 ** -4, "float32", "float16", 0),
    (70000, 256, 2, 2.0 ** -8, "bfloat16", "float16", 0),
    (300, 256, 2, 2.0 ** -8, "float32", "float16", 0),
])
@pytest.mark.parametrize("metric", [0, 1])
def test_rows_with_a_shared_offset(torch, engine, n, k, batch, small, x, scale, page_rows, metric):
    rows, values = close_rows(torch, engine, 50 + k, n, small, scale, page_rows, with_norms=metric == 0)
    # near the shared values, and apart from them by whole numbers
    q = values[torch.arange(batch) * 17].clone()
    q[:, :128] += torch.randint(-2, 3, (batch, 128), device="cuda",
                                generator=torch.Generator(device="cuda").manual_seed(k)) * 16.0
    q[:, 128:] = (randn(torch, 8, batch, 128).double() * small * 4).mul(2.0 ** 12).round().mul(2.0 ** -12)
    q = q.to(getattr(torch, x))
    got = rows.search(q, k, metric=metric, seq=1 if page_rows else None, count=n)
    check_search(torch, got, values, torch.arange(n, device="cuda"), q, k, metric)


@pytest.mark.parametrize("metric", [0, 1])
def test_near_copies_of_one_row(torch, engine, metric):
    """20,000 copies of a row, one value of some changed a little: what is exact in
    64 bits decides, then the index."""
    n = 20000
    rows, _ = random_rows(torch, engine, 61, n, 256, 128, False, torch.float16)
    rows.codes[:] = rows.codes[11].clone()
    rows.scales[:, 0] = 8.0
    rows.scales[:, 1] = 2.0 ** -9
    g = torch.Generator(device="cuda").manual_seed(3)
    changed = torch.randperm(n, device="cuda", generator=g)[:700]
    rows.codes[changed, 100] = torch.randint(0, 256, (700,), device="cuda", generator=g, dtype=torch.uint8)
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = values[:2].float()
    q[:, 200:202] += torch.tensor([[0.25, -0.5], [-0.125, 1.0]], device="cuda")
    for k in (5, 200):
        check_search(torch, rows.search(q, k, metric=metric), values, torch.arange(n, device="cuda"), q, k, metric)


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("batch", [1, 16])
def test_one_row_far_larger_than_the_rest(torch, engine, metric, batch):
    """It does not make the others' order uncertain, nor lose them."""
    n = 30000
    rows, _ = random_rows(torch, engine, 62, n, 512, 64, True, torch.bfloat16)
    rows.scales[[77, 20001]] *= 1e6
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = randn(torch, 6, batch, 512)
    check_search(torch, rows.search(q, 50, metric=metric), values, torch.arange(n, device="cuda"), q, 50, metric)


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("power", [-60, -64, -68])
def test_rows_whose_squares_are_subnormal(torch, engine, metric, power):
    """Squares near the smallest numbers of 32 bits: the order is that of 64 bits all
    the same."""
    n = 3000
    rows, _ = random_rows(torch, engine, 63, n, 256, 128, False, torch.bfloat16)
    j = torch.randint(0, 64, (n, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    rows.scales[:] = ((1 + j / 64) * 2.0 ** power).bfloat16()
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = (values[:3] * 1.25).float()
    near, _ = rows.search(q, 60, metric=metric)
    want, _, _ = plain_search(torch, values, q, 60, metric)
    assert torch.equal(near, want)


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("x", ["float32", "float16"])
def test_near_copies_of_wide_rows(torch, engine, metric, x):
    """Rows wider than a query that is kept on chip, more queries than one pass takes."""
    n, dim = 900, 8300
    rows, _ = random_rows(torch, engine, 64, n, dim, 128, False, torch.float16)
    rows.codes[:] = rows.codes[0].clone()
    rows.scales[:] = 2.0 ** -9
    rows.scales[:, 0] = 16.0
    g = torch.Generator(device="cuda").manual_seed(3)
    rows.codes[:, 4100:4140] = torch.randint(0, 256, (n, 40), device="cuda", generator=g, dtype=torch.uint8)
    rows.codes[300:500] = rows.codes[7].clone()
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = values[torch.arange(18) * 50].to(getattr(torch, x))
    q[:, 8200:8290] += (torch.randint(-9, 10, (18, 90), device="cuda", generator=g) * 2.0 ** -9).to(q.dtype)
    for k in (1, 30):
        check_search(torch, rows.search(q, k, metric=metric), values, torch.arange(n, device="cuda"), q, k, metric)


def test_easy_and_hard_queries_of_one_graph(torch, engine):
    """A captured search whose queries need more rows scored in one replay than in another."""
    n = 5000
    rows, values = close_rows(torch, engine, 65, n, 2.0 ** -8, "float16", 64)
    index = torch.arange(n, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)

    def queries(hard):
        q = values[torch.arange(3) * 100].clone()
        q[:, 128:] = torch.randint(-9, 10, (3, 128), device="cuda", generator=g) * 2.0 ** (-9 if hard else 7)
        return q.float()

    q = queries(True)
    rows.search(q, 20, seq=1, count=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rows.search(q, 20, seq=1, count=n)
    for hard in (True, False, True, False):
        q.copy_(queries(hard))
        graph.replay()
        check_search(torch, got, values, index, q, 20, 0)


def test_rows_whose_norms_are_no_pool(torch, engine):
    """A fork would leave such norms behind, and searches by L2 with them."""
    rows, _ = random_rows(torch, engine, 71, 100, 64, 32, False, torch.float16, 16)
    bare = engine.Pages(rows.pages.table, rows.pages.rows, rows.pages.refs, [rows.codes, rows.scales])
    engine.Q4Rows(rows.codes, rows.scales, 64, 32, pages=bare)
    with pytest.raises(ValueError, match="norms"):
        engine.Q4Rows(rows.codes, rows.scales, 64, 32, norms=rows.norms, pages=bare)
    with pytest.raises(ValueError, match="scales"):
        engine.Q4Rows(rows.codes, rows.scales.clone(), 64, 32, norms=rows.norms, pages=rows.pages)
