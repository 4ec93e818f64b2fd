"""The row store on the GPU: rows in 4 bits (pack, read, products, search) and
pages of rows (grow, free, copy, fork, compact), against plain forms in 64 bits
and a plain-Python store.

Tolerances.  A value has at most 16 significant bits and is exact in fp32, as a
product with a 16-bit number is; a product with an fp32 number is rounded, or
split exactly.  A sum of n terms in fp32, in any order, each step rounded or
cut, is off by at most n * 2^-23 of the sum of magnitudes; the last rounding to
a type adds half its step.  Packed codes and scales, pages and searches'
neighbours have to be equal.
"""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = "float32", "float16", "bfloat16"


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def randn(torch, seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def nearest(torch, q, t):
    """q / t to the nearest whole number, ties to even; 0 where t is of no use."""
    ok = (t > 0) & torch.isfinite(t)
    return torch.where(ok, q / torch.where(ok, t, 1.0), 0.0).round()


def plain_pack(torch, x, group, zero_points, scale_dtype):
    """(codes one to a value, scales, zeros, values, all but scales in float64)."""
    n, dim = x.shape
    groups = -(-dim // group)
    v = torch.nn.functional.pad(x.double(), (0, groups * group - dim)).view(n, groups, group)
    if zero_points:
        low = v.amin(-1).clamp(max=0.0)
        high = v.amax(-1).clamp(min=0.0)
        wide, over = (high - low).float().double(), 15.0
    else:
        wide, over = v.abs().amax(-1), 7.0
    s = (wide / over).float().to(scale_dtype)
    sd = s.double()
    z = nearest(torch, -low, sd).clamp(0, 15) if zero_points else torch.full_like(sd, 8.0)
    c = (nearest(torch, v, sd[..., None].expand_as(v)) + z[..., None]).clamp(0, 15)
    values = ((c - z[..., None]) * sd[..., None]).view(n, -1)[:, :dim]
    return c.view(n, -1)[:, :dim], s, z, values


def unpack(torch, codes, dim):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :dim]


def random_rows(torch, engine, seed, n, dim, group, zeros, scale_dtype, page_rows=0):
    """Q4Rows with random codes, scales and zero points, and their values in float64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width, groups = 16 * -(-dim // 32), -(-dim // group)

    def ints(high, *shape):
        return torch.randint(0, high, shape, dtype=torch.uint8, device="cuda", generator=g)

    codes = ints(256, n, width)  # what lies behind the last value counts for nothing
    scales = (randn(torch, seed + 1, n, groups) * 0.05).to(scale_dtype)  # negative ones too
    z = ints(16, n, groups) if zeros else None
    zz = z.double() if zeros else torch.full((n, groups), 8.0, dtype=torch.float64, device="cuda")
    values = (unpack(torch, codes, dim).double() - zz.repeat_interleave(group, 1)[:, :dim]) * \
        scales.double().repeat_interleave(group, 1)[:, :dim]
    norms = values.square().sum(1).float()
    if not page_rows:
        return engine.Q4Rows(codes, scales, dim, group, z, norms), values
    need = -(-n // page_rows)
    order = torch.randperm(need + 3, device="cuda", generator=g)[:need]
    at = torch.arange(n, device="cuda")
    place = order[at // page_rows] * page_rows + at % page_rows

    def pool(t):
        if t is None:
            return None
        p = ints(256, (need + 3) * page_rows * (t[0].numel() or 1) * t.element_size()).view(t.dtype)
        p = p.view((need + 3) * page_rows, *t.shape[1:])
        p[place] = t
        return p.view(need + 3, page_rows, *t.shape[1:])

    held = [pool(t) for t in (codes, scales, z, norms)]
    pages = engine.Pages.empty([t for t in held if t is not None], 3, need + 2)
    pages.table[1, :need] = order.int()
    pages.refs[order] = 1
    pages.rows[1] = n
    return engine.Q4Rows(held[0], held[1], dim, group, held[2], held[3], pages), values


def check_products(torch, got, x, values, dtype):
    want = x.double() @ values.T
    size = x.double().abs() @ values.abs().T
    n = values.shape[1]
    bound = (n + 8) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + torch.finfo(dtype).tiny
    assert got.dtype == dtype and got.shape == want.shape
    over = want.abs() > torch.finfo(dtype).max * 0.999
    off = (got.double() - want).abs()
    bad = (off > bound) & ~over
    assert not bad.any(), (off - bound)[bad].max()


# ---------------------------------------------------------------- products
@pytest.mark.parametrize("n,dim,batch,group,x,out,zeros,scale,page_rows", [
    (1, 1, 1, 32, F32, F32, False, F16, 0),
    (5, 31, 1, 32, F16, F32, True, F16, 0),
    (17, 33, 2, 64, BF16, BF16, False, BF16, 0),
    (16, 128, 1, 128, F16, F16, True, F16, 0),
    (1000, 128, 1, 32, F16, F32, False, F16, 0),
    (1003, 1000, 3, 32, F32, F32, True, F16, 0),
    (1003, 1000, 3, 64, F32, BF16, True, BF16, 37),
    (777, 1000, 8, 128, F16, F16, False, F16, 100),
    (4096, 1024, 1, 64, F32, F32, False, F16, 0),
    (4096, 4096, 1, 128, BF16, BF16, True, F16, 0),
    (300, 4095, 5, 32, BF16, F32, False, F16, 1),
    (300, 2049, 16, 64, F32, F32, True, F16, 64),
    (2500, 1024, 16, 32, F16, F32, True, F16, 128),
    (2500, 960, 17, 32, F16, F32, False, F16, 128),
    (2500, 960, 33, 128, BF16, F32, True, F16, 48),
    (129, 200, 100, 64, F32, F32, False, F16, 16),
    (70, 20000, 16, 128, F32, F32, True, F16, 0),
    (70, 14336, 9, 32, F16, F32, False, F16, 0),
    (33, 65536, 2, 64, BF16, F32, False, F16, 0),
    (33, 65535, 7, 128, F32, F32, True, F16, 0),
    (40000, 96, 4, 32, F16, F32, True, F16, 0),
    (40000, 160, 12, 64, F32, F32, False, F16, 256),
])
def test_products(torch, engine, n, dim, batch, group, x, out, zeros, scale, page_rows):
    rows, values = random_rows(torch, engine, n + dim, n, dim, group, zeros, getattr(torch, scale), page_rows)
    v = randn(torch, 5, batch, dim).to(getattr(torch, x))
    got = rows.products(v, seq=1 if page_rows else None, count=n, dtype=getattr(torch, out))
    check_products(torch, got, v, values, getattr(torch, out))
    # the same call gives the same bits, alone or among others of the batch
    again = rows.products(v, seq=1 if page_rows else None, count=n, dtype=getattr(torch, out))
    assert torch.equal(got, again)


def test_products_of_one_vector_some_rows_and_strides(torch, engine):
    rows, values = random_rows(torch, engine, 1, 200, 100, 32, True, torch.float16)
    v = randn(torch, 2, 7, 100)
    assert rows.products(v[0]).shape == (200,)
    check_products(torch, rows.products(v[0])[None], v[:1], values, torch.float32)
    check_products(torch, rows.products(v, count=77), v, values[:77], torch.float32)
    assert rows.products(v, count=0).shape == (7, 0) and rows.products(v[:0]).shape == (0, 200)
    wide = randn(torch, 3, 7, 131).half()
    out = torch.full((7, 210), 9.0, device="cuda")
    got = rows.products(wide[:, 3:103], out=out[:, 5:205])  # odd offsets: 2-byte alignment
    check_products(torch, got, wide[:, 3:103], values, torch.float32)
    assert (out[:, :5] == 9).all() and (out[:, 205:] == 9).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_products_far_numbers(torch, engine, dtype):
    """Infinities and NaN in x reach their own vector alone; the largest and the
    smallest numbers of the type are multiplied as they are."""
    dt = getattr(torch, dtype)
    rows, values = random_rows(torch, engine, 9, 100, 70, 32, True, torch.float16)
    v = randn(torch, 4, 6, 70).to(dt)
    v[1, 3], v[2, 5] = float("inf"), float("nan")
    v[3] = torch.finfo(dt).max * 2.0 ** -14 * torch.sign(v[3])
    v[4] = torch.finfo(dt).tiny * 1024 * torch.sign(v[4])
    got = rows.products(v)
    for b in (0, 3, 4, 5):
        check_products(torch, got[b:b + 1], v[b:b + 1], values, torch.float32)
    want = v[1].double() * values
    want = torch.where(torch.isnan(want).any(1), float("nan"), want.sum(1))
    assert torch.equal(torch.isnan(got[1]), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.equal(got[1][fine].double(), want[fine])
    assert torch.isnan(got[2]).all()


def test_products_of_rows_with_nan_scales(torch, engine):
    rows, values = random_rows(torch, engine, 11, 64, 200, 64, False, torch.float16)
    rows.scales[7, 2], rows.scales[40, 0] = float("nan"), float("inf")
    v = randn(torch, 4, 3, 200)
    got = rows.products(v)
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    keep[[7, 40]] = False
    check_products(torch, got[:, keep], v, values[keep], torch.float32)
    assert torch.isnan(got[:, 7]).all() and not torch.isfinite(got[:, 40]).any()


def test_products_beyond_the_length_and_without_pages(torch, engine):
    rows, values = random_rows(torch, engine, 12, 150, 96, 32, False, torch.float16, page_rows=32)
    v = randn(torch, 4, 3, 96)
    got = rows.products(v, seq=1, count=180)
    check_products(torch, got[:, :150], v, values, torch.float32)
    assert (got[:, 150:] == 0).all()
    assert (rows.products(v, seq=0, count=20) == 0).all()  # an empty sequence
    rows.pages.table[1, 2] = -1
    rows.pages.table[1, 3] = 1 << 20
    got = rows.products(v, seq=1, count=150)
    assert torch.isnan(got[:, 64:128]).all()
    kept = list(range(64)) + list(range(128, 150))
    check_products(torch, got[:, kept], v, values[kept], torch.float32)
    near, far = rows.search(v, 100, metric=1, seq=1, count=150)
    assert (near[:, 86:] == -1).all() and torch.isinf(far[:, 86:]).all()
    assert sorted(near[0, :86].tolist()) == kept


def test_products_past_32_bit_offsets(torch, engine):
    """Codes of more than 2^32 bytes, the rows at their end."""
    page_rows, total, dim = 4096, 2200, 1024
    codes = torch.zeros(total, page_rows, 512, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(total, page_rows, 8, dtype=torch.float16, device="cuda")
    assert codes.numel() > 1 << 32
    rows, values = random_rows(torch, engine, 13, 5000, dim, 128, False, torch.float16)
    pages = engine.Pages.empty([codes, scales], 1, 4)
    for column, page in ((0, total - 1), (1, 3)):
        part = slice(column * page_rows, min(5000, (column + 1) * page_rows))
        codes[page, :part.stop - part.start] = rows.codes[part]
        scales[page, :part.stop - part.start] = rows.scales[part]
        pages.table[0, column] = page
        pages.refs[page] = 1
    pages.rows[0] = 5000
    far = engine.Q4Rows(codes, scales, dim, 128, pages=pages)
    v = randn(torch, 4, 2, dim)
    assert torch.equal(far.products(v, seq=0, count=5000), rows.products(v))
    a, b = far.search(v, 20, metric=1, seq=0, count=5000), rows.search(v, 20, metric=1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ search
def plain_search(torch, values, q, k, metric):
    key = torch.stack([(values - row).square().sum(1) if metric == 0 else -(values * row).sum(1)
                       for row in q.double()])
    key, order = key.sort(dim=1, stable=True)
    have = min(k, values.shape[0])
    near = torch.full((q.shape[0], k), -1, dtype=torch.int64, device="cuda")
    far = torch.full((q.shape[0], k), math.inf, dtype=torch.float64, device="cuda")
    near[:, :have], far[:, :have] = order[:, :have], key[:, :have]
    return near, (far if metric == 0 else -far), key


@pytest.mark.parametrize("n,dim,batch,k,group,x,zeros,metric,page_rows", [
    (1, 8, 1, 1, 32, F32, False, 0, 0),
    (5, 40, 2, 10, 32, F32, True, 1, 0),
    (100, 100, 3, 256, 64, F16, False, 0, 7),
    (1000, 128, 1, 10, 32, F32, True, 0, 0),
    (20000, 64, 16, 100, 32, BF16, False, 1, 64),
    (20001, 96, 17, 256, 32, F32, True, 0, 100),
    (50000, 1024, 1, 1, 128, F16, False, 0, 0),
    (50000, 130, 40, 16, 64, F32, False, 1, 0),
    (140000, 64, 5, 256, 64, F32, False, 1, 128),
    (600, 9001, 3, 20, 64, F32, True, 0, 0),
    (600, 8192, 2, 20, 128, F16, False, 1, 16),
    (1100000, 32, 2, 50, 32, BF16, True, 0, 0),
])
def test_search(torch, engine, n, dim, batch, k, group, x, zeros, metric, page_rows):
    rows, values = random_rows(torch, engine, n + k, n, dim, group, zeros, torch.float16, page_rows)
    q = (values[randn(torch, 6, batch).abs().mul(1000).long() % n] + 0.2 * randn(torch, 7, batch, dim)).to(
        getattr(torch, x))
    near, far = rows.search(q, k, metric=metric, seq=1 if page_rows else None, count=n)
    want, distance, _ = plain_search(torch, values, q, k, metric)
    assert torch.equal(near, want)
    fine = torch.isfinite(distance)
    # sums in 64 bits, rounded once to 32; near 0 what 64 bits leave of the terms
    off = (far.double() - distance).abs()[fine]
    assert (off <= 2.0 ** -24 * 1.01 * distance.abs()[fine] + 2.0 ** -40).all()
    assert torch.equal(torch.isinf(far), ~fine) and (far[~fine] == (math.inf if metric == 0 else -math.inf)).all()


@pytest.mark.parametrize("metric", [0, 1])
def test_search_equal_rows(torch, engine, metric):
    """Rows that are copies of one another come by index, however many there are."""
    rows, values = random_rows(torch, engine, 3, 60000, 64, 32, True, torch.float16)
    rows.codes[:] = rows.codes[0]
    rows.scales[:] = rows.scales[0]
    rows.zeros[:] = rows.zeros[0]
    rows.norms[:] = rows.norms[0]
    q = randn(torch, 4, 3, 64)
    near, _ = rows.search(q, 200, metric=metric)
    assert torch.equal(near, torch.arange(200, device="cuda").expand(3, 200))
    # a few groups of copies among other rows
    rows, values = random_rows(torch, engine, 5, 30000, 64, 32, False, torch.float16)
    for t in (rows.codes, rows.scales, rows.norms):
        t[10000:10300] = t[17:18]
        t[29990:] = t[17:18]
    values[10000:10300] = values[17]
    values[29990:] = values[17]
    q = (values[17] * 3).float()[None]
    near, far = rows.search(q, 256, metric=metric)
    want, _, _ = plain_search(torch, values, q, 256, metric)
    assert torch.equal(near, want) and near[0, 0] == 17 and near[0, 1] == 10000


def test_search_near_rows_are_ordered_in_64_bits(torch, engine):
    """Rows that differ by less than fp32's rounding of their distances."""
    n, dim = 4000, 1024
    rows, values = random_rows(torch, engine, 3, n, dim, 128, False, torch.float16)
    rows.scales[:, 0] = 16.0  # one large group, the same for all rows, hides the others
    rows.codes[:, :64] = rows.codes[0, :64]
    rows.scales[:, 1:] = (rows.scales[:, 1:].float() * 1e-2).half()
    values = rows.read().double()
    rows.norms[:] = values.square().sum(1).float()
    q = values[:4].float() + 0.5
    near, _ = rows.search(q, 8, metric=0, count=12)
    want, _, _ = plain_search(torch, values[:12], q, 8, 0)
    assert torch.equal(near, want)


def test_search_without_finite_distances(torch, engine):
    rows, values = random_rows(torch, engine, 8, 300, 64, 32, False, torch.float16)
    rows.scales[::2] = float("nan")
    rows.norms[::2] = float("nan")
    q = randn(torch, 1, 2, 64)
    for metric in (0, 1):
        near, far = rows.search(q, 256, metric=metric)
        assert (near[:, :150] % 2 == 1).all() and (near[:, 150:] == -1).all()
        want, _, _ = plain_search(torch, values[1::2], q, 150, metric)
        assert torch.equal(near[:, :150], 2 * want + 1)
    near, _ = rows.search(torch.full((1, 64), float("nan"), device="cuda"), 5)
    assert (near == -1).all()
    near, _ = rows.search(q, 5, count=0)
    assert (near == -1).all()


# -------------------------------------------------------------------- pack
@pytest.mark.parametrize("n,dim,group,x,zero_points,scale", [
    (1, 1, 32, F32, False, F16), (3, 31, 32, F16, True, F16), (50, 100, 64, BF16, False, BF16),
    (100, 1000, 32, F32, True, F16), (1000, 1024, 64, F16, False, F16), (77, 1025, 128, F32, True, BF16),
    (400, 130, 128, BF16, True, F16), (20000, 64, 32, F32, False, F16), (300, 4096, 128, F32, False, F16)])
def test_pack_and_read(torch, engine, n, dim, group, x, zero_points, scale):
    v = (randn(torch, n, n, dim) * torch.exp(3 * randn(torch, 1, n, 1))).to(getattr(torch, x))
    rows = engine.q4_pack(v, group, zero_points, getattr(torch, scale))
    codes, scales, zeros, values = plain_pack(torch, v, group, zero_points, getattr(torch, scale))
    assert torch.equal(rows.scales, scales)
    assert torch.equal(unpack(torch, rows.codes, dim).double(), codes)
    if zero_points:
        assert torch.equal(rows.zeros.double(), zeros)
    assert torch.equal(rows.read().double(), values)
    assert torch.equal(rows.read(first=n // 2, total=n - n // 2).double(), values[n // 2:])
    want = values.square().sum(1)
    assert ((rows.norms.double() - want).abs() <= (dim + 8) * 2.0 ** -23 * want).all()


def test_pack_ties_and_odd_groups(torch, engine):
    s = torch.tensor([0.75, 2.0 ** -20, 3.0, 100.0], device="cuda")
    steps = torch.arange(-14, 15, device="cuda") / 2
    v = torch.zeros(4, 64, device="cuda")
    v[:, :29] = steps * s[:, None]          # every tie; the largest is 7 s
    v[:, 29] = torch.nextafter(2.5 * s, s * 100)
    v[:, 30] = torch.nextafter(2.5 * s, -s)
    v[:, 31] = torch.nextafter(-3.5 * s, -s * 100)
    v[1, 32:] = 1e-9                        # a scale below the smallest fp16: reads as 0
    v[2, 40] = 65504.0 * 8                  # over 7 above the largest scale (reads as NaN), over 15 below
    v[3, 50] = float("nan")
    for zero_points in (False, True):
        rows = engine.q4_pack(v, 32, zero_points)
        codes, scales, zeros, values = plain_pack(torch, v, 32, zero_points, torch.float16)
        assert torch.equal(torch.nan_to_num(rows.scales, 7.0, 9.0), torch.nan_to_num(scales, 7.0, 9.0))
        got = rows.read().double()
        assert torch.equal(torch.isnan(got), torch.isnan(values))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(values))
        assert torch.isnan(got[3, 32:]).all() and (got[1, 32:] == 0).all()
        assert torch.isnan(got[2, 32:]).all() != zero_points
        assert torch.isnan(rows.norms).tolist() == [False, False, not zero_points, True]


def test_pack_small_and_large_scales(torch, engine):
    """Scales among the subnormal numbers of fp16 and bf16 (codes have to be clamped
    there) and near bf16's largest."""
    v = randn(torch, 3, 200, 128)
    size = 2.0 ** torch.linspace(-30, -16, 200, dtype=torch.float64, device="cuda")
    cases = [((v.double() * size[:, None]).float(), torch.float16)]
    for power in (-128, -124, -100, -98, 118, 124):
        cases.append(((v.double() * 2.0 ** power).float(), torch.bfloat16))
    for x, scale in cases:
        for zero_points in (False, True):
            rows = engine.q4_pack(x, 32, zero_points, scale)
            codes, scales, zeros, values = plain_pack(torch, x, 32, zero_points, scale)
            assert torch.equal(rows.scales, scales)
            assert torch.equal(unpack(torch, rows.codes, 128).double(), codes)
            assert torch.equal(rows.read().double(), values.float().double())


def test_pack_strided_rows(torch, engine):
    wide = randn(torch, 3, 40, 211)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for first, dim in ((0, 200), (1, 200), (2, 77), (3, 128)):
            v = wide.to(dtype)[:, first:first + dim]
            assert torch.equal(engine.q4_pack(v, 32).read(), engine.q4_pack(v.contiguous(), 32).read())


# ------------------------------------------------------------------- pages
class PlainStore:
    """The store in plain Python: a list of rows for each sequence, and pages by
    the rule that fresh ones are the lowest free ones."""

    def __init__(self, sequences, columns, pages, page_rows):
        self.table = [[] for _ in range(sequences)]
        self.rows = [0] * sequences
        self.refs = [0] * pages
        self.page_rows, self.columns = page_rows, columns
        self.held = [[None] * page_rows for _ in range(pages)]

    def need(self, rows):
        return -(-rows // self.page_rows)

    def fresh(self, n):
        got = [p for p, r in enumerate(self.refs) if r == 0][:n]
        for p in got:
            self.refs[p] = 1
        return got if len(got) == n else None

    def content(self, s):
        return [self.held[self.table[s][j // self.page_rows]][j % self.page_rows] for j in range(self.rows[s])]

    def put(self, s, first, values):
        for j, v in enumerate(values, first):
            self.held[self.table[s][j // self.page_rows]][j % self.page_rows] = v

    def grow(self, seqs, counts, values):
        for s, c, v in zip(seqs, counts, values):
            self.table[s] += self.fresh(self.need(self.rows[s] + c) - self.need(self.rows[s]))
            self.put(s, self.rows[s], v)
            self.rows[s] += c

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.rows[s] = [], 0

    def fork(self, parents, children):
        before = [(list(self.table[p]), self.rows[p]) for p in parents]
        for c, (table, rows) in zip(children, before):
            full = rows // self.page_rows
            for p in table[:full]:
                self.refs[p] += 1
            self.table[c], self.rows[c] = table[:full], rows
        for c, (table, rows) in zip(children, before):
            if rows % self.page_rows:
                page, = self.fresh(1)
                self.table[c] = self.table[c] + [page]
                m = rows % self.page_rows
                self.held[page][:m] = self.held[table[-1]][:m]

    def compact(self, sources, targets, keep):
        kept = [[v for v, k in zip(self.content(s), flags) if k] for s, flags in zip(sources, keep)]
        tables = [self.fresh(self.need(len(v))) for v in kept]
        for s, t, table, v in zip(sources, targets, tables, kept):
            if s == t:
                self.free([t])
            self.table[t], self.rows[t] = table, len(v)
            self.put(t, 0, v)


def same_store(torch, pages, plain):
    table = [[p for p in row if p >= 0] for row in pages.table.tolist()]
    assert table == plain.table
    assert all(p == -1 for row, t in zip(pages.table.tolist(), plain.table) for p in row[len(t):])
    assert pages.rows.tolist() == plain.rows
    assert pages.refs.tolist() == plain.refs
    for k, pool in enumerate(pages.pools):
        rows = pool.flatten(2).tolist() if pool.dim() > 2 else pool[..., None].tolist()
        for s in range(len(plain.rows)):
            got = [rows[plain.table[s][j // plain.page_rows]][j % plain.page_rows] for j in range(plain.rows[s])]
            want = [pool_row(k, len(r), v) for r, v in zip(got, plain.content(s))]
            assert got == want, (s, k)


def pool_row(k, width, v):
    """What pool k holds for the row numbered v."""
    return [(v * 7 + k * 3 + j) % 251 for j in range(width)]


def ints(torch, values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def make_store(torch, engine, sequences, columns, total, page_rows, widths):
    pools = [torch.zeros(total, page_rows, w, dtype=dt, device="cuda") if w else
             torch.zeros(total, page_rows, dtype=dt, device="cuda") for w, dt in widths]
    return engine.Pages.empty(pools, sequences, columns), PlainStore(sequences, columns, total, page_rows)


def write_rows(torch, pages, plain, s, first, values):
    for j, v in enumerate(values, first):
        page, slot = plain.table[s][j // plain.page_rows], j % plain.page_rows
        for k, pool in enumerate(pages.pools):
            width = pool[0, 0].numel()
            pool[page, slot] = torch.tensor(pool_row(k, width, v), device="cuda").to(pool.dtype).view(pool[0, 0].shape)


@pytest.mark.parametrize("seed,page_rows,widths", [
    (1, 4, "bytes"), (2, 16, "rows"), (3, 1, "bytes"), (4, 5, "odd"), (5, 130, "rows")])
def test_pages_against_a_plain_store(torch, engine, seed, page_rows, widths):
    """A random run of calls; every state equals the plain store's."""
    widths = {"bytes": [(7, torch.uint8)], "rows": [(24, torch.float16), (0, torch.float32), (64, torch.uint8)],
              "odd": [(3, torch.float16), (1, torch.uint8), (5, torch.float32)]}[widths]
    r = random.Random(seed)
    sequences, columns, total = 9, 12, 60
    pages, plain = make_store(torch, engine, sequences, columns, total, page_rows, widths)
    number = 0
    pages.free(ints(torch, (0,)))  # a step below may find nothing to do: status tells of the last call
    for step in range(60):
        empty = [s for s in range(sequences) if plain.rows[s] == 0]
        full = [s for s in range(sequences) if plain.rows[s]]
        free = sum(x == 0 for x in plain.refs)
        op = r.choice(("grow", "grow", "fork", "free", "compact", "compact", "copy"))
        if op == "grow":
            seqs = r.sample(range(sequences), r.randint(1, 4))
            counts = [r.randint(0, min(3 * page_rows, columns * page_rows - plain.rows[s])) for s in seqs]
            if sum(plain.need(plain.rows[s] + c) - plain.need(plain.rows[s]) for s, c in zip(seqs, counts)) > free:
                continue
            values = []
            for c in counts:
                values.append(list(range(number, number + c)))
                number += c
            pages.grow(ints(torch, seqs), ints(torch, counts))
            starts = [plain.rows[s] for s in seqs]
            plain.grow(seqs, counts, values)
            for s, first, v in zip(seqs, starts, values):
                write_rows(torch, pages, plain, s, first, v)
        elif op == "free":
            seqs = [r.randrange(sequences) for _ in range(r.randint(1, 3))]  # some empty, some twice
            pages.free(ints(torch, seqs))
            plain.free(dict.fromkeys(seqs))
        elif op == "fork" and empty:
            children = r.sample(empty, r.randint(1, len(empty)))
            parents = [r.choice(full or empty) for _ in children]
            if sum(plain.rows[p] % page_rows != 0 for p in parents) > free:
                continue
            pages.fork(ints(torch, parents), ints(torch, children))
            plain.fork(parents, children)
        elif op == "compact" and full:
            sources = [r.choice(full) for _ in range(r.randint(1, 3))]
            targets, left = [], list(empty)
            for s in sources:
                if s not in targets and r.random() < 0.5:
                    targets.append(s)
                elif left:
                    targets.append(left.pop())
                else:
                    targets.append(None)
            sources = [s for s, t in zip(sources, targets) if t is not None]
            targets = [t for t in targets if t is not None]
            if not sources:
                continue
            longest = max(plain.rows[s] for s in sources) + r.randint(0, 3)
            keep = [[r.random() < r.choice((0.0, 0.3, 0.9, 1.0)) for _ in range(longest)] for _ in sources]
            if sum(plain.need(sum(k[:plain.rows[s]])) for s, k in zip(sources, keep)) > free:
                continue
            flags = torch.tensor(keep, device="cuda").view(len(sources), longest)
            if r.random() < 0.5:
                flags = torch.cat((flags, flags), 1)[:, :longest]  # sequences further apart
            pages.compact(ints(torch, sources), ints(torch, targets), flags)
            plain.compact(sources, targets, keep)
        elif op == "copy":
            used, spare = [p for p in range(total) if plain.refs[p]], [p for p in range(total) if not plain.refs[p]]
            n = min(len(used), len(spare), r.randint(1, 5))
            if not n:
                continue
            source, target = [r.choice(used) for _ in range(n)], r.sample(spare, n)
            pages.copy(ints(torch, source), ints(torch, target))
            for pool in pages.pools:
                assert torch.equal(pool[target], pool[source])
        pages.check()
        assert pages.status[1] == 1
        same_store(torch, pages, plain)


def snapshot(pages):
    return [t.clone() for t in (pages.table, pages.rows, pages.refs, *pages.pools)]


def unchanged(torch, pages, before):
    return all(torch.equal(a, b) for a, b in zip(before, (pages.table, pages.rows, pages.refs, *pages.pools)))


def test_pages_refuse_what_the_device_sees(torch, engine):
    pages, _ = make_store(torch, engine, 6, 5, 12, 8, [(16, torch.uint8)])
    pages.grow(ints(torch, (0, 1)), ints(torch, (30, 9)))  # 4 + 2 pages, 6 free
    pages.pools[0].random_(0, 256)
    pages.check()
    before = snapshot(pages)
    keep = torch.ones(2, 40, dtype=torch.bool, device="cuda")
    calls = [
        ("does not exist", lambda: pages.grow(ints(torch, (2, 6)), ints(torch, (1, 1)))),
        ("does not exist", lambda: pages.grow(ints(torch, (-1,)), ints(torch, (1,)))),
        ("listed twice", lambda: pages.grow(ints(torch, (2, 2)), ints(torch, (1, 1)))),
        ("counts", lambda: pages.grow(ints(torch, (2, 3)), ints(torch, (1, -1)))),
        ("columns", lambda: pages.grow(ints(torch, (0,)), ints(torch, (11,)))),
        ("columns", lambda: pages.grow(ints(torch, (0,)), ints(torch, (0x7fffffff,)))),
        ("too few", lambda: pages.grow(ints(torch, (2, 3)), ints(torch, (40, 9)))),
        ("does not exist", lambda: pages.free(ints(torch, (0, 6)))),
        ("does not exist", lambda: pages.copy(ints(torch, (0, 12)), ints(torch, (7, 8)))),
        ("does not exist", lambda: pages.copy(ints(torch, (0, 1)), ints(torch, (7, -1)))),
        ("listed twice", lambda: pages.copy(ints(torch, (0, 1)), ints(torch, (7, 7)))),
        ("listed twice", lambda: pages.copy(ints(torch, (0, 7)), ints(torch, (7, 8)))),
        ("listed twice", lambda: pages.copy(ints(torch, (3,)), ints(torch, (3,)))),
        ("does not exist", lambda: pages.fork(ints(torch, (0, 0)), ints(torch, (2, 6)))),
        ("does not exist", lambda: pages.fork(ints(torch, (9, 0)), ints(torch, (2, 3)))),
        ("listed twice", lambda: pages.fork(ints(torch, (0, 1)), ints(torch, (2, 2)))),
        ("holds rows", lambda: pages.fork(ints(torch, (0, 0)), ints(torch, (2, 1)))),
        ("holds rows", lambda: pages.fork(ints(torch, (0,)), ints(torch, (0,)))),
        ("does not exist", lambda: pages.compact(ints(torch, (0, 6)), ints(torch, (2, 3)), keep)),
        ("does not exist", lambda: pages.compact(ints(torch, (0, 1)), ints(torch, (2, -5)), keep)),
        ("listed twice", lambda: pages.compact(ints(torch, (0, 1)), ints(torch, (2, 2)), keep)),
        ("holds rows", lambda: pages.compact(ints(torch, (0, 1)), ints(torch, (1, 2)), keep)),
        ("counts", lambda: pages.compact(ints(torch, (0, 1)), ints(torch, (2, 3)), keep[:, :29])),
        ("too few", lambda: pages.compact(ints(torch, (0, 0)), ints(torch, (2, 3)), keep)),
    ]
    for text, call in calls:
        call()
        assert pages.status[1] == 0
        with pytest.raises(ValueError, match=text):
            pages.check()
        assert unchanged(torch, pages, before), text
    pages.check()
    # a fork that finds too few pages
    pages.grow(ints(torch, (2,)), ints(torch, (40,)))
    before = snapshot(pages)
    pages.fork(ints(torch, (0, 1)), ints(torch, (3, 4)))
    with pytest.raises(ValueError, match="too few"):
        pages.check()
    assert unchanged(torch, pages, before)
    # the first error is kept until it is asked for, and later calls run
    pages.free(ints(torch, (77,)))
    pages.grow(ints(torch, (3, 3)), ints(torch, (1, 1)))
    pages.free(ints(torch, (2,)))
    with pytest.raises(ValueError, match="does not exist"):
        pages.check()
    assert pages.rows.tolist() == [30, 9, 0, 0, 0, 0]


def test_pages_fork_of_an_empty_parent_that_is_a_child(torch, engine):
    pages, _ = make_store(torch, engine, 4, 3, 8, 4, [(8, torch.uint8)])
    pages.grow(ints(torch, (0,)), ints(torch, (6,)))
    pages.fork(ints(torch, (0, 1)), ints(torch, (1, 2)))  # 1 is empty before the call
    pages.check()
    assert pages.rows.tolist() == [6, 6, 0, 0] and pages.refs.tolist() == [2, 1, 1, 0, 0, 0, 0, 0]


@pytest.mark.parametrize("page_rows,rows", [(1, 3000), (16, 5000), (64, 40000)])
def test_pages_compact_long_sequences_in_place(torch, engine, page_rows, rows):
    """Calls too large for one plan to do it all: a source that is a target too, and a
    source of another, while a fork holds its pages."""
    need = -(-rows // page_rows)
    pool = torch.zeros(4 * need, page_rows, 2, dtype=torch.int32, device="cuda")
    pages = engine.Pages.empty([pool], 4, need + 3)
    pages.grow(ints(torch, (0,)), ints(torch, (rows,)))
    value = torch.arange(rows, dtype=torch.int32, device="cuda")

    def content(s, n):
        at = torch.arange(n, device="cuda")
        return pool[pages.table[s, at // page_rows].long(), at % page_rows]

    at = torch.arange(rows, device="cuda")
    pool[pages.table[0, at // page_rows].long(), at % page_rows] = torch.stack((value, -value), 1)
    pages.fork(ints(torch, (0,)), ints(torch, (1,)))
    keep = randn(torch, 5, 2, rows + 7) > 0.5
    pages.compact(ints(torch, (0, 0)), ints(torch, (0, 2)), keep)
    pages.check()
    for s, want in ((0, value[keep[0, :rows]]), (1, value), (2, value[keep[1, :rows]])):
        assert int(pages.rows[s]) == len(want)
        assert torch.equal(content(s, len(want)), torch.stack((want, -want), 1)), s
    held = pages.table[pages.table >= 0]
    assert torch.equal(pages.refs, torch.bincount(held, minlength=4 * need).int())
    pages.free(ints(torch, (0, 1, 2)))
    assert int(pages.refs.abs().sum()) == 0


def test_pages_of_a_large_store(torch, engine):
    """Many pages, lists as long as allowed, a scan over hundreds of thousands of counts."""
    total, n = 300001, 4096
    pool = torch.zeros(total, 2, 4, dtype=torch.uint8, device="cuda")
    pages = engine.Pages.empty([pool], 2 * n + 1, 80000)
    pages.grow(ints(torch, (2 * n,)), ints(torch, (2 * 75000,)))
    assert torch.equal(pages.table[2 * n, :75000], torch.arange(75000, dtype=torch.int32, device="cuda"))
    g = torch.Generator().manual_seed(4)
    counts = torch.randint(0, 100, (n,), generator=g).int()
    seqs = torch.randperm(n, generator=g).int()
    pages.grow(seqs.cuda(), counts.cuda())
    pages.check()
    need = (counts + 1) // 2
    first = 75000 + need.cumsum(0) - need
    table = pages.table.cpu()
    for i in list(range(0, n, 97)) + [n - 1]:
        assert table[seqs[i], :need[i]].tolist() == list(range(int(first[i]), int(first[i] + need[i])))
    children = torch.arange(n, 2 * n).int()
    pages.fork(seqs.cuda(), children.cuda())
    pages.check()
    odd = counts % 2
    top = 75000 + int(need.sum())
    want = torch.zeros(total, dtype=torch.int32)
    want[:top] = 1
    for i in range(n):
        want[first[i]:first[i] + counts[i] // 2] += 1
    want[top:top + int(odd.sum())] = 1
    assert torch.equal(pages.refs.cpu(), want)
    keep = torch.ones(n, 100, dtype=torch.uint8, device="cuda")
    pages.free(children.cuda())
    pages.compact(seqs.cuda(), children.cuda(), keep)
    pages.check()
    table = pages.table.cpu()
    assert [int(x) for x in table[n:2 * n, 0][need > 0]] == (top + need.cumsum(0) - need)[need > 0].tolist()
    pages.free(torch.cat((seqs, children)).cuda()[:n])
    pages.free(children.cuda())
    pages.check()
    assert int(pages.refs.sum()) == 75000


def test_pages_copy_past_32_bit_offsets(torch, engine):
    total, page_rows = 2100, 1024
    pool = torch.zeros(total, page_rows, 1024, dtype=torch.float16, device="cuda")
    assert pool.numel() * 2 > 1 << 32
    pool[5] = randn(torch, 1, page_rows, 1024).half()
    pool[total - 2] = randn(torch, 2, page_rows, 1024).half()
    pages = engine.Pages.empty([pool], 2, 4)
    pages.copy(ints(torch, (5, total - 2)), ints(torch, (total - 1, 6)))
    assert torch.equal(pool[total - 1], pool[5]) and torch.equal(pool[6], pool[total - 2])
    pages.check()


# ---------------------------------------------------------------- together
def small_store(torch, engine, dim=200, group=64, zeros=True, total=64, page_rows=16, sequences=8, columns=20):
    width, groups = 16 * -(-dim // 32), -(-dim // group)
    codes = torch.zeros(total, page_rows, width, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(total, page_rows, groups, dtype=torch.float16, device="cuda")
    z = torch.zeros(total, page_rows, groups, dtype=torch.uint8, device="cuda") if zeros else None
    norms = torch.zeros(total, page_rows, device="cuda")
    pages = engine.Pages.empty([t for t in (codes, scales, z, norms) if t is not None], sequences, columns)
    return engine.Q4Rows(codes, scales, dim, group, z, norms, pages)


def held(torch, v, group=64, zero_points=True):
    return plain_pack(torch, v, group, zero_points, torch.float16)[3]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_collection_lives(torch, engine, dtype):
    """Append, fork, append to both, drop rows, search, free."""
    rows = small_store(torch, engine)
    pages = rows.pages
    a, b, c = (randn(torch, s, n, 200).to(getattr(torch, dtype)) for s, n in ((1, 50), (2, 33), (3, 21)))
    rows.append(ints(torch, (2, 5)), ints(torch, (50, 33)), torch.cat((a, b)))
    assert torch.equal(rows.read(ints(torch, (5, 2)), ints(torch, (33, 20)), 53).double(),
                       torch.cat((held(torch, b), held(torch, a)[30:])))
    pages.fork(ints(torch, (2,)), ints(torch, (0,)))
    rows.append(ints(torch, (0, 2)), ints(torch, (21, 1)), torch.cat((c, c[:1])))
    want = {0: torch.cat((a, c)), 2: torch.cat((a, c[:1])), 5: b}
    for s, v in want.items():
        got = rows.read(ints(torch, (s,)), ints(torch, (len(v),)), len(v))
        assert torch.equal(got.double(), held(torch, v)), s
    q = randn(torch, 9, 3, 200)
    for s, v in want.items():
        near, _ = rows.search(q, 10, seq=s, count=200)
        assert torch.equal(near, plain_search(torch, held(torch, v), q, 10, 0)[0])
        check_products(torch, rows.products(q, seq=s, count=len(v)), q, held(torch, v), torch.float32)
    keep = torch.zeros(1, 80, dtype=torch.bool, device="cuda")
    keep[0, 3:71:2] = True
    pages.compact(ints(torch, (0,)), ints(torch, (0,)), keep)
    v = held(torch, want[0])[3:71:2]
    near, _ = rows.search(q, 10, metric=1, seq=0, count=len(v))
    assert torch.equal(near, plain_search(torch, v, q, 10, 1)[0])
    assert torch.equal(rows.read(ints(torch, (2,)), ints(torch, (51,)), 51).double(), held(torch, want[2]))
    pages.free(ints(torch, (0, 2, 5)))
    pages.check()
    assert int(pages.refs.abs().sum()) == 0 and (pages.table == -1).all()


def test_append_and_read_refuse_wrong_lists(torch, engine):
    rows = small_store(torch, engine)
    v = randn(torch, 1, 30, 200)
    rows.append(ints(torch, (1,)), ints(torch, (30,)), v)
    before = snapshot(rows.pages)
    for seqs, counts in (((2, 3), (10, 19)), ((2, 3), (10, 21)), ((2, 2), (10, 20)), ((2, 8), (10, 20)),
                         ((2, 3), (31, -1)), ((1,), (30,)), ((2,), (1 << 30,))):
        if (seqs, counts) == ((1,), (30,)):
            continue
        rows.append(ints(torch, seqs), ints(torch, counts), v)
        with pytest.raises(ValueError):
            rows.pages.check()
        assert unchanged(torch, rows.pages, before)
    for seqs, counts, total in (((1,), (31,), 31), ((1, 9), (5, 5), 10), ((1,), (5,), 6), ((1,), (-1,), 1),
                                ((1, 1), (30, 30), 59)):
        rows.read(ints(torch, seqs), ints(torch, counts), total)
        with pytest.raises(ValueError):
            rows.pages.check()
    # one sequence twice is fine to read, and nothing may be appended
    assert torch.equal(rows.read(ints(torch, (1, 1)), ints(torch, (2, 1)), 3)[:2][1:],
                       rows.read(ints(torch, (1,)), ints(torch, (1,)), 1))
    rows.append(ints(torch, (1, 2)), ints(torch, (0, 0)), v[:0])
    rows.pages.check()
    assert unchanged(torch, rows.pages, before)


def test_wrong_tensors_are_refused(torch, engine):
    rows = small_store(torch, engine)
    dense = engine.q4_pack(randn(torch, 1, 10, 64), 32)
    i32 = ints(torch, (0, 1))
    v = randn(torch, 1, 2, 200)
    wrong = [
        lambda: rows.pages.free(i32.long()), lambda: rows.pages.free(i32.cpu()),
        lambda: rows.pages.free(ints(torch, range(8))[::2]), lambda: rows.pages.free(i32.view(1, 2)),
        lambda: rows.pages.grow(i32, i32[:1]), lambda: rows.pages.fork(i32, i32[:1]),
        lambda: rows.pages.free(torch.zeros(4097, dtype=torch.int32, device="cuda")),
        lambda: rows.pages.compact(i32, i32, torch.ones(1, 5, dtype=torch.bool, device="cuda")),
        lambda: rows.pages.compact(i32, i32, torch.ones(2, 5, device="cuda")),
        lambda: rows.pages.compact(i32, i32, torch.ones(5, 2, dtype=torch.bool, device="cuda").T),
        lambda: rows.append(i32, i32, v.double()), lambda: rows.append(i32, i32, v[:, :100]),
        lambda: rows.append(i32, i32, v.T.contiguous().T), lambda: dense.append(i32, i32, v),
        lambda: rows.products(v), lambda: rows.products(v, seq=0), lambda: rows.products(v, seq=8, count=1),
        lambda: rows.products(v, seq=0, count=5000), lambda: rows.products(v.cpu(), seq=0, count=5),
        lambda: rows.products(v, seq=0, count=-1), lambda: rows.products(v.expand(2, 2, 200), seq=0, count=1),
        lambda: rows.products(v, seq=0, count=5, out=torch.zeros(2, 6, device="cuda")),
        lambda: rows.products(v, seq=0, count=5, out=torch.zeros(2, 5, dtype=torch.float64, device="cuda")),
        lambda: rows.products(v[:1].expand(2, 200), seq=0, count=5),
        lambda: dense.products(v[:, :64], seq=0), lambda: dense.products(v[:, :64], dtype=torch.int32),
        lambda: rows.search(v, 0, seq=0, count=5), lambda: rows.search(v, 257, seq=0, count=5),
        lambda: rows.search(v[0], 5, seq=0, count=5), lambda: rows.search(v, 5, metric=2, seq=0, count=5),
        lambda: engine.Q4Rows(dense.codes, dense.scales, 64, 32).search(v[:, :64], 3),
        lambda: dense.read(i32, i32, 3), lambda: dense.read(first=5, total=6), lambda: rows.read(i32, i32),
        lambda: engine.Q4Rows(dense.codes, dense.scales, 65, 32),
        lambda: engine.Q4Rows(dense.codes, dense.scales, 64, 64),
        lambda: engine.Q4Rows(dense.codes, dense.scales.float(), 64, 32),
        lambda: engine.Q4Rows(dense.codes, dense.scales, 64, 32, norms=dense.norms.half()),
        lambda: engine.Q4Rows(rows.codes, rows.scales, 200, 64),
        lambda: engine.Q4Rows(dense.codes, dense.scales, 64, 32, pages=rows.pages),
        lambda: engine.q4_pack(v, 100), lambda: engine.q4_pack(v[0]), lambda: engine.q4_pack(v.double()),
        lambda: engine.Pages(rows.pages.table.long(), rows.pages.rows, rows.pages.refs, rows.pages.pools),
        lambda: engine.Pages(rows.pages.table, rows.pages.rows[:3], rows.pages.refs, rows.pages.pools),
        lambda: engine.Pages(rows.pages.table, rows.pages.rows, rows.pages.refs, []),
        lambda: engine.Pages(rows.pages.table, rows.pages.rows, rows.pages.refs, [rows.codes[:5]]),
    ]
    for k, call in enumerate(wrong):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was taken")


def test_in_a_graph(torch, engine):
    """A captured step (free, append, fork, drop rows, search, products), replayed on
    new contents, equals the step run directly; two graphs share one store."""
    v, q = randn(torch, 1, 40, 200), randn(torch, 2, 3, 200)
    keep = randn(torch, 3, 1, 40) > 0
    seqs, counts, one, two, all_three = (ints(torch, x) for x in ((0,), (40,), (1,), (2,), (0, 1, 2)))

    def step(rows):
        rows.pages.free(all_three)
        rows.append(seqs, counts, v)
        rows.pages.fork(seqs, one)
        rows.pages.compact(one, two, keep)
        near, far = rows.search(q, 12, seq=2, count=60)
        return near, far, rows.products(q, seq=1, count=60), rows.read(one, counts, 40)

    rows, other = small_store(torch, engine), small_store(torch, engine)
    step(rows)  # first calls, outside of a capture
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(rows)
        graphs.append((graph, out))
    for seed in (5, 6):
        v.copy_(randn(torch, seed, 40, 200))
        q.copy_(randn(torch, seed + 10, 3, 200))
        keep.copy_(randn(torch, seed + 20, 1, 40) > 0)
        want = step(other)
        for graph, out in graphs + graphs:
            for t in out:
                t.zero_()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    rows.pages.check()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(rows.pages)[:3], snapshot(other.pages)[:3]))


def test_on_other_streams_at_once(torch, engine):
    rows, values = random_rows(torch, engine, 21, 30000, 256, 64, False, torch.float16)
    q = randn(torch, 2, 8, 256)
    want = rows.search(q, 20), rows.products(q)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for turn in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((rows.search(q, 20), rows.products(q)))
    torch.cuda.synchronize()
    for (near, far), y in got:
        assert torch.equal(near, want[0][0]) and torch.equal(far, want[0][1]) and torch.equal(y, want[1])


def test_kernels_are_counted(torch, engine):
    rows, _ = random_rows(torch, engine, 21, 300, 64, 64, False, torch.float16)
    engine.reset_dispatch_count()
    rows.products(randn(torch, 1, 1, 64))
    assert engine.dispatch_count() >= 1
