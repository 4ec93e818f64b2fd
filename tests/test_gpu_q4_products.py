"""Products with rows in 4 bits where a loss of bits or of range would show, or
vectors that get in each other's way.

Tolerances.  An fp32 vector is held in two fp16 parts, to 2^-23 of a value and
2^-51 of its vector's largest; a bf16 one in one part, to 2^-39 of the largest.
One product scaled, moved to its vector's scale and added to zeros is rounded
four times more at the most, 2^-24 each.  A sum of n terms in fp32, in any
order, each step rounded or cut, is off by at most n * 2^-23 of the sum of
magnitudes.
"""
import pytest

from test_gpu_row_store import check_products, randn, random_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


@pytest.mark.parametrize("dim,group,zeros", [(100, 32, True), (1000, 32, False), (2049, 64, True), (4096, 128, False),
                                             (20000, 128, True), (65535, 64, False)])
@pytest.mark.parametrize("batch", [1, 3, 4, 7, 16])
def test_every_place_takes_all_bits_of_a_value(torch, engine, dim, group, zeros, batch):
    """Vectors with one value each, of 24 bits, at places of every stage."""
    rows, values = random_rows(torch, engine, dim, 65, dim, group, zeros, torch.float16)
    g = torch.Generator(device="cuda").manual_seed(dim + batch)
    for turn in range(-(-40 // batch)):
        at = (torch.arange(batch, device="cuda") + turn * batch) * dim // (40 + batch)
        v = torch.zeros(batch, dim, device="cuda")
        value = torch.rand(batch, device="cuda", generator=g) + torch.randint(1, 9, (batch,), device="cuda", generator=g)
        v[torch.arange(batch, device="cuda"), at] = value
        want = value.double()[:, None] * values.T[at]
        off = (rows.products(v).double() - want).abs()
        assert (off <= 2.0 ** -23 * (1 + 4 / 2) * want.abs()).all(), (turn, (off / want.abs()).max())


@pytest.mark.parametrize("dim,batch,group", [(200, 1, 32), (1024, 4, 64), (1024, 8, 128), (2049, 16, 64), (4096, 2, 128),
                                             (14336, 9, 32)])
def test_low_parts_are_all_there_is(torch, engine, dim, batch, group):
    """Pairs of values that differ in their last bits against opposite codes: what a
    single fp16 part keeps of them adds up to nothing."""
    n = 70
    rows, _ = random_rows(torch, engine, dim, n, dim, group, False, torch.float16)
    g = torch.Generator(device="cuda").manual_seed(dim)
    low = torch.randint(1, 16, rows.codes.shape, device="cuda", generator=g, dtype=torch.uint8)
    rows.codes[:] = low | ((16 - low) << 4)  # c - 8 and 8 - c
    values = rows.read().double()
    v = randn(torch, 5, batch, dim)
    even = v[:, 0:dim - dim % 2:2]
    v[:, 1::2] = even * (1 + 2.0 ** -14 * torch.rand(even.shape, device="cuda", generator=g))
    if dim % 2:
        v[:, -1] = 0
    want = v.double() @ values.T
    size = v.double().abs() @ values.abs().T
    # each value to 2^-23, and sums of at most a group's values, the groups, and what splits them
    steps = 2 * group + -(-dim // group) + 32
    off = (rows.products(v).double() - want).abs()
    assert (off <= steps * 2.0 ** -23 * size).all()
    assert off.square().mean().sqrt() <= 2.0 ** -23 * size.mean()
    # without low parts the error would be all there is, and that is more
    assert want.square().mean().sqrt() > 2.0 ** -23 * size.mean()


@pytest.mark.parametrize("x", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch", [1, 4, 6, 16])
def test_small_values_beside_a_large_one(torch, engine, x, batch):
    """Magnitudes of one vector from 1 to 1e-7; rows that are zero where it is large."""
    n, dim = 200, 512
    rows, _ = random_rows(torch, engine, 5, n, dim, 64, True, torch.float16)
    rows.codes[:, 50] = 0x11 * rows.zeros[:, 1]  # values 100 and 101, of group 1
    values = rows.read().double()
    assert (values[:, 100] == 0).all()
    dt = getattr(torch, x)
    for power in (0, -10, -17, -20, -23, -26, -28):
        v = (randn(torch, power + 50, batch, dim) * 2.0 ** power)
        v[:, 100] = torch.linspace(1.0, 1.99, batch, device="cuda")
        v = v.to(dt)
        others = v.clone()
        others[:, 100] = 0
        want = others.double() @ values.T
        size = others.double().abs() @ values.abs().T
        held = (2.0 ** -50 if x == "float32" else 2.0 ** -38) * values.abs().sum(1)
        off = (rows.products(v).double() - want).abs()
        assert (off <= (2 * 64 + 8 + 32) * 2.0 ** -23 * size + held).all()
        assert off.square().mean().sqrt() <= 2.0 ** -22 * size.mean() + held.mean(), power


@pytest.mark.parametrize("x", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("batch", [1, 5, 16])
@pytest.mark.parametrize("zeros", [False, True])
def test_large_and_small_scales(torch, engine, x, batch, zeros):
    """Scales near both ends of bf16 with vectors that bring the products back."""
    n, dim = 100, 300
    dt = getattr(torch, x)
    pairs = [(100, -20), (100, -90), (119, -120), (90, 20), (-100, 20), (-110, 100), (-120, 110), (0, -120), (0, 110)]
    if x == "float16":
        pairs = [(100, -20), (100, 10), (-100, 10), (-110, 0)]
    for scale, size in pairs:
        rows, _ = random_rows(torch, engine, 7, n, dim, 32, zeros, torch.bfloat16)
        rows.scales[:] = (rows.scales.double() * 2.0 ** scale).to(torch.bfloat16)
        values = rows.read().double()
        v = (randn(torch, 3, batch, dim).double() * 2.0 ** size).to(dt)
        check_products(torch, rows.products(v), v, values, torch.float32)
        again = rows.search(v, 5, metric=1)
        want = (v.double() @ values.T).sort(dim=1, descending=True, stable=True)
        assert torch.equal(again[0], want.indices[:, :5])


@pytest.mark.parametrize("x", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,dim,batch,page_rows", [(3000, 1000, 3, 0), (100, 4096, 16, 16), (70, 2049, 8, 0)])
def test_a_vector_gets_the_same_bits_among_others(torch, engine, x, n, dim, batch, page_rows):
    rows, _ = random_rows(torch, engine, 8, n, dim, 64, True, torch.float16, page_rows)
    seq = 1 if page_rows else None
    v = randn(torch, 3, batch, dim).to(getattr(torch, x))
    first = rows.products(v, seq=seq, count=n)
    other = (randn(torch, 4, batch, dim) * 1e3).to(getattr(torch, x))
    other[batch // 2] = v[batch // 2]
    assert torch.equal(rows.products(other, seq=seq, count=n)[batch // 2], first[batch // 2])


def test_a_gradient_is_refused_not_lost(torch, engine):
    rows, _ = random_rows(torch, engine, 9, 50, 64, 32, False, torch.float16)
    x = randn(torch, 1, 3, 64).requires_grad_()
    for call in (lambda: rows.products(x), lambda: rows.products(x[0]),
                 lambda: rows.products(x.detach(), out=torch.zeros(3, 50, device="cuda", requires_grad=True))):
        with pytest.raises(ValueError, match="gradient"):
            call()
    want = rows.products(x.detach())
    with torch.no_grad():
        assert torch.equal(rows.products(x), want)
    with torch.inference_mode():
        assert torch.equal(rows.products(x), want)
    # a weight that requires a gradient can be packed: its codes have none
    assert torch.equal(engine.q4_pack(x, 32).codes, engine.q4_pack(x.detach(), 32).codes)
