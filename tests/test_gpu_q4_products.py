"""Products with rows in 4 bits where a loss of range would show, or vectors
that get in each other's way.

Tolerances.  A sum of n terms in fp32, in any order, each step rounded or cut,
is off by at most n * 2^-23 of the sum of magnitudes.
"""
import pytest

from test_gpu_row_store import check_products, randn, random_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


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
