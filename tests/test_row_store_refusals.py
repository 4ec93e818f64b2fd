"""CPU tests of what the row store's entry points refuse: rows that are no pools
of their store, and addresses that a kernel could not load from.  No call here
reaches a GPU: products of no vectors and lists without entries check their
arguments and return."""
import ctypes

import pytest


def make_store(engine, zeros=True, norms=True):
    """Rows of 100 values in groups of 32, and the store that they are pools of."""
    p = engine.KnnPages(table=4096, rows=4096, refs=4096, status=4096, sequences=4, columns=8, pages=16, page_rows=32,
                        device=0)
    q = engine.KnnQ4Rows(codes=0x10000, scales=0x20000, n_rows=512, dim=100, group=32, scale_dtype=1, device=0)
    held = [(0x10000, 64), (0x20000, 8)]
    if zeros:
        q.zeros = 0x30000
        held.append((0x30000, 4))
    if norms:
        q.norms = 0x40000
        held.append((0x40000, 4))
    for k, (at, size) in enumerate(held):
        p.pools[k], p.row_bytes[k] = at, size
    p.n_pools = len(held)
    q.pages = ctypes.pointer(p)
    return p, q


def status(engine, q):
    return engine.lib().knn_q4_products(ctypes.byref(q), 0, 0, None, 0, 0, 0, None, 0, 0, None)


def test_rows_are_pools_of_their_store(engine):
    for zeros in (False, True):
        for norms in (False, True):
            p, q = make_store(engine, zeros, norms)
            assert status(engine, q) == engine.KNN_OK
            # more pools than the rows use, in another order
            p.pools[p.n_pools], p.row_bytes[p.n_pools] = 0x90000, 4
            p.n_pools += 1
            p.pools[0], p.pools[1] = p.pools[1], p.pools[0]
            p.row_bytes[0], p.row_bytes[1] = p.row_bytes[1], p.row_bytes[0]
            assert status(engine, q) == engine.KNN_OK


@pytest.mark.parametrize("name", ["codes", "scales", "zeros", "norms"])
def test_rows_outside_their_store_are_refused(engine, name):
    p, q = make_store(engine)
    setattr(q, name, 0x50000)
    assert status(engine, q) == engine.KNN_EINVAL
    assert name.encode() in engine.lib().knn_last_error()
    p, q = make_store(engine)
    k = ["codes", "scales", "zeros", "norms"].index(name)
    p.row_bytes[k] += 4  # a pool at the same place with other rows
    assert status(engine, q) == engine.KNN_EINVAL
    p, q = make_store(engine)
    p.n_pools = k  # the pool is not the store's
    assert status(engine, q) == engine.KNN_EINVAL
    lib, r = engine.lib(), ctypes.byref(q)
    assert lib.knn_q4_append(r, 4096, 4096, 1, 4096, 0, 1, 100, None) == engine.KNN_EINVAL
    assert lib.knn_q4_search(r, 0, 1, 4096, 0, 1, 100, 1, 0, 4096, 4096, 4096, None) == engine.KNN_EINVAL
