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


@pytest.mark.parametrize("name", ["table", "rows", "refs", "status"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_stores_at_odd_addresses_are_refused(engine, name, off):
    lib = engine.lib()
    p, q = make_store(engine)
    assert lib.knn_pages_free(ctypes.byref(p), None, 0, None) == engine.KNN_OK
    setattr(p, name, 4096 + off)
    r = ctypes.byref(p)
    assert [lib.knn_pages_free(r, None, 0, None), lib.knn_pages_copy(r, None, None, 0, None),
            lib.knn_pages_grow(r, None, None, 0, -1, None), lib.knn_pages_fork(r, None, None, 0, None),
            lib.knn_pages_compact(r, None, None, 0, None, 0, 0, None, None), status(engine, q)
            ] == [engine.KNN_EINVAL] * 6


def test_buffers_at_odd_addresses_are_refused(engine):
    lib, (p, q) = engine.lib(), make_store(engine)
    dense = engine.KnnQ4Rows(codes=0x10000, scales=0x20000, norms=0x40000, n_rows=512, dim=100, group=32, scale_dtype=1,
                             device=0)
    r, s, d = ctypes.byref(p), ctypes.byref(q), ctypes.byref(dense)
    ok, odd, half = 4096, 4097, 4098
    refused = [
        lib.knn_pages_grow(r, half, ok, 1, -1, None), lib.knn_pages_grow(r, ok, half, 1, -1, None),
        lib.knn_pages_free(r, half, 1, None), lib.knn_pages_copy(r, half, ok, 1, None),
        lib.knn_pages_copy(r, ok, odd, 1, None), lib.knn_pages_fork(r, ok, half, 1, None),
        lib.knn_pages_compact(r, half, ok, 1, ok, 10, 10, ok, None), lib.knn_pages_compact(r, ok, odd, 1, ok, 10, 10, ok, None),
        lib.knn_q4_pack(d, half, 0, 1, 200, 0, None), lib.knn_q4_pack(d, odd, 1, 1, 200, 0, None),
        lib.knn_q4_append(s, half, ok, 1, ok, 0, 1, 200, None), lib.knn_q4_append(s, ok, ok, 1, half, 0, 1, 200, None),
        lib.knn_q4_append(s, ok, ok, 1, odd, 2, 1, 200, None),
        lib.knn_q4_read(d, None, None, 0, 0, 1, half, 200, None), lib.knn_q4_read(s, ok, half, 1, 0, 1, ok, 200, None),
        lib.knn_q4_products(d, -1, 10, half, 0, 1, 200, ok, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, odd, 1, 1, 200, ok, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, ok, 1, 1, 200, half, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, ok, 1, 1, 200, odd, 2, 10, None),
        lib.knn_q4_search(d, -1, 10, half, 0, 1, 200, 5, 0, ok, ok, ok, None),
        lib.knn_q4_search(d, -1, 10, ok, 0, 1, 200, 5, 0, ok + 4, ok, ok, None),
        lib.knn_q4_search(d, -1, 10, ok, 0, 1, 200, 5, 0, ok, half, ok, None),
        lib.knn_q4_search(d, -1, 10, ok, 0, 1, 200, 5, 0, ok, ok, ok + 8, None)]
    assert refused == [engine.KNN_EINVAL] * len(refused), refused
    dense.norms = 0x40002
    assert lib.knn_q4_products(d, -1, 0, None, 0, 0, 0, None, 0, 0, None) == engine.KNN_EINVAL
