"""CPU tests of the row store's entry points: sizes, and refusals of what the
host can see.  No call here reaches a GPU."""
import ctypes

import pytest


def make_pages(engine, **change):
    c = engine.KnnPages(table=4096, rows=4096, refs=4096, status=4096, sequences=4, columns=8, pages=16,
                        page_rows=32, n_pools=1, device=0)
    c.pools[0], c.row_bytes[0] = 4096, 64
    for name, value in change.items():
        if name == "row_bytes":
            c.row_bytes[0] = value
        elif name == "pool":
            c.pools[0] = value
        else:
            setattr(c, name, value)
    return c


def make_rows(engine, pages=None, **change):
    c = engine.KnnQ4Rows(codes=4096, scales=4096, norms=4096, n_rows=512, dim=100, group=32, scale_dtype=1,
                         device=0)
    if pages is not None:
        c.pages = ctypes.pointer(pages)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def test_sizes(engine):
    lib = engine.lib()
    assert [lib.knn_q4_row_bytes(d) for d in (0, 1, 32, 33, 1000, 1024)] == [0, 16, 16, 32, 512, 512]
    assert lib.knn_q4_search_workspace(-1, 1) == -1 and lib.knn_q4_search_workspace(1, -1) == -1
    assert lib.knn_q4_search_workspace(1, 1) >= 4
    # a key a row and query, for up to 16 queries at once
    assert 4e6 < lib.knn_q4_search_workspace(10**6, 1) < 5e6
    assert lib.knn_q4_search_workspace(10**6, 100) == lib.knn_q4_search_workspace(10**6, 16) < 80e6
    p = make_pages(engine)
    # flags' counts, totals and new table rows: room for 4 bytes of each
    assert lib.knn_pages_compact_workspace(ctypes.byref(p), 3, 1000) >= 4 * 3 * (8 + 2)
    assert lib.knn_pages_compact_workspace(None, 3, 1000) == -1
    assert lib.knn_pages_compact_workspace(ctypes.byref(p), 5000, 1000) == -1


@pytest.mark.parametrize("change", [
    dict(table=None), dict(rows=None), dict(refs=None), dict(status=None), dict(sequences=0),
    dict(sequences=(1 << 20) + 1), dict(columns=0), dict(pages=0), dict(pages=(1 << 20) + 1),
    dict(page_rows=0), dict(page_rows=1 << 30), dict(n_pools=9), dict(n_pools=-1), dict(pool=None),
    dict(row_bytes=0), dict(row_bytes=(1 << 24) + 1)])
def test_wrong_pages_are_refused(engine, change):
    lib, p = engine.lib(), make_pages(engine, **change)
    r = ctypes.byref(p)
    for status in (lib.knn_pages_grow(r, 4096, 4096, 1, -1, None), lib.knn_pages_free(r, 4096, 1, None),
                   lib.knn_pages_copy(r, 4096, 4096, 1, None), lib.knn_pages_fork(r, 4096, 4096, 1, None),
                   lib.knn_pages_compact(r, 4096, 4096, 1, 4096, 10, 10, 4096, None)):
        assert status == engine.KNN_EINVAL, engine.lib().knn_last_error()


def test_wrong_lists_are_refused(engine):
    lib, p = engine.lib(), make_pages(engine)
    r = ctypes.byref(p)
    refused = [
        lib.knn_pages_grow(r, None, 4096, 1, -1, None), lib.knn_pages_grow(r, 4096, None, 1, -1, None),
        lib.knn_pages_grow(r, 4096, 4096, -1, -1, None), lib.knn_pages_grow(r, 4096, 4096, 4097, -1, None),
        lib.knn_pages_grow(r, None, None, 0, 5, None), lib.knn_pages_free(r, None, 1, None),
        lib.knn_pages_free(r, 4096, 4097, None), lib.knn_pages_copy(r, 4096, None, 1, None),
        lib.knn_pages_copy(r, 4096, 4096, (1 << 20) + 1, None), lib.knn_pages_fork(r, None, 4096, 1, None),
        lib.knn_pages_compact(r, 4096, None, 1, 4096, 10, 10, 4096, None),
        lib.knn_pages_compact(r, 4096, 4096, 1, None, 10, 10, 4096, None),
        lib.knn_pages_compact(r, 4096, 4096, 2, 4096, 10, 9, 4096, None),
        lib.knn_pages_compact(r, 4096, 4096, 1, 4096, -1, 10, 4096, None),
        lib.knn_pages_compact(r, 4096, 4096, 1, 4096, 10, 10, None, None),
        lib.knn_pages_compact(r, 4096, 4096, 1, 4096, 10, 10, 4097, None)]
    assert refused == [engine.KNN_EINVAL] * len(refused)
    assert lib.knn_pages_compact(r, 4096, 4096, 4096, 4096, 0x7fffffff, 0x7fffffff, 4096,
                                 None) == engine.KNN_EUNSUPPORTED
    # nothing to do: no GPU needed
    assert lib.knn_pages_free(r, None, 0, None) == engine.KNN_OK
    assert lib.knn_pages_copy(r, None, None, 0, None) == engine.KNN_OK
    assert lib.knn_pages_free(None, None, 0, None) == engine.KNN_EINVAL


@pytest.mark.parametrize("change", [
    dict(dim=0), dict(dim=65537), dict(group=0), dict(group=16), dict(group=100), dict(scale_dtype=0),
    dict(n_rows=-1), dict(n_rows=1 << 31), dict(codes=None), dict(codes=4104), dict(scales=None),
    dict(scales=4097)])
def test_wrong_rows_are_refused(engine, change):
    lib, q = engine.lib(), make_rows(engine, **change)
    r = ctypes.byref(q)
    for status in (lib.knn_q4_pack(r, 4096, 0, 1, 200, 0, None),
                   lib.knn_q4_read(r, None, None, 0, 0, 1, 4096, 200, None),
                   lib.knn_q4_products(r, -1, 1, 4096, 0, 1, 200, 4096, 0, 1, None),
                   lib.knn_q4_search(r, -1, 1, 4096, 0, 1, 200, 1, 0, 4096, 4096, 4096, None)):
        assert status == engine.KNN_EINVAL, engine.lib().knn_last_error()


def test_wrong_calls_are_refused(engine):
    lib = engine.lib()
    dense, store = make_rows(engine), make_rows(engine, make_pages(engine))
    d, s = ctypes.byref(dense), ctypes.byref(store)
    wrong = ctypes.byref(make_rows(engine, make_pages(engine), n_rows=500))
    bare = make_rows(engine, norms=None)
    refused = [
        lib.knn_q4_pack(None, 4096, 0, 1, 200, 0, None), lib.knn_q4_pack(d, 4096, 3, 1, 200, 0, None),
        lib.knn_q4_pack(d, None, 0, 1, 200, 0, None), lib.knn_q4_pack(d, 4096, 0, 2, 99, 0, None),
        lib.knn_q4_pack(d, 4096, 0, 2, 200, 511, None), lib.knn_q4_pack(d, 4096, 0, 1, 200, -1, None),
        lib.knn_q4_pack(s, 4096, 0, 1, 200, 0, None),
        lib.knn_q4_append(d, 4096, 4096, 1, 4096, 0, 1, 200, None),
        lib.knn_q4_append(s, 4096, 4096, 1, None, 0, 1, 200, None),
        lib.knn_q4_append(s, 4096, 4096, 1, 4096, 0, 2, 99, None),
        lib.knn_q4_append(s, 4096, 4096, 1, 4096, 0, -1, 200, None),
        lib.knn_q4_append(s, None, None, 0, 4096, 0, 1, 200, None),
        lib.knn_q4_read(d, 4096, 4096, 1, 0, 1, 4096, 200, None),
        lib.knn_q4_read(d, None, None, 0, 500, 13, 4096, 200, None),
        lib.knn_q4_read(s, 4096, 4096, 1, 1, 1, 4096, 200, None),
        lib.knn_q4_read(s, 4096, None, 1, 0, 1, 4096, 200, None),
        lib.knn_q4_read(s, 4096, 4096, 1, 0, 2, 4096, 99, None),
        lib.knn_q4_products(d, 0, 1, 4096, 0, 1, 200, 4096, 0, 1, None),
        lib.knn_q4_products(s, -1, 1, 4096, 0, 1, 200, 4096, 0, 1, None),
        lib.knn_q4_products(s, 4, 1, 4096, 0, 1, 200, 4096, 0, 1, None),
        lib.knn_q4_products(d, -1, 513, 4096, 0, 1, 200, 4096, 0, 513, None),
        lib.knn_q4_products(d, -1, 10, None, 0, 1, 200, 4096, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, 4096, 7, 1, 200, 4096, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, 4096, 0, 1, 200, 4096, 7, 10, None),
        lib.knn_q4_products(d, -1, 10, 4096, 0, 2, 99, 4096, 0, 10, None),
        lib.knn_q4_products(d, -1, 10, 4096, 0, 2, 200, 4096, 0, 9, None),
        lib.knn_q4_products(d, -1, 10, 4096, 0, -1, 200, 4096, 0, 10, None),
        lib.knn_q4_search(d, -1, 10, 4096, 0, 1, 200, 0, 0, 4096, 4096, 4096, None),
        lib.knn_q4_search(d, -1, 10, 4096, 0, 1, 200, 257, 0, 4096, 4096, 4096, None),
        lib.knn_q4_search(d, -1, 10, 4096, 0, 1, 200, 5, 2, 4096, 4096, 4096, None),
        lib.knn_q4_search(d, -1, 10, 4096, 0, 1, 200, 5, 0, 4096, 4096, None, None),
        lib.knn_q4_search(d, -1, 10, 4096, 0, 1, 200, 5, 0, None, 4096, 4096, None),
        lib.knn_q4_search(ctypes.byref(bare), -1, 10, 4096, 0, 1, 200, 5, 0, 4096, 4096, 4096, None),
        lib.knn_q4_products(wrong, 0, 1, 4096, 0, 1, 200, 4096, 0, 1, None)]
    assert refused == [engine.KNN_EINVAL] * len(refused), refused
    assert lib.knn_q4_products(d, -1, 0, None, 0, 1, 200, None, 0, 0, None) == engine.KNN_OK
    assert lib.knn_q4_pack(d, None, 0, 0, 200, 512, None) == engine.KNN_OK


def test_host_tensors_are_refused(engine):
    import torch

    ints = torch.zeros(4, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        engine.Pages(ints, ints[0], ints[0], [torch.zeros(4, 2, 8)])
    with pytest.raises(ValueError, match="CUDA"):
        engine.Pages.empty([torch.zeros(4, 2, 8)], 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        engine.Q4Rows(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16), 32, 32)
    with pytest.raises(ValueError, match="CUDA"):
        engine.q4_pack(torch.zeros(4, 32))
    with pytest.raises(ValueError):
        engine.q4_pack(torch.zeros(4, 32), group=48)
