"""Python binding of the B200 exact k-NN engine (ctypes over the C ABI in
include/cuvs_b200.h).

Mirrors the reference's search interface for this path:
``cuvs::neighbors::cagra::build`` / ``search`` with a graph-less index
(include/cuvs/neighbors/cagra.hpp:94-106 of ysys143/cuvs-silicon) and the
``brute_force`` build/search pair the engine adds.  Argument errors raise
``ValueError`` (the reference throws ``std::invalid_argument``,
src/cagra.cpp:26-32,100-111); device and communication errors raise
``RuntimeError`` (src/metal_context.mm:146-147,245-246).

Inputs may be numpy arrays (host memory) or CUDA tensors exposing
``data_ptr()`` (device memory); results come back in the same kind of memory
the caller provides, or as new numpy arrays.

The compiled engine (lib/libcuvs_b200.so) is required; there is no CPU
fallback: importing this module on a machine without the library raises.
"""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libcuvs_b200.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "cuvs_b200.h")

KNN_OK = 0
KNN_EINVAL = 1
KNN_ECUDA = 2
KNN_ENCCL = 3
KNN_ETIMEOUT = 4
KNN_ENOMEM = 5
KNN_EUNSUPPORTED = 6
DTYPE_F32 = 0
DTYPE_F16 = 1
DTYPE_BF16 = 2
METRIC_L2_EXPANDED = 0
METRIC_INNER_PRODUCT = 1
FILE_FVECS = 0
FILE_BIN_F32 = 1
NO_INDEX = 0xFFFFFFFF
MAX_K = 256


class KnnPlan(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in (
        "query_block", "query_tiles", "row_tiles", "splits", "units", "grid",
        "stages", "smem_bytes", "partial_bytes", "pair", "unit_queries",
        "compact_heap")]


PAGES_MAX_POOLS = 8


class KnnPages(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("rows", ctypes.c_void_p), ("refs", ctypes.c_void_p),
                ("status", ctypes.c_void_p), ("pools", ctypes.c_void_p * PAGES_MAX_POOLS),
                ("row_bytes", ctypes.c_int64 * PAGES_MAX_POOLS), ("sequences", ctypes.c_int64),
                ("columns", ctypes.c_int64), ("pages", ctypes.c_int64),
                ("page_rows", ctypes.c_int32), ("n_pools", ctypes.c_int32),
                ("device", ctypes.c_int32)]


class KnnQ4Rows(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("zeros", ctypes.c_void_p),
                ("norms", ctypes.c_void_p), ("n_rows", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("group", ctypes.c_int32), ("scale_dtype", ctypes.c_int32),
                ("device", ctypes.c_int32), ("pages", ctypes.POINTER(KnnPages))]


_lib = None


def lib() -> ctypes.CDLL:
    """Loads lib/libcuvs_b200.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build the CUDA engine first "
                           "(python -c 'import __graft_entry__ as g; g.build()')")
    L = ctypes.CDLL(LIB_PATH)
    P, I64, I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    sig = {
        "knn_last_error": (ctypes.c_char_p, []),
        "knn_status_string": (ctypes.c_char_p, [I]),
        "knn_index_create": (I, [I, ctypes.POINTER(P)]),
        "knn_index_destroy": (I, [P]),
        "knn_index_set_stream": (I, [P, P]),
        "knn_index_build": (I, [P, P, I, I64, I64, I]),
        "knn_index_build_shard": (I, [P, P, I, I64, I64, I, I64, I64]),
        "knn_index_rows": (I64, [P]),
        "knn_index_dim": (I64, [P]),
        "knn_index_copy_rows": (I, [P, P, I]),
        "knn_index_search": (I, [P, P, I64, I64, P, P]),
        "knn_index_search_i64": (I, [P, P, I64, I64, P, P]),
        "knn_index_search_async": (I, [P, P, I64, I64, P, P]),
        "knn_index_sync": (I, [P]),
        "knn_plan_search": (I, [I64, I64, I64, I64, I, ctypes.POINTER(KnnPlan)]),
        "knn_shard_range": (I, [I64, I, I, ctypes.POINTER(I64), ctypes.POINTER(I64)]),
        "knn_comm_unique_id": (I, [P]),
        "knn_index_attach_comm": (I, [P, P, I, I]),
        "knn_index_set_profiling": (I, [P, I]),
        "knn_index_set_graphs": (I, [P, I]),
        "knn_index_set_peer_exchange": (I, [P, I]),
        "knn_index_set_peer_timeout": (I, [P, I64]),
        "knn_index_device": (I, [P]),
        "knn_index_device_rows": (I, [P, ctypes.POINTER(P), ctypes.POINTER(I64)]),
        "knn_index_device_norms": (I, [P, ctypes.POINTER(P)]),
        "knn_index_build_prepared": (I, [P, P, P, I64, I64, I, I64, I64]),
        "knn_index_search_lists": (I, [P, P, I64, I64, P, P]),
        "knn_merge_lists": (I, [I, P, P, P, I, I64, I64, I, P, I, P]),
        "knn_index_kernel_stats": (I, [P, ctypes.POINTER(ctypes.c_double),
                                       ctypes.POINTER(ctypes.c_double),
                                       ctypes.POINTER(I64), ctypes.POINTER(I64)]),
        "knn_index_reset_kernel_stats": (I, [P]),
        "knn_index_set_rerank": (I, [P, I]),
        "knn_index_build_file": (I, [P, ctypes.c_char_p, I, I, I, I]),
        "knn_rerank_bound": (ctypes.c_double, [I, ctypes.c_double, ctypes.c_double,
                                               ctypes.c_double, I64]),
        "knn_index_rerank_stats": (I, [P, ctypes.POINTER(I64), ctypes.POINTER(I64)]),
        "knn_index_search_noalloc": (I, [P, P, I64, I64, P, P]),
        "knn_selftest_bounded_wait": (I, [I, I64]),
        "knn_pages_grow": (I, [P, P, P, I64, I64, P]),
        "knn_pages_free": (I, [P, P, I64, P]),
        "knn_pages_copy": (I, [P, P, P, I64, P]),
        "knn_pages_fork": (I, [P, P, P, I64, P]),
        "knn_pages_compact_workspace": (I64, [P, I64, I64]),
        "knn_pages_compact": (I, [P, P, P, I64, P, I64, I64, P, P]),
        "knn_q4_row_bytes": (I64, [I64]),
        "knn_q4_pack": (I, [P, P, I, I64, I64, I64, P]),
        "knn_q4_append": (I, [P, P, P, I64, P, I, I64, I64, P]),
        "knn_q4_read": (I, [P, P, P, I64, I64, I64, P, I64, P]),
        "knn_q4_products": (I, [P, I64, I64, P, I, I64, I64, P, I, I64, P]),
        "knn_q4_search_workspace": (I64, [I64, I64]),
        "knn_q4_search": (I, [P, I64, I64, P, I, I64, I64, I64, I, P, P, P, P]),
        "knn_dispatch_count": (ctypes.c_uint64, []),
        "knn_reset_dispatch_count": (None, []),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def header_functions() -> list[str]:
    """Names of every function include/cuvs_b200.h declares."""
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(knn_[a-z0-9_]+)\s*\(", text)))


def _check(status: int) -> None:
    if status == KNN_OK:
        return
    msg = lib().knn_last_error().decode(errors="replace")
    name = lib().knn_status_string(status).decode()
    if status == KNN_EINVAL:
        raise ValueError(f"{name}: {msg}")
    raise RuntimeError(f"{name}: {msg}")


def plan_search(n_rows: int, dim: int, n_queries: int, k: int, num_sms: int = 148) -> dict:
    p = KnnPlan()
    _check(lib().knn_plan_search(n_rows, dim, n_queries, k, num_sms, ctypes.byref(p)))
    return {n: getattr(p, n) for n, _ in KnnPlan._fields_}


def shard_range(n_rows: int, n_ranks: int, rank: int) -> tuple[int, int]:
    b, e = ctypes.c_int64(), ctypes.c_int64()
    _check(lib().knn_shard_range(n_rows, n_ranks, rank, ctypes.byref(b), ctypes.byref(e)))
    return b.value, e.value


def comm_unique_id() -> bytes:
    buf = ctypes.create_string_buffer(128)
    _check(lib().knn_comm_unique_id(buf))
    return buf.raw


def dispatch_count() -> int:
    return int(lib().knn_dispatch_count())


def reset_dispatch_count() -> None:
    lib().knn_reset_dispatch_count()


def _ptr(x):
    """(pointer, keepalive) for a numpy array or a tensor with data_ptr()."""
    if hasattr(x, "data_ptr"):
        if not x.is_contiguous():
            raise ValueError("tensors must be contiguous")
        return ctypes.c_void_p(x.data_ptr()), x
    a = np.ascontiguousarray(x)
    return ctypes.c_void_p(a.ctypes.data), a


def _shape(x):
    return tuple(int(s) for s in x.shape)


def _dtype_code(x) -> int:
    name = str(x.dtype)
    if name.endswith("float32"):
        return DTYPE_F32
    if name.endswith("float16"):
        return DTYPE_F16
    raise ValueError(f"dataset dtype {name} is not float32 or float16")


class Index:
    """Exact brute-force index on one B200 (or one row shard of a dataset).

    The index owns the fp16 rows and fp32 row norms in HBM (filled at build
    time); the reference computed them lazily at the first search and cached
    them by raw pointer (src/metal_context.mm:155-175).
    """

    def __init__(self, device: int = 0):
        h = ctypes.c_void_p()
        _check(lib().knn_index_create(device, ctypes.byref(h)))
        self._h = h
        self.device = device

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            lib().knn_index_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def rows(self) -> int:
        return int(lib().knn_index_rows(self._h))

    @property
    def dim(self) -> int:
        return int(lib().knn_index_dim(self._h))

    def copy_rows(self, dtype=np.float32) -> np.ndarray:
        """The stored (fp16-rounded) rows, as a host array."""
        out = np.empty((self.rows, self.dim), dtype=dtype)
        code = DTYPE_F32 if out.dtype == np.float32 else DTYPE_F16
        _check(lib().knn_index_copy_rows(self._h, ctypes.c_void_p(out.ctypes.data), code))
        return out

    def set_stream(self, stream_handle: int | None) -> None:
        _check(lib().knn_index_set_stream(self._h, ctypes.c_void_p(stream_handle or 0)))

    def build(self, dataset, metric: int = METRIC_L2_EXPANDED, row_offset: int = 0,
              total_rows: int | None = None) -> "Index":
        if len(_shape(dataset)) != 2:
            raise ValueError("dataset must be 2-D")
        n, d = _shape(dataset)
        ptr, keep = _ptr(dataset)
        code = _dtype_code(keep)
        if row_offset == 0 and total_rows is None:
            _check(lib().knn_index_build(self._h, ptr, code, n, d, metric))
        else:
            total = n + row_offset if total_rows is None else total_rows
            _check(lib().knn_index_build_shard(self._h, ptr, code, n, d, metric,
                                               row_offset, total))
        return self

    def build_file(self, path: str, fmt: int = FILE_FVECS, metric: int = METRIC_L2_EXPANDED,
                   n_ranks: int = 1, rank: int = 0) -> None:
        """Streams a dataset file (FILE_FVECS or FILE_BIN_F32) into the index;
        with n_ranks > 1 only this rank's row shard is read."""
        _check(lib().knn_index_build_file(self._h, os.fsencode(path), fmt, metric,
                                          n_ranks, rank))

    def attach_comm(self, unique_id: bytes, n_ranks: int, rank: int) -> None:
        buf = ctypes.create_string_buffer(bytes(unique_id), 128)
        _check(lib().knn_index_attach_comm(self._h, buf, n_ranks, rank))

    def search(self, queries, k: int, neighbors=None, distances=None, int64: bool = False):
        """Exact k-NN; returns (neighbors, distances) of shape (n_queries, k)."""
        shp = _shape(queries)
        if len(shp) != 2:
            raise ValueError("queries must be 2-D")
        nq = shp[0]
        if neighbors is None:
            neighbors = np.empty((nq, k), dtype=np.int64 if int64 else np.uint32)
        if distances is None:
            distances = np.empty((nq, k), dtype=np.float32)
        if _shape(neighbors) != (nq, k) or _shape(distances) != (nq, k):
            # reference: src/cagra.cpp:107-111
            raise ValueError("output shape mismatch")
        if shp[1] != self.dim and self.rows > 0:
            # reference: src/cagra.cpp:104-106
            raise ValueError("query dimension mismatch")
        if not hasattr(queries, "data_ptr"):
            queries = np.ascontiguousarray(queries, dtype=np.float32)
        qp, qk = _ptr(queries)
        ip, ik = _ptr(neighbors)
        dp, dk = _ptr(distances)
        fn = lib().knn_index_search_i64 if int64 else lib().knn_index_search
        _check(fn(self._h, qp, nq, k, ip, dp))
        return neighbors, distances

    def search_async(self, queries, k: int, neighbors, distances) -> None:
        qp, _ = _ptr(queries)
        ip, _ = _ptr(neighbors)
        dp, _ = _ptr(distances)
        _check(lib().knn_index_search_async(self._h, qp, _shape(queries)[0], k, ip, dp))

    def sync(self) -> None:
        _check(lib().knn_index_sync(self._h))

    def set_rerank(self, on: bool) -> None:
        """Exact fp32 re-ranking (call before build; see knn_index_set_rerank)."""
        _check(lib().knn_index_set_rerank(self._h, 1 if on else 0))

    def rerank_stats(self) -> dict:
        """{'uncertified': queries of the last search not proven exact,
        'widened': queries searched again with more candidates}."""
        u, w = ctypes.c_int64(), ctypes.c_int64()
        _check(lib().knn_index_rerank_stats(self._h, ctypes.byref(u), ctypes.byref(w)))
        return {"uncertified": u.value, "widened": w.value}

    def set_peer_exchange(self, on: bool) -> None:
        _check(lib().knn_index_set_peer_exchange(self._h, 1 if on else 0))

    def set_peer_timeout(self, seconds: float) -> None:
        """Bound of the peer-exchange wait (every rank must issue each search
        within it of the others; see knn_index_set_peer_timeout)."""
        _check(lib().knn_index_set_peer_timeout(self._h, int(round(seconds * 1e6))))

    def set_graphs(self, on: bool) -> None:
        _check(lib().knn_index_set_graphs(self._h, 1 if on else 0))

    def set_profiling(self, on: bool) -> None:
        _check(lib().knn_index_set_profiling(self._h, 1 if on else 0))

    def kernel_stats(self) -> dict:
        a, b = ctypes.c_double(), ctypes.c_double()
        c, d = ctypes.c_int64(), ctypes.c_int64()
        _check(lib().knn_index_kernel_stats(self._h, ctypes.byref(a), ctypes.byref(b),
                                            ctypes.byref(c), ctypes.byref(d)))
        return {"scan_ms": a.value, "merge_ms": b.value, "scan_launches": c.value,
                "kernel_launches": d.value}

    def reset_kernel_stats(self) -> None:
        _check(lib().knn_index_reset_kernel_stats(self._h))


# ---------------------------------------------------------------- row store
# Rows in 4 bits, and pages of rows.  Everything here takes CUDA tensors of one
# device, works on that device's current torch stream without synchronising,
# and can be captured into a CUDA graph.

PAGES_ERRORS = {1: "a sequence or page that does not exist",
                2: "a target listed twice, or as a source too",
                3: "a fork's child or a compaction's target holds rows",
                4: "counts below 0, above the length, or not the total",
                5: "more pages than the table has columns",
                6: "too few free pages"}


def _on_device(name, t, device, dtype=None, shape=None, dense=True):
    """Refuses a tensor that a kernel could not take."""
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _list(name, t, device):
    # one test where nothing is wrong: this is most of what a small call costs here
    if not (getattr(t, "is_cuda", False) and t.dtype is _torch().int32 and t.dim() == 1
            and t.device == device and t.is_contiguous()):
        _on_device(name, t, device, _torch().int32)
        raise ValueError(f"{name} must be a list of int32")
    return t


def _two_lists(names, a, b, device):
    _list(names[0], a, device)
    _list(names[1], b, device)
    if a.shape != b.shape:
        raise ValueError(f"{names[0]} and {names[1]} differ in length")


_torch_module = None
_raw_stream = None


def _torch():
    """torch, which only the row store needs."""
    global _torch_module, _raw_stream
    if _torch_module is None:
        import torch

        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _torch_module = torch
    return _torch_module


def _stream(device) -> int:
    """The device's current torch stream."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return _torch().cuda.current_stream(device).cuda_stream


def _float_code(name, dtype) -> int:
    torch = _torch()
    if dtype is torch.float32:
        return DTYPE_F32
    if dtype is torch.float16:
        return DTYPE_F16
    if dtype is torch.bfloat16:
        return DTYPE_BF16
    raise ValueError(f"{name} of {dtype}: not float32, float16 or bfloat16")


def _rows_of(name, t, device, dim):
    """A matrix of vectors (or one vector) of floats whose values lie side by side."""
    if not getattr(t, "is_cuda", False) or t.device != device:
        _on_device(name, t, device, dense=False)
    code = _float_code(name, t.dtype)
    shape = t.shape
    flat = len(shape) == 1
    if (not flat and len(shape) != 2) or shape[-1] != dim:
        raise ValueError(f"{name} has shape {tuple(shape)}, not (n, {dim})")
    n = 1 if flat else shape[0]
    ld = dim if n == 1 else t.stride(0)
    if (dim > 1 and t.stride(-1) != 1) or ld < dim and n > 0:
        raise ValueError(f"{name}: the values of a row must lie side by side, rows apart")
    return n, ld, code


class Pages:
    """Sequences of rows in pages, over the caller's tensors (nothing is
    copied; they stay alive with this object):

    table  int32 [sequences, columns]: page numbers, -1 where there is none
    rows   int32 [sequences]: lengths
    refs   int32 [pages]: table entries that hold the page; 0: free
    pools  up to 8 tensors [pages, page_rows, ...]: the rows' contents

    ``Pages.empty`` makes the first three.  Lists are int32 CUDA tensors.  A
    call that breaks a rule that only the device can see (an index out of
    range, a target listed twice, too few free pages, ...) changes nothing and
    leaves a note that ``check`` raises; see knn_pages_* in the C header.
    """

    def __init__(self, table, rows, refs, pools):
        torch = _torch()
        _on_device("table", table, None, torch.int32)
        device = table.device
        if table.dim() != 2:
            raise ValueError("table must be 2-D")
        _on_device("rows", rows, device, torch.int32, (table.shape[0],))
        _on_device("refs", refs, device, torch.int32)
        if refs.dim() != 1:
            raise ValueError("refs must be 1-D")
        pools = list(pools)
        if len(pools) > PAGES_MAX_POOLS:
            raise ValueError(f"{len(pools)} pools: at most {PAGES_MAX_POOLS}")
        if not pools:
            raise ValueError("at least one pool")
        c = KnnPages(table=table.data_ptr(), rows=rows.data_ptr(), refs=refs.data_ptr())
        for k, t in enumerate(pools):
            _on_device(f"pool {k}", t, device)
            if t.dim() < 2 or t.shape[0] != refs.shape[0] or t.shape[1] != pools[0].shape[1]:
                raise ValueError(f"pool {k} has shape {tuple(t.shape)}, not (pages, page_rows, ...)")
            c.pools[k] = t.data_ptr()
            c.row_bytes[k] = t[0, 0].numel() * t.element_size() if t.numel() else 0
        self.status = torch.zeros(2, dtype=torch.int32, device=device)
        c.status = self.status.data_ptr()
        c.sequences, c.columns = table.shape
        c.pages, c.page_rows, c.n_pools = refs.shape[0], pools[0].shape[1], len(pools)
        c.device = device.index
        self.table, self.rows, self.refs, self.pools, self.device = table, rows, refs, pools, device
        self.page_rows = int(c.page_rows)
        self._c = c
        self._ref = ctypes.byref(c)
        # the C checks of sizes, once
        _check(lib().knn_pages_free(self._ref, None, 0, None))

    @classmethod
    def empty(cls, pools, sequences: int, columns: int):
        """A store of empty sequences over the given pools."""
        torch = _torch()
        pools = list(pools)
        if not pools or not getattr(pools[0], "is_cuda", False):
            raise ValueError("pools must be CUDA tensors")
        if sequences < 1 or columns < 1:
            raise ValueError("a store has at least one sequence and one column")
        new = dict(dtype=torch.int32, device=pools[0].device)
        return cls(torch.full((sequences, columns), -1, **new), torch.zeros(sequences, **new),
                   torch.zeros(pools[0].shape[0], **new), pools)

    def grow(self, seqs, counts) -> None:
        """Room for counts[i] more rows at the end of sequence seqs[i]."""
        _two_lists(("seqs", "counts"), seqs, counts, self.device)
        _check(lib().knn_pages_grow(self._ref, seqs.data_ptr(), counts.data_ptr(), seqs.shape[0], -1,
                                    _stream(self.device)))

    def free(self, seqs) -> None:
        """Empties the listed sequences."""
        _list("seqs", seqs, self.device)
        _check(lib().knn_pages_free(self._ref, seqs.data_ptr(), seqs.shape[0], _stream(self.device)))

    def copy(self, sources, targets) -> None:
        """Copies page sources[i] onto page targets[i] in every pool."""
        _two_lists(("sources", "targets"), sources, targets, self.device)
        _check(lib().knn_pages_copy(self._ref, sources.data_ptr(), targets.data_ptr(),
                                    sources.shape[0], _stream(self.device)))

    def fork(self, parents, children) -> None:
        """Makes the empty sequences children[i] copies of parents[i]: full
        pages are shared, a part-filled last page is copied."""
        _two_lists(("parents", "children"), parents, children, self.device)
        _check(lib().knn_pages_fork(self._ref, parents.data_ptr(), children.data_ptr(),
                                    parents.shape[0], _stream(self.device)))

    def compact(self, sources, targets, keep) -> None:
        """targets[i] (empty, or sources[i] itself) becomes the rows j of
        sources[i] with keep[i, j], in order, in fresh pages."""
        torch = _torch()
        _two_lists(("sources", "targets"), sources, targets, self.device)
        _on_device("keep", keep, self.device, dense=False)
        n = sources.shape[0]
        if keep.dtype not in (torch.bool, torch.uint8) or keep.dim() != 2 or keep.shape[0] != n:
            raise ValueError(f"keep must be bool or uint8 of shape ({n}, rows)")
        columns = keep.shape[1]
        stride = keep.stride(0) if n > 1 else columns
        if (columns > 1 and keep.stride(1) != 1) or stride < columns:
            raise ValueError("keep: the flags of a sequence must lie side by side, sequences apart")
        work = torch.empty(max(1, lib().knn_pages_compact_workspace(self._ref, n, columns)),
                           dtype=torch.uint8, device=self.device)
        _check(lib().knn_pages_compact(self._ref, sources.data_ptr(), targets.data_ptr(), n,
                                       keep.data_ptr(), columns, stride, work.data_ptr(),
                                       _stream(self.device)))

    def check(self) -> None:
        """Waits for the store's calls; raises the first error that one of
        them found (and forgets it)."""
        error = int(self.status[0].item())
        if error:
            self.status[0] = 0
            raise ValueError(f"row store: {PAGES_ERRORS.get(error, error)}")


class Q4Rows:
    """Rows in 4 bits, over the caller's tensors:

    codes   uint8 [n, 16 * ceil(dim / 32)], two codes a byte, the first low
    scales  float16 or bfloat16 [n, ceil(dim / group)], group 32, 64 or 128
    zeros   uint8 like scales, or None: 8 throughout
    norms   float32 [n], |row|^2 to (dim / 256 + 16) 2^-24 of it, as packing makes
            them, or None (only needed to search by L2)

    ``value = (code - zero) * scale``.  With ``pages`` the tensors are pools
    [pages, page_rows, ...] of that store, all of them, and calls name a sequence.
    """

    def __init__(self, codes, scales, dim: int, group: int, zeros=None, norms=None, pages=None):
        torch = _torch()
        _on_device("codes", codes, None, torch.uint8)
        device, lead = codes.device, tuple(codes.shape[:-1])
        if dim < 1 or group not in (32, 64, 128):
            raise ValueError(f"rows of {dim} values in groups of {group}")
        groups, width = -(-dim // group), 16 * (-(-dim // 32))
        if pages is not None and lead != (pages.refs.shape[0], pages.page_rows):
            raise ValueError(f"codes have shape {tuple(codes.shape)}, not (pages, page_rows, {width})")
        if pages is None and len(lead) != 1:
            raise ValueError(f"codes have shape {tuple(codes.shape)}, not (n, {width})")
        if pages is not None and pages.device != device:
            raise ValueError(f"the pages are on {pages.device}, the codes on {device}")
        _on_device("codes", codes, device, torch.uint8, lead + (width,))
        _on_device("scales", scales, device, None, lead + (groups,))
        if scales.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"scales of {scales.dtype}: not float16 or bfloat16")
        if zeros is not None:
            _on_device("zeros", zeros, device, torch.uint8, lead + (groups,))
        if norms is not None:
            _on_device("norms", norms, device, torch.float32, lead)
        c = KnnQ4Rows(codes=codes.data_ptr(), scales=scales.data_ptr(), dim=dim, group=group,
                      device=device.index)
        c.zeros = zeros.data_ptr() if zeros is not None else None
        c.norms = norms.data_ptr() if norms is not None else None
        c.scale_dtype = DTYPE_F16 if scales.dtype is torch.float16 else DTYPE_BF16
        c.n_rows = lead[0] if pages is None else lead[0] * lead[1]
        if pages is not None:
            c.pages = ctypes.pointer(pages._c)
        self.codes, self.scales, self.zeros, self.norms, self.pages = codes, scales, zeros, norms, pages
        self.dim, self.group, self.device, self.n_rows = dim, group, device, int(c.n_rows)
        self._c = c
        self._ref = ctypes.byref(c)
        # the C checks of sizes, once
        _check(lib().knn_q4_products(self._ref, -1 if pages is None else 0, 0, None, 0, 0, 0, None, 0,
                                     0, None))

    def _range(self, seq, count):
        if self.pages is None:
            if seq is not None:
                raise ValueError("dense rows have no sequences")
            return -1, self.n_rows if count is None else count
        if seq is None or count is None:
            raise ValueError("rows in pages need seq and count")
        return seq, count

    def append(self, seqs, counts, rows) -> None:
        """Quantises ``rows``, counts[i] of them for the end of seqs[i], those
        of seqs[0] first (Pages.grow, then the rows)."""
        if self.pages is None:
            raise ValueError("dense rows do not grow")
        _two_lists(("seqs", "counts"), seqs, counts, self.device)
        n, ld, dtype = _rows_of("rows", rows, self.device, self.dim)
        _check(lib().knn_q4_append(self._ref, seqs.data_ptr(), counts.data_ptr(), seqs.shape[0],
                                   rows.data_ptr(), dtype, n, ld, _stream(self.device)))

    def read(self, seqs=None, counts=None, total=None, first: int = 0):
        """The values of rows, float32: rows first .. first + total - 1 of dense
        rows, or the last counts[i] rows of seqs[i], ``total`` in all."""
        torch = _torch()
        if self.pages is None:
            if seqs is not None or counts is not None:
                raise ValueError("dense rows have no sequences")
            total = self.n_rows - first if total is None else total
            if total < 0:
                raise ValueError(f"{total} rows")
            out = torch.empty((total, self.dim), dtype=torch.float32, device=self.device)
            _check(lib().knn_q4_read(self._ref, None, None, 0, first, total, out.data_ptr(), self.dim,
                                     _stream(self.device)))
            return out
        if seqs is None or counts is None or total is None or total < 0:
            raise ValueError("rows in pages need seqs, counts and their total")
        _two_lists(("seqs", "counts"), seqs, counts, self.device)
        out = torch.empty((total, self.dim), dtype=torch.float32, device=self.device)
        _check(lib().knn_q4_read(self._ref, seqs.data_ptr(), counts.data_ptr(), seqs.shape[0], first,
                                 total, out.data_ptr(), self.dim, _stream(self.device)))
        return out

    def products(self, x, seq=None, count=None, out=None, dtype=None):
        """x [batch, dim] (or one vector) times rows 0 .. count - 1: [batch,
        count] in ``dtype`` (float32 unless given).  In pages: of sequence
        ``seq``, 0 beyond its length.  Products have no gradient: an x (or out)
        that requires one is refused, unless under torch.no_grad()."""
        torch = _torch()
        seq, count = self._range(seq, count)
        n, ldx, code = _rows_of("x", x, self.device, self.dim)
        if (x.requires_grad or out is not None and out.requires_grad) and torch.is_grad_enabled():
            raise ValueError("x requires a gradient, which products do not have: detach it, or call under "
                             "torch.no_grad()")
        if count < 0 or count > self.n_rows:
            raise ValueError(f"{count} of {self.n_rows} rows")
        shape = (n, count) if x.dim() == 2 else (count,)
        if out is None:
            dtype = dtype or torch.float32
            out_code, ldo = _float_code("dtype", dtype), count
            out = torch.empty(shape, dtype=dtype, device=self.device)
        else:
            if dtype is not None and out.dtype is not dtype:
                raise ValueError(f"out is {out.dtype}, not {dtype}")
            if tuple(out.shape) != shape:
                raise ValueError(f"out has shape {tuple(out.shape)}, not {shape}")
            _, ldo, out_code = _rows_of("out", out, self.device, count)
        _check(lib().knn_q4_products(self._ref, seq, count, x.data_ptr(), code, n, ldx, out.data_ptr(),
                                     out_code, ldo, _stream(self.device)))
        return out

    def search(self, queries, k: int, metric: int = METRIC_L2_EXPANDED, seq=None, count=None):
        """The k nearest rows of each query: (neighbors int64, distances
        float32, which have no gradient), as Index.search orders and pads them."""
        torch = _torch()
        seq, count = self._range(seq, count)
        n, ld, code = _rows_of("queries", queries, self.device, self.dim)
        if queries.dim() != 2:
            raise ValueError("queries must be 2-D")
        if k < 1 or k > MAX_K:
            raise ValueError(f"k = {k}: 1 to {MAX_K}")
        if count < 0 or count > self.n_rows:
            raise ValueError(f"{count} of {self.n_rows} rows")
        neighbors = torch.empty((n, k), dtype=torch.int64, device=self.device)
        distances = torch.empty((n, k), dtype=torch.float32, device=self.device)
        work = torch.empty(lib().knn_q4_search_workspace(count, n), dtype=torch.uint8, device=self.device)
        _check(lib().knn_q4_search(self._ref, seq, count, queries.data_ptr(), code, n, ld, k, metric,
                                   neighbors.data_ptr(), distances.data_ptr(), work.data_ptr(),
                                   _stream(self.device)))
        return neighbors, distances


def q4_pack(rows, group: int = 64, zero_points: bool = False, scale_dtype=None) -> Q4Rows:
    """Quantises rows [n, dim] (float32, float16 or bfloat16) to 4 bits with a
    scale (float16 unless ``scale_dtype`` says bfloat16), and where asked a
    zero point, for every ``group`` values; see knn_q4_pack in the C header."""
    torch = _torch()
    if getattr(rows, "ndim", 0) != 2 or rows.shape[1] < 1 or group not in (32, 64, 128):
        raise ValueError("rows must be 2-D, in groups of 32, 64 or 128")
    n, dim = rows.shape
    _, ld, code = _rows_of("rows", rows, rows.device, dim)
    groups, new = -(-dim // group), dict(device=rows.device)
    out = Q4Rows(torch.empty((n, 16 * (-(-dim // 32))), dtype=torch.uint8, **new),
                 torch.empty((n, groups), dtype=scale_dtype or torch.float16, **new), dim, group,
                 torch.empty((n, groups), dtype=torch.uint8, **new) if zero_points else None,
                 torch.empty(n, dtype=torch.float32, **new))
    _check(lib().knn_q4_pack(out._ref, rows.data_ptr(), code, n, ld, 0, _stream(out.device)))
    return out


# ------------------------------------------------------------ dataset files
# numpy readers and writers of the formats knn_index_build_file streams and
# the C++ loaders (include/cuvs_silicon/sift_loader.hpp) read.

def write_fvecs(path: str, rows) -> None:
    rows = np.ascontiguousarray(rows, dtype=np.float32)
    rec = np.empty((rows.shape[0], rows.shape[1] + 1), dtype=np.float32)
    rec[:, 0] = np.array([rows.shape[1]], dtype=np.int32).view(np.float32)[0]
    rec[:, 1:] = rows
    rec.tofile(path)


def read_fvecs(path: str) -> np.ndarray:
    raw = np.fromfile(path, dtype=np.int32)
    if raw.size == 0:
        return np.empty((0, 0), np.float32)
    dim = int(raw[0])
    if dim <= 0 or raw.size % (dim + 1):
        raise ValueError(f"{path}: not an fvecs file")
    rec = raw.reshape(-1, dim + 1)
    if np.any(rec[:, 0] != dim):
        raise ValueError(f"{path}: rows of different widths")
    return rec[:, 1:].view(np.float32).copy()


def write_bin(path: str, matrix) -> None:
    m = np.ascontiguousarray(matrix)
    if m.dtype not in (np.float32, np.int32):
        raise ValueError("bin matrices hold float32 or int32")
    with open(path, "wb") as f:
        np.array(m.shape, dtype=np.int32).tofile(f)
        m.tofile(f)


def read_bin(path: str, dtype=np.float32) -> np.ndarray:
    raw = np.fromfile(path, dtype=np.int32)
    rows, cols = int(raw[0]), int(raw[1])
    if rows < 0 or cols < 0 or raw.size != 2 + rows * cols:
        raise ValueError(f"{path}: shape {rows} x {cols} does not match the file")
    return raw[2:].view(dtype).reshape(rows, cols).copy()


def rerank_bound(metric: int, r: float, query_norm: float, row_norm: float, dim: int) -> float:
    """The exact re-rank certificate's bound (knn_rerank_bound)."""
    return float(lib().knn_rerank_bound(metric, r, query_norm, row_norm, dim))
