// knn_store_capi.cu -- C entry points of the row store (include/cuvs_b200.h):
// checks of what the host can see, then launches.  What only the device sees
// (indices, counts, free pages) is checked by the kernels.
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "knn_q4.h"

using knn::store_fail;

namespace {

int fail(int status, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return store_fail(status, buf);
}

// Makes `device` current for a call and puts the thread's own back.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    error_ = cudaGetDevice(&before_);
    if (error_ == cudaSuccess && before_ != device) {
      error_ = cudaSetDevice(device);
      back_ = error_ == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (back_) cudaSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  cudaError_t error() const { return error_; }

 private:
  int before_ = 0;
  bool back_ = false;
  cudaError_t error_;
};

int done(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return KNN_OK;
  return fail(KNN_ECUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

// An address that a kernel could not load a value of `size` bytes from would
// fault the GPU.
bool aligned(const void* p, int64_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }
int64_t size_of(int dtype) { return dtype == KNN_DTYPE_F32 ? 4 : 2; }

int check_pages(const char* what, const knn_pages* p) {
  if (!p) return fail(KNN_EINVAL, "%s: null pages", what);
  if (!p->table || !p->rows || !p->refs || !p->status)
    return fail(KNN_EINVAL, "%s: null table, rows, refs or status", what);
  if (!aligned(p->table, 4) || !aligned(p->rows, 4) || !aligned(p->refs, 4) || !aligned(p->status, 4))
    return fail(KNN_EINVAL, "%s: table, rows, refs and status must be 4-byte aligned", what);
  if (p->sequences < 1 || p->sequences > KNN_PAGES_MAX_SEQUENCES || p->columns < 1 ||
      p->columns > KNN_PAGES_MAX_PAGES || p->pages < 1 || p->pages > KNN_PAGES_MAX_PAGES ||
      p->page_rows < 1 || p->pages * static_cast<int64_t>(p->page_rows) > 0x7fffffffLL)
    return fail(KNN_EINVAL, "%s: %lld sequences x %lld columns, %lld pages of %d rows", what,
                (long long)p->sequences, (long long)p->columns, (long long)p->pages,
                p->page_rows);
  if (p->n_pools < 0 || p->n_pools > KNN_PAGES_MAX_POOLS)
    return fail(KNN_EINVAL, "%s: %d pools", what, p->n_pools);
  for (int k = 0; k < p->n_pools; ++k)
    if (!p->pools[k] || p->row_bytes[k] < 1 || p->row_bytes[k] > (1 << 24))
      return fail(KNN_EINVAL, "%s: pool %d is null or has rows of %lld bytes", what, k,
                  (long long)p->row_bytes[k]);
  return KNN_OK;
}

int check_list(const char* what, int64_t n, int64_t most, const void* a, const void* b) {
  if (n < 0 || n > most)
    return fail(KNN_EINVAL, "%s: a list of %lld (at most %lld)", what, (long long)n,
                (long long)most);
  if (n > 0 && (!a || !b)) return fail(KNN_EINVAL, "%s: null list", what);
  if (n > 0 && (!aligned(a, 4) || !aligned(b, 4)))
    return fail(KNN_EINVAL, "%s: lists must be 4-byte aligned", what);
  return KNN_OK;
}

bool is_dtype(int dtype) {
  return dtype == KNN_DTYPE_F32 || dtype == KNN_DTYPE_F16 || dtype == KNN_DTYPE_BF16;
}

// A buffer of rows in pages is one of the store's pools: what forks, compactions
// and copies move is then all of a row.
bool is_pool(const knn_pages& p, const void* buffer, int64_t row_bytes) {
  for (int k = 0; k < p.n_pools; ++k)
    if (p.pools[k] == buffer && p.row_bytes[k] == row_bytes) return true;
  return false;
}

int check_q4(const char* what, const knn_q4_rows* q) {
  if (!q) return fail(KNN_EINVAL, "%s: null rows", what);
  if (q->dim < 1 || q->dim > KNN_Q4_MAX_DIM || (q->group != 32 && q->group != 64 && q->group != 128))
    return fail(KNN_EINVAL, "%s: rows of %lld values in groups of %d", what, (long long)q->dim,
                q->group);
  if (q->scale_dtype != KNN_DTYPE_F16 && q->scale_dtype != KNN_DTYPE_BF16)
    return fail(KNN_EINVAL, "%s: scales of type %d", what, q->scale_dtype);
  if (q->n_rows < 0 || q->n_rows > 0x7fffffffLL)
    return fail(KNN_EINVAL, "%s: %lld rows", what, (long long)q->n_rows);
  if (q->n_rows > 0 && (!q->codes || !q->scales))
    return fail(KNN_EINVAL, "%s: null codes or scales", what);
  if (!aligned(q->codes, 16) || !aligned(q->scales, 2) || !aligned(q->norms, 4))
    return fail(KNN_EINVAL, "%s: codes must be 16-byte aligned, scales 2-byte, norms 4-byte", what);
  if (q->pages) {
    if (int st = check_pages(what, q->pages)) return st;
    if (q->pages->device != q->device ||
        q->n_rows != q->pages->pages * static_cast<int64_t>(q->pages->page_rows))
      return fail(KNN_EINVAL, "%s: %lld rows do not fill the store's pages", what,
                  (long long)q->n_rows);
    const int64_t groups = (q->dim + q->group - 1) / q->group;
    const char* other = !is_pool(*q->pages, q->codes, knn_q4_row_bytes(q->dim)) ? "codes"
                        : !is_pool(*q->pages, q->scales, 2 * groups)            ? "scales"
                        : q->zeros && !is_pool(*q->pages, q->zeros, groups)     ? "zeros"
                        : q->norms && !is_pool(*q->pages, q->norms, 4)          ? "norms"
                                                                                : nullptr;
    if (other) return fail(KNN_EINVAL, "%s: the %s are no pool of the store", what, other);
  }
  return KNN_OK;
}

knn::Q4View view_of(const knn_q4_rows& q) {
  knn::Q4View v = {};
  v.codes = q.codes;
  v.scales = static_cast<const uint16_t*>(q.scales);
  v.zeros = q.zeros;
  v.norms = q.norms;
  v.dim = q.dim;
  v.group = q.group;
  v.group_shift = q.group == 32 ? 5 : q.group == 64 ? 6 : 7;
  v.groups = static_cast<int32_t>((q.dim + q.group - 1) / q.group);
  v.width = static_cast<int32_t>(knn_q4_row_bytes(q.dim));
  v.scale_bf16 = q.scale_dtype == KNN_DTYPE_BF16;
  if (q.pages)
    v.places = knn::Places{q.pages->table, q.pages->columns, q.pages->pages, q.pages->page_rows};
  else
    v.places = knn::Places{nullptr, 0, 0, 1};
  return v;
}

knn::Q4List list_of(const knn_q4_rows& q, const int32_t* seqs, const int32_t* counts, int64_t n,
                    int64_t first, int64_t total) {
  knn::Q4List l = {};
  l.total = total;
  l.first = first;
  if (q.pages) {
    l.seqs = seqs;
    l.counts = counts;
    l.n = static_cast<int32_t>(n);
    l.rows = q.pages->rows;
    l.sequences = q.pages->sequences;
    l.status = q.pages->status;
  }
  return l;
}

// The rows that a product or search covers.
int range_of(const char* what, const knn_q4_rows& q, int64_t seq, int64_t count,
             knn::Q4Range* out) {
  if (count < 0 || count > q.n_rows)
    return fail(KNN_EINVAL, "%s: %lld of %lld rows", what, (long long)count, (long long)q.n_rows);
  if (q.pages ? seq < 0 || seq >= q.pages->sequences : seq != -1)
    return fail(KNN_EINVAL, "%s: sequence %lld", what, (long long)seq);
  out->seq = q.pages ? seq : 0;
  out->count = count;
  out->length = q.pages ? q.pages->rows + seq : nullptr;
  return KNN_OK;
}

}  // namespace

extern "C" {

int knn_pages_grow(const knn_pages* p, const int32_t* seqs, const int32_t* counts, int64_t n,
                   int64_t total, void* stream) {
  if (int st = check_pages("knn_pages_grow", p)) return st;
  if (int st = check_list("knn_pages_grow", n, KNN_PAGES_MAX_LIST, seqs, counts)) return st;
  if (n == 0 && total <= 0) return KNN_OK;
  if (n == 0) return fail(KNN_EINVAL, "knn_pages_grow: %lld rows for no sequence", (long long)total);
  OnDevice on(p->device);
  if (on.error()) return done("knn_pages_grow", on.error());
  return done("knn_pages_grow", knn::launch_pages_grow(*p, seqs, counts, n, total,
                                                       static_cast<cudaStream_t>(stream)));
}

int knn_pages_free(const knn_pages* p, const int32_t* seqs, int64_t n, void* stream) {
  if (int st = check_pages("knn_pages_free", p)) return st;
  if (int st = check_list("knn_pages_free", n, KNN_PAGES_MAX_LIST, seqs, seqs)) return st;
  if (n == 0) return KNN_OK;
  OnDevice on(p->device);
  if (on.error()) return done("knn_pages_free", on.error());
  return done("knn_pages_free",
              knn::launch_pages_free(*p, seqs, n, static_cast<cudaStream_t>(stream)));
}

int knn_pages_copy(const knn_pages* p, const int32_t* sources, const int32_t* targets, int64_t n,
                   void* stream) {
  if (int st = check_pages("knn_pages_copy", p)) return st;
  if (int st = check_list("knn_pages_copy", n, KNN_PAGES_MAX_PAGES, sources, targets)) return st;
  if (n == 0) return KNN_OK;
  OnDevice on(p->device);
  if (on.error()) return done("knn_pages_copy", on.error());
  return done("knn_pages_copy", knn::launch_pages_copy(*p, sources, targets, n,
                                                       static_cast<cudaStream_t>(stream)));
}

int knn_pages_fork(const knn_pages* p, const int32_t* parents, const int32_t* children, int64_t n,
                   void* stream) {
  if (int st = check_pages("knn_pages_fork", p)) return st;
  if (int st = check_list("knn_pages_fork", n, KNN_PAGES_MAX_LIST, parents, children)) return st;
  if (n == 0) return KNN_OK;
  OnDevice on(p->device);
  if (on.error()) return done("knn_pages_fork", on.error());
  return done("knn_pages_fork", knn::launch_pages_fork(*p, parents, children, n,
                                                       static_cast<cudaStream_t>(stream)));
}

int64_t knn_pages_compact_workspace(const knn_pages* p, int64_t n, int64_t keep_columns) {
  if (!p || n < 0 || n > KNN_PAGES_MAX_LIST || keep_columns < 0 || keep_columns > 0x7fffffffLL ||
      p->columns < 1)
    return -1;
  return 4 * knn::pages_compact_words(*p, n, keep_columns);
}

int knn_pages_compact(const knn_pages* p, const int32_t* sources, const int32_t* targets,
                      int64_t n, const uint8_t* keep, int64_t keep_columns, int64_t keep_stride,
                      void* workspace, void* stream) {
  if (int st = check_pages("knn_pages_compact", p)) return st;
  if (int st = check_list("knn_pages_compact", n, KNN_PAGES_MAX_LIST, sources, targets)) return st;
  if (n == 0) return KNN_OK;
  if (keep_columns < 0 || keep_columns > 0x7fffffffLL || (n > 1 && keep_stride < keep_columns) ||
      (keep_columns > 0 && !keep))
    return fail(KNN_EINVAL, "knn_pages_compact: keep of %lld columns, stride %lld",
                (long long)keep_columns, (long long)keep_stride);
  if (!workspace || !aligned(workspace, 16))
    return fail(KNN_EINVAL, "knn_pages_compact: null or unaligned workspace");
  if (knn::pages_compact_words(*p, n, keep_columns) > 0x7fffffffLL)
    return fail(KNN_EUNSUPPORTED, "knn_pages_compact: %lld sequences of %lld rows in one call",
                (long long)n, (long long)keep_columns);
  OnDevice on(p->device);
  if (on.error()) return done("knn_pages_compact", on.error());
  return done("knn_pages_compact",
              knn::launch_pages_compact(*p, sources, targets, n, keep, keep_columns, keep_stride,
                                        static_cast<int32_t*>(workspace),
                                        static_cast<cudaStream_t>(stream)));
}

int64_t knn_q4_row_bytes(int64_t dim) { return dim < 1 ? 0 : 16 * ((dim + 31) / 32); }

int knn_q4_pack(const knn_q4_rows* q, const void* rows, int dtype, int64_t n, int64_t ld,
                int64_t first, void* stream) {
  if (int st = check_q4("knn_q4_pack", q)) return st;
  if (q->pages) return fail(KNN_EINVAL, "knn_q4_pack: rows in pages are appended");
  if (!is_dtype(dtype)) return fail(KNN_EINVAL, "knn_q4_pack: rows of type %d", dtype);
  if (n < 0 || first < 0 || first > q->n_rows - n)
    return fail(KNN_EINVAL, "knn_q4_pack: rows %lld .. %lld of %lld", (long long)first,
                (long long)(first + n - 1), (long long)q->n_rows);
  if (n == 0) return KNN_OK;
  if (!rows || !aligned(rows, size_of(dtype)) || (n > 1 && ld < q->dim))
    return fail(KNN_EINVAL, "knn_q4_pack: null or unaligned rows, or rows %lld apart", (long long)ld);
  OnDevice on(q->device);
  if (on.error()) return done("knn_q4_pack", on.error());
  return done("knn_q4_pack",
              knn::launch_q4_pack(view_of(*q), list_of(*q, nullptr, nullptr, 0, first, n), rows,
                                  dtype, ld, static_cast<cudaStream_t>(stream)));
}

int knn_q4_append(const knn_q4_rows* q, const int32_t* seqs, const int32_t* counts, int64_t n,
                  const void* rows, int dtype, int64_t total, int64_t ld, void* stream) {
  if (int st = check_q4("knn_q4_append", q)) return st;
  if (!q->pages) return fail(KNN_EINVAL, "knn_q4_append: dense rows do not grow");
  if (int st = check_list("knn_q4_append", n, KNN_PAGES_MAX_LIST, seqs, counts)) return st;
  if (!is_dtype(dtype)) return fail(KNN_EINVAL, "knn_q4_append: rows of type %d", dtype);
  if (total < 0 || total > q->n_rows || (total > 0 && n == 0))
    return fail(KNN_EINVAL, "knn_q4_append: %lld rows for %lld sequences", (long long)total,
                (long long)n);
  if (total > 0 && (!rows || !aligned(rows, size_of(dtype)) || (total > 1 && ld < q->dim)))
    return fail(KNN_EINVAL, "knn_q4_append: null or unaligned rows, or rows %lld apart", (long long)ld);
  if (n == 0) return KNN_OK;
  OnDevice on(q->device);
  if (on.error()) return done("knn_q4_append", on.error());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaError_t e = knn::launch_pages_grow(*q->pages, seqs, counts, n, total, s))
    return done("knn_q4_append", e);
  if (total == 0) return KNN_OK;
  return done("knn_q4_append", knn::launch_q4_pack(view_of(*q), list_of(*q, seqs, counts, n, 0, total),
                                                   rows, dtype, ld, s));
}

int knn_q4_read(const knn_q4_rows* q, const int32_t* seqs, const int32_t* counts, int64_t n,
                int64_t first, int64_t total, float* out, int64_t ld, void* stream) {
  if (int st = check_q4("knn_q4_read", q)) return st;
  if (q->pages) {
    if (int st = check_list("knn_q4_read", n, KNN_PAGES_MAX_LIST, seqs, counts)) return st;
    if (first != 0 || total < 0 || total > 0x7fffffffLL || (total > 0 && n == 0))
      return fail(KNN_EINVAL, "knn_q4_read: %lld rows of %lld sequences", (long long)total,
                  (long long)n);
    if (n == 0) return KNN_OK;
  } else if (seqs || counts || n != 0 || total < 0 || first < 0 || first > q->n_rows - total) {
    return fail(KNN_EINVAL, "knn_q4_read: rows %lld .. %lld of %lld dense rows", (long long)first,
                (long long)(first + total - 1), (long long)q->n_rows);
  }
  if (total == 0 && !q->pages) return KNN_OK;
  if (total > 0 && (!out || !aligned(out, 4) || (total > 1 && ld < q->dim)))
    return fail(KNN_EINVAL, "knn_q4_read: null or unaligned output, or rows %lld apart", (long long)ld);
  OnDevice on(q->device);
  if (on.error()) return done("knn_q4_read", on.error());
  return done("knn_q4_read", knn::launch_q4_read(view_of(*q), list_of(*q, seqs, counts, n, first, total),
                                                 out, ld, static_cast<cudaStream_t>(stream)));
}

int knn_q4_products(const knn_q4_rows* q, int64_t seq, int64_t count, const void* x, int dtype,
                    int64_t batch, int64_t ldx, void* out, int out_dtype, int64_t ldo,
                    void* stream) {
  if (int st = check_q4("knn_q4_products", q)) return st;
  knn::Q4Range r;
  if (int st = range_of("knn_q4_products", *q, seq, count, &r)) return st;
  if (!is_dtype(dtype) || !is_dtype(out_dtype))
    return fail(KNN_EINVAL, "knn_q4_products: types %d and %d", dtype, out_dtype);
  if (batch < 0) return fail(KNN_EINVAL, "knn_q4_products: %lld vectors", (long long)batch);
  if (batch == 0 || count == 0) return KNN_OK;
  if (!x || !out || !aligned(x, size_of(dtype)) || !aligned(out, size_of(out_dtype)) ||
      (batch > 1 && (ldx < q->dim || ldo < count)))
    return fail(KNN_EINVAL, "knn_q4_products: null or unaligned buffer, or rows %lld and %lld apart",
                (long long)ldx, (long long)ldo);
  OnDevice on(q->device);
  if (on.error()) return done("knn_q4_products", on.error());
  return done("knn_q4_products",
              knn::launch_q4_products(view_of(*q), r, x, dtype, batch, ldx, out, out_dtype, ldo,
                                      static_cast<cudaStream_t>(stream)));
}

int64_t knn_q4_search_workspace(int64_t count, int64_t n_queries) {
  return count < 0 || n_queries < 0 ? -1 : 16 + knn::q4_search_bytes(count, n_queries);
}

int knn_q4_search(const knn_q4_rows* q, int64_t seq, int64_t count, const void* queries, int dtype,
                  int64_t n_queries, int64_t ld, int64_t k, int metric, int64_t* neighbors,
                  float* distances, void* workspace, void* stream) {
  if (int st = check_q4("knn_q4_search", q)) return st;
  knn::Q4Range r;
  if (int st = range_of("knn_q4_search", *q, seq, count, &r)) return st;
  if (metric != KNN_METRIC_L2_EXPANDED && metric != KNN_METRIC_INNER_PRODUCT)
    return fail(KNN_EINVAL, "metric %d is not L2Expanded (0) or InnerProduct (1)", metric);
  if (!is_dtype(dtype)) return fail(KNN_EINVAL, "knn_q4_search: queries of type %d", dtype);
  if (k < 1 || k > KNN_MAX_K || n_queries < 0)
    return fail(KNN_EINVAL, "knn_q4_search: k %lld (1 .. %d), %lld queries", (long long)k,
                KNN_MAX_K, (long long)n_queries);
  if (n_queries == 0) return KNN_OK;
  if (metric == KNN_METRIC_L2_EXPANDED && count > 0 && !q->norms)
    return fail(KNN_EINVAL, "knn_q4_search: squared L2 distances need the rows' norms");
  if (!queries || !neighbors || !distances || !workspace || !aligned(queries, size_of(dtype)) ||
      !aligned(neighbors, 8) || !aligned(distances, 4) || !aligned(workspace, 16) ||
      (n_queries > 1 && ld < q->dim))
    return fail(KNN_EINVAL, "knn_q4_search: null or unaligned buffer, or queries %lld apart",
                (long long)ld);
  OnDevice on(q->device);
  if (on.error()) return done("knn_q4_search", on.error());
  return done("knn_q4_search",
              knn::launch_q4_search(view_of(*q), r, queries, dtype, n_queries, ld,
                                    static_cast<int>(k), metric, neighbors, distances, workspace,
                                    static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
