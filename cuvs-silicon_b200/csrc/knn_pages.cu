// knn_pages.cu -- pages of rows: growing, copying, forking, compacting and
// freeing them.
//
// A store is a table of page numbers for every sequence, the sequences'
// lengths in rows, a count of references for every page, and up to
// KNN_PAGES_MAX_POOLS pools [pages][page_rows][row bytes] that share the page
// numbers.  Row j of sequence s is row j % page_rows of page
// table[s][j / page_rows].  A page with no references is free; there is no
// list of free pages that could disagree with the counts.
//
// Fresh pages are always the lowest-numbered free ones, given out in the
// order of the call's list, so that results never depend on the order in
// which threads run.  A call that breaks a rule (an index out of range, a
// target listed twice, too few free pages, ...) changes nothing: the kernel
// that plans it records the error and clears status[1] ("applied"), and the
// kernels that move data check that word first.
//
// What bounds them: planning is a latency (one CTA: a list of a few
// sequences, a scan of the counts; 3 to 8 us), moving rows is HBM bandwidth.
// Measured: 256 MB of pages copied in 80 to 84 us (513 MB moved, 6.2 TB/s), 210 MB of
// kept rows gathered in 76 us (420 MB, 5.5 TB/s); 64 children of sequences of
// 1250 pages forked in 14 us, their freeing included.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "knn_store.h"

namespace knn {

namespace {

// Threads of a plan kernel.  Small calls are a chain of loads and barriers:
// 256 threads go through it faster than 1024 (the plan of a fork 9.3 -> 6.7 us),
// which long lists and many pages need.
constexpr int kFewThreads = 256, kManyThreads = 1024;
constexpr int64_t kFewList = 1024, kFewPages = 32768;
constexpr int kMaxList = KNN_PAGES_MAX_LIST;
constexpr int kMoveThreads = 256;
constexpr int64_t kMoveChunk = 16384;  // bytes of a page that one CTA moves at a time
constexpr int kShareChunk = 1024;      // table entries that one CTA shares at a time
constexpr int kKeepChunk = 64;         // positions of a sequence that one CTA compacts

// ------------------------------------------------------------------- moves
// Copies `bytes` bytes with all threads of the block, 16 at a time where
// both ends allow it.
__device__ __forceinline__ void block_copy(uint8_t* to, const uint8_t* from, int64_t bytes) {
  if (((reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(from)) & 15) == 0) {
    const int64_t n = bytes >> 4;
    const uint4* f = reinterpret_cast<const uint4*>(from);
    uint4* t = reinterpret_cast<uint4*>(to);
    int64_t i = threadIdx.x;
    for (; i + 3 * kMoveThreads < n; i += 4 * kMoveThreads) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __ldcs(f + i + j * kMoveThreads);
#pragma unroll
      for (int j = 0; j < 4; ++j) __stcs(t + i + j * kMoveThreads, v[j]);
    }
    for (; i < n; i += kMoveThreads) __stcs(t + i, __ldcs(f + i));
    for (int64_t b = (n << 4) + threadIdx.x; b < bytes; b += kMoveThreads) to[b] = from[b];
  } else {
    for (int64_t b = threadIdx.x; b < bytes; b += kMoveThreads) to[b] = from[b];
  }
}

// Copies one chunk of one pool of pair i's pages.
__device__ __forceinline__ void copy_item(const knn_pages& p, const int32_t* sources,
                                          const int32_t* targets, int64_t item, int64_t chunks) {
  const int64_t i = item / chunks;
  int64_t chunk = item - i * chunks;
  for (int k = 0; k < p.n_pools; ++k) {
    const int64_t bytes = p.row_bytes[k] * p.page_rows;
    const int64_t parts = (bytes + kMoveChunk - 1) / kMoveChunk;
    if (chunk < parts) {
      uint8_t* pool = static_cast<uint8_t*>(p.pools[k]);
      const int64_t off = chunk * kMoveChunk;
      const int64_t left = bytes - off;
      block_copy(pool + targets[i] * bytes + off, pool + sources[i] * bytes + off,
                 left < kMoveChunk ? left : kMoveChunk);
      break;
    }
    chunk -= parts;
  }
}

// ------------------------------------------------------------ plan kernels
struct PlanSmem {
  unsigned long long part[kManyThreads / 32];
  int bad;
};

// Exclusive prefix sum over the block; *total gets the sum.
template <int kThreads>
__device__ unsigned long long block_exclusive(unsigned long long v, PlanSmem& sm,
                                              unsigned long long* total) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // the last call's readers are done with part
  if (lane == 31) sm.part[warp] = inc;
  __syncthreads();
  // every warp adds the warps' sums up for itself
  unsigned long long w = lane < kWarps ? sm.part[lane] : 0, s = w;
#pragma unroll
  for (int d = 1; d < kWarps; d <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  *total = __shfl_sync(0xffffffffu, s, kWarps - 1);
  return __shfl_sync(0xffffffffu, s - w, warp) + inc - v;
}

// Sets a bit of a shared bitmap; false if it was set already.
__device__ __forceinline__ bool mark(uint32_t* bits, int64_t i) {
  const uint32_t m = 1u << (i & 31);
  return (atomicOr(&bits[i >> 5], m) & m) == 0;
}

__device__ __forceinline__ void raise(PlanSmem& sm, int code) { atomicCAS(&sm.bad, 0, code); }

// Ends a plan: records an error and whether the call goes on.  All threads.
__device__ bool plan_goes_on(const knn_pages& p, PlanSmem& sm) {
  __syncthreads();
  const int bad = sm.bad;
  if (threadIdx.x == 0) {
    if (bad) atomicCAS(&p.status[kStatusError], 0, bad);
    p.status[kStatusApplied] = bad == 0;
  }
  return bad == 0;
}

// The counts of references of a tile of 16 pages a thread: four 16-byte loads
// that are each coalesced.
template <int kThreads>
struct RefsTile {
  int4 r[4];
  __device__ __forceinline__ void load(const knn_pages& p, int64_t base) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = base + j * 4 * kThreads + 4 * threadIdx.x;
      if (i + 4 <= p.pages && (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0) {
        r[j] = *reinterpret_cast<const int4*>(p.refs + i);
      } else {
        r[j].x = i < p.pages ? p.refs[i] : 1;
        r[j].y = i + 1 < p.pages ? p.refs[i + 1] : 1;
        r[j].z = i + 2 < p.pages ? p.refs[i + 2] : 1;
        r[j].w = i + 3 < p.pages ? p.refs[i + 3] : 1;
      }
    }
  }
};

// Gives out the `need` lowest-numbered free pages: give(rank, page) for ranks
// 0 .. need - 1 in order of the page numbers.  Returns how many there were.
// `tile` holds the first tile, asked for when the kernel began; the next is
// asked for while one is ranked.  The four runs of a tile are ranked by one
// prefix sum over four 16-bit fields (a run counts at most 4096).
template <int kThreads, class Give>
__device__ int take_free(const knn_pages& p, int need, PlanSmem& sm, RefsTile<kThreads>& tile,
                         Give give) {
  constexpr int kRun = 4 * kThreads;
  int given = 0;
  for (int64_t base = 0; base < p.pages && given < need; base += 4 * kRun) {
    const RefsTile<kThreads> now = tile;
    tile.load(p, base + 4 * kRun);
    unsigned long long count = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int4& r = now.r[j];
      const int c = (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
      count |= static_cast<unsigned long long>(c) << (16 * j);
    }
    unsigned long long total;
    const unsigned long long before = block_exclusive<kThreads>(count, sm, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int4& r = now.r[j];
      const int64_t i = base + j * kRun + 4 * threadIdx.x;
      int rank = given + static_cast<int>((before >> (16 * j)) & 0xffff);
      if (r.x == 0 && rank < need) give(rank, static_cast<int32_t>(i));
      rank += r.x == 0;
      if (r.y == 0 && rank < need) give(rank, static_cast<int32_t>(i + 1));
      rank += r.y == 0;
      if (r.z == 0 && rank < need) give(rank, static_cast<int32_t>(i + 2));
      rank += r.z == 0;
      if (r.w == 0 && rank < need) give(rank, static_cast<int32_t>(i + 3));
      given += static_cast<int>((total >> (16 * j)) & 0xffff);
    }
  }
  return given < need ? given : need;
}

// Index of the run that rank falls in: the last i with first[i] <= rank.
__device__ __forceinline__ int run_of(const int32_t* first, int n, int rank) {
  int low = 0, high = n - 1;
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (first[mid] <= rank) low = mid;
    else high = mid - 1;
  }
  return low;
}

__device__ __forceinline__ int64_t pages_for(int64_t rows, int page_rows) {
  return (rows + page_rows - 1) / page_rows;
}

// grow: counts[i] more rows for sequence seqs[i].
template <int kThreads>
__global__ void __launch_bounds__(kThreads) grow_kernel(knn_pages p, const int32_t* seqs,
                                                            const int32_t* counts, int n,
                                                            int64_t wanted) {
  extern __shared__ uint32_t dyn[];
  __shared__ PlanSmem sm;
  int32_t* first = reinterpret_cast<int32_t*>(dyn);  // [n + 1] pages before entry i
  uint32_t* seen = dyn + n + 1;                      // bitmap of the sequences
  const int64_t words = (p.sequences + 31) / 32;
  if (threadIdx.x == 0) sm.bad = 0;
  for (int64_t i = threadIdx.x; i < words; i += kThreads) seen[i] = 0;
  wait_for_stream();
  RefsTile<kThreads> tile;
  tile.load(p, 0);
  __syncthreads();
  constexpr int kPer = (kThreads == kFewThreads ? kFewList : kMaxList) / kThreads;
  unsigned long long fresh[kPer], mine = 0, rows_sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = threadIdx.x * kPer + j;
    fresh[j] = 0;
    if (i >= n) continue;
    const int64_t s = seqs[i], c = counts[i];
    if (s < 0 || s >= p.sequences) raise(sm, KNN_PAGES_OUT_OF_RANGE);
    else if (c < 0) raise(sm, KNN_PAGES_BAD_COUNT);
    else if (!mark(seen, s)) raise(sm, KNN_PAGES_LISTED_TWICE);
    else {
      const int64_t length = p.rows[s];
      const int64_t after = pages_for(length + c, p.page_rows);
      if (length < 0 || after > p.columns || length + c > 0x7fffffff) raise(sm, KNN_PAGES_TOO_LONG);
      else fresh[j] = after - pages_for(length, p.page_rows);
      rows_sum += c;
    }
    mine += fresh[j];
  }
  unsigned long long need = 0, rows_total = 0;
  unsigned long long before = block_exclusive<kThreads>(mine, sm, &need);
  block_exclusive<kThreads>(rows_sum, sm, &rows_total);
  if (wanted >= 0 && rows_total != static_cast<unsigned long long>(wanted))
    raise(sm, KNN_PAGES_BAD_COUNT);
  if (need > static_cast<unsigned long long>(p.pages)) raise(sm, KNN_PAGES_NONE_FREE);
  __syncthreads();
  if (sm.bad == 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = threadIdx.x * kPer + j;
      if (i < n) first[i] = static_cast<int32_t>(before);
      before += fresh[j];
    }
    __syncthreads();
    auto entry = [&](int rank) -> int32_t* {
      const int i = run_of(first, n, rank);
      const int64_t s = seqs[i];
      return p.table + s * p.columns + pages_for(p.rows[s], p.page_rows) + (rank - first[i]);
    };
    const int want = static_cast<int>(need);
    const int got = take_free<kThreads>(p, want, sm, tile, [&](int rank, int32_t page) {
      *entry(rank) = page;
      p.refs[page] = 1;
    });
    __syncthreads();
    if (got < want) {  // too few: give them back
      for (int rank = threadIdx.x; rank < got; rank += kThreads) {
        int32_t* e = entry(rank);
        p.refs[*e] = 0;
        *e = -1;
      }
      raise(sm, KNN_PAGES_NONE_FREE);
    }
  }
  if (!plan_goes_on(p, sm)) return;
  for (int i = threadIdx.x; i < n; i += kThreads) p.rows[seqs[i]] += counts[i];
}

// ------------------------------------------------------------------- free
// One CTA a listed sequence.  Every CTA looks the whole list over (a few KB
// out of L2), so that a bad index stops all of them; a sequence that is
// listed again is freed by its first mention alone.
__global__ void __launch_bounds__(kMoveThreads) free_kernel(knn_pages p, const int32_t* seqs,
                                                            int n) {
  wait_for_stream();
  const int i = blockIdx.x;
  const int32_t s = seqs[i];
  bool bad = false, again = false;
  for (int j = threadIdx.x; j < n; j += kMoveThreads) {
    const int32_t o = seqs[j];
    bad |= o < 0 || o >= p.sequences;
    again |= j < i && o == s;
  }
  bad = __syncthreads_or(bad);
  again = __syncthreads_or(again);
  if (i == 0 && threadIdx.x == 0) {
    if (bad) atomicCAS(&p.status[kStatusError], 0, KNN_PAGES_OUT_OF_RANGE);
    p.status[kStatusApplied] = !bad;
  }
  if (bad || again) return;
  int64_t used = pages_for(p.rows[s], p.page_rows);
  if (used > p.columns) used = p.columns;
  // four entries of a thread's under way at once: a long sequence is a latency
  int32_t* entries = p.table + s * p.columns;
  for (int64_t c = threadIdx.x; c < used; c += 4 * kMoveThreads) {
    int32_t page[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      page[j] = c + j * kMoveThreads < used ? entries[c + j * kMoveThreads] : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (page[j] >= 0 && page[j] < p.pages) atomicSub(&p.refs[page[j]], 1);
      if (c + j * kMoveThreads < used) entries[c + j * kMoveThreads] = -1;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) p.rows[s] = 0;
}

// copy, plan: every index in range, no target twice, no target a source.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) copy_plan_kernel(knn_pages p,
                                                             const int32_t* sources,
                                                             const int32_t* targets, int64_t n,
                                                             int64_t chunks, bool here) {
  extern __shared__ uint32_t dyn[];
  __shared__ PlanSmem sm;
  const int64_t words = (p.pages + 31) / 32;
  if (threadIdx.x == 0) sm.bad = 0;
  for (int64_t i = threadIdx.x; i < words; i += kThreads) dyn[i] = 0;
  wait_for_stream();
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const int32_t t = targets[i];
    if (t < 0 || t >= p.pages) raise(sm, KNN_PAGES_OUT_OF_RANGE);
    else if (!mark(dyn, t)) raise(sm, KNN_PAGES_LISTED_TWICE);
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const int32_t s = sources[i];
    if (s < 0 || s >= p.pages) raise(sm, KNN_PAGES_OUT_OF_RANGE);
    else if ((dyn[s >> 5] >> (s & 31)) & 1) raise(sm, KNN_PAGES_LISTED_TWICE);
  }
  if (!plan_goes_on(p, sm) || !here) return;
  if constexpr (kThreads == kMoveThreads)
    for (int64_t item = 0; item < n * chunks; ++item) copy_item(p, sources, targets, item, chunks);
}

__global__ void __launch_bounds__(kMoveThreads) copy_kernel(knn_pages p, const int32_t* sources,
                                                            const int32_t* targets, int64_t n,
                                                            int64_t chunks) {
  wait_for_stream();
  if (!p.status[kStatusApplied]) return;
  for (int64_t item = blockIdx.x; item < n * chunks; item += gridDim.x)
    copy_item(p, sources, targets, item, chunks);
}

// -------------------------------------------------------------------- fork
// fork, move: full pages are shared (table entry, one more reference), the
// rows of a part-filled last page are copied.
__device__ __forceinline__ void fork_item(const knn_pages& p, const int32_t* parents,
                                          const int32_t* children, int64_t item, int64_t shares,
                                          int64_t per) {
  const int64_t i = item / per;
  int64_t part = item - i * per;
  const int64_t s = parents[i], c = children[i];
  const int64_t length = p.rows[c];
  const int64_t full = length / p.page_rows;
  const int32_t* theirs = p.table + s * p.columns;
  int32_t* ours = p.table + c * p.columns;
  if (part < shares) {
    int64_t end = (part + 1) * kShareChunk;
    if (end > full) end = full;
    for (int64_t col = part * kShareChunk + threadIdx.x; col < end; col += kMoveThreads) {
      const int32_t page = theirs[col];
      ours[col] = page;
      if (page >= 0 && page < p.pages) atomicAdd(&p.refs[page], 1);
    }
    return;
  }
  part -= shares;
  const int64_t tail = length - full * p.page_rows;
  if (tail == 0) return;
  const int32_t from = theirs[full], to = ours[full];
  if (from < 0 || from >= p.pages) return;
  for (int k = 0; k < p.n_pools; ++k) {
    const int64_t page_bytes = p.row_bytes[k] * p.page_rows;
    const int64_t parts = (page_bytes + kMoveChunk - 1) / kMoveChunk;
    if (part < parts) {
      uint8_t* pool = static_cast<uint8_t*>(p.pools[k]);
      const int64_t off = part * kMoveChunk;
      const int64_t left = tail * p.row_bytes[k] - off;
      if (left > 0)
        block_copy(pool + to * page_bytes + off, pool + from * page_bytes + off,
                   left < kMoveChunk ? left : kMoveChunk);
      break;
    }
    part -= parts;
  }
}

// fork, plan: the children's lengths, and a fresh page for each child whose
// parent's last page is not full.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) fork_plan_kernel(knn_pages p,
                                                             const int32_t* parents,
                                                             const int32_t* children, int n,
                                                             int64_t shares, int64_t chunks,
                                                             bool here) {
  extern __shared__ uint32_t dyn[];
  __shared__ PlanSmem sm;
  int32_t* who = reinterpret_cast<int32_t*>(dyn);  // [n] the children that need a page
  int32_t* length = who + n;                       // [n] their parents' lengths
  uint32_t* seen = dyn + 2 * n;
  const int64_t words = (p.sequences + 31) / 32;
  if (threadIdx.x == 0) sm.bad = 0;
  for (int64_t i = threadIdx.x; i < words; i += kThreads) seen[i] = 0;
  wait_for_stream();
  RefsTile<kThreads> tile;
  tile.load(p, 0);
  __syncthreads();
  constexpr int kPer = (kThreads == kFewThreads ? kFewList : kMaxList) / kThreads;
  unsigned long long mine = 0;
  bool part[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = threadIdx.x * kPer + j;
    part[j] = false;
    if (i >= n) continue;
    const int64_t s = parents[i], c = children[i];
    if (s < 0 || s >= p.sequences || c < 0 || c >= p.sequences) raise(sm, KNN_PAGES_OUT_OF_RANGE);
    else if (!mark(seen, c)) raise(sm, KNN_PAGES_LISTED_TWICE);
    else if (p.rows[c] != 0) raise(sm, KNN_PAGES_NOT_EMPTY);
    else {
      const int32_t rows = p.rows[s];
      if (rows < 0 || pages_for(rows, p.page_rows) > p.columns) raise(sm, KNN_PAGES_TOO_LONG);
      length[i] = rows;
      part[j] = rows % p.page_rows != 0;
    }
    mine += part[j];
  }
  unsigned long long need = 0;
  int before = static_cast<int>(block_exclusive<kThreads>(mine, sm, &need));
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (part[j]) who[before++] = threadIdx.x * kPer + j;
  __syncthreads();
  if (sm.bad == 0 && need > 0) {
    auto entry = [&](int rank) {
      const int i = who[rank];
      return p.table + children[i] * p.columns + length[i] / p.page_rows;
    };
    const int want = static_cast<int>(need);
    const int got = take_free<kThreads>(p, want, sm, tile, [&](int rank, int32_t page) {
      *entry(rank) = page;
      p.refs[page] = 1;
    });
    __syncthreads();
    if (got < want) {
      for (int rank = threadIdx.x; rank < got; rank += kThreads) {
        int32_t* e = entry(rank);
        p.refs[*e] = 0;
        *e = -1;
      }
      raise(sm, KNN_PAGES_NONE_FREE);
    }
  }
  if (!plan_goes_on(p, sm)) return;
  for (int i = threadIdx.x; i < n; i += kThreads) p.rows[children[i]] = length[i];
  if (!here) return;
  __syncthreads();  // table entries and lengths
  if constexpr (kThreads == kMoveThreads)
    for (int64_t item = 0; item < n * (shares + chunks); ++item)
      fork_item(p, parents, children, item, shares, shares + chunks);
}

__global__ void __launch_bounds__(kMoveThreads) fork_kernel(knn_pages p, const int32_t* parents,
                                                            const int32_t* children, int64_t n,
                                                            int64_t shares, int64_t chunks) {
  wait_for_stream();
  if (!p.status[kStatusApplied]) return;
  const int64_t per = shares + chunks;
  for (int64_t item = blockIdx.x; item < n * per; item += gridDim.x)
    fork_item(p, parents, children, item, shares, per);
}

// ----------------------------------------------------------------- compact
// Workspace: kept[n][chunks] rows kept in each chunk of kKeepChunk positions
// (then, after the plan, those kept before it), total[n], fresh[n][columns],
// and where the plan itself makes the targets' entries (`here`: small calls,
// two launches in place of four) length[n] and old[n][columns], what the
// sources were.
struct CompactWork {
  int32_t* kept;
  int32_t* total;
  int32_t* fresh;
  int32_t* length;
  int32_t* old;
  int64_t chunks;
  int32_t here;
};

// The target's table row and length; a target that is its own source lets its
// old pages go.
__device__ __forceinline__ void commit_target(const knn_pages& p, const int32_t* sources,
                                              const int32_t* targets, const CompactWork& w,
                                              int64_t i) {
  const int64_t s = sources[i], t = targets[i];
  const int64_t used = s == t ? pages_for(p.rows[t], p.page_rows) : 0;
  const int64_t fresh = pages_for(w.total[i], p.page_rows);
  int32_t* ours = p.table + t * p.columns;
  for (int64_t c = threadIdx.x; c < (used > fresh ? used : fresh); c += kMoveThreads) {
    if (c < used) {
      const int32_t page = ours[c];
      if (page >= 0 && page < p.pages) atomicSub(&p.refs[page], 1);
    }
    ours[c] = c < fresh ? w.fresh[i * p.columns + c] : -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) p.rows[t] = w.total[i];
}

__global__ void __launch_bounds__(kKeepChunk) compact_count_kernel(
    knn_pages p, const int32_t* sources, const uint8_t* keep, int64_t keep_columns,
    int64_t keep_stride, CompactWork w) {
  wait_for_stream();
  const int64_t i = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks;
  const int64_t s = sources[i];
  const int64_t length = s >= 0 && s < p.sequences ? p.rows[s] : 0;
  const int64_t at = chunk * kKeepChunk + threadIdx.x;
  const bool kept = at < keep_columns && at < length && keep[i * keep_stride + at] != 0;
  const int count = __syncthreads_count(kept);
  if (threadIdx.x == 0) w.kept[i * w.chunks + chunk] = count;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) compact_plan_kernel(knn_pages p,
                                                                    const int32_t* sources,
                                                                const int32_t* targets, int n,
                                                                const uint8_t* keep,
                                                                int64_t keep_columns,
                                                                int64_t keep_stride,
                                                                CompactWork w) {
  extern __shared__ uint32_t dyn[];
  __shared__ PlanSmem sm;
  int32_t* first = reinterpret_cast<int32_t*>(dyn);  // [n]
  uint32_t* seen = dyn + n;
  const int64_t words = (p.sequences + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) sm.bad = 0;
  for (int64_t i = threadIdx.x; i < words; i += kThreads) seen[i] = 0;
  wait_for_stream();
  RefsTile<kThreads> tile;
  tile.load(p, 0);
  if (w.here) {  // rows kept in each chunk, a warp to a chunk
    for (int64_t item = warp; item < n * w.chunks; item += kThreads / 32) {
      const int64_t i = item / w.chunks, chunk = item - i * w.chunks;
      const int64_t s = sources[i];
      const int64_t length = s >= 0 && s < p.sequences ? p.rows[s] : 0;
      int count = 0;
#pragma unroll
      for (int j = 0; j < kKeepChunk; j += 32) {
        const int64_t at = chunk * kKeepChunk + j + lane;
        count += at < keep_columns && at < length && keep[i * keep_stride + at] != 0;
      }
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) w.kept[item] = count;
    }
    __syncthreads();
  }
  // rows kept before each chunk, a warp to a sequence
  for (int64_t i = warp; i < n; i += (kThreads / 32)) {
    int32_t* kept = w.kept + i * w.chunks;
    int sum = 0;
    for (int64_t base = 0; base < w.chunks; base += 128) {
      const int64_t c = base + 4 * lane;
      int v[4], mine = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c + j < w.chunks ? kept[c + j] : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += v[j];
      int inc = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
      }
      int before = sum + inc - mine;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + j < w.chunks) kept[c + j] = before;
        before += v[j];
      }
      sum += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) w.total[i] = sum;
  }
  __syncthreads();
  constexpr int kPer = (kThreads == kFewThreads ? kFewList : kMaxList) / kThreads;
  unsigned long long fresh[kPer], mine = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = threadIdx.x * kPer + j;
    fresh[j] = 0;
    if (i >= n) continue;
    const int64_t s = sources[i], t = targets[i];
    if (s < 0 || s >= p.sequences || t < 0 || t >= p.sequences) raise(sm, KNN_PAGES_OUT_OF_RANGE);
    else if (!mark(seen, t)) raise(sm, KNN_PAGES_LISTED_TWICE);
    else if (t != s && p.rows[t] != 0) raise(sm, KNN_PAGES_NOT_EMPTY);
    else if (p.rows[s] > keep_columns) raise(sm, KNN_PAGES_BAD_COUNT);
    else if (p.rows[s] < 0 || pages_for(p.rows[s], p.page_rows) > p.columns)
      raise(sm, KNN_PAGES_TOO_LONG);
    else fresh[j] = pages_for(w.total[i], p.page_rows);
    mine += fresh[j];
  }
  unsigned long long need = 0;
  unsigned long long before = block_exclusive<kThreads>(mine, sm, &need);
  if (need > static_cast<unsigned long long>(p.pages)) raise(sm, KNN_PAGES_NONE_FREE);
  __syncthreads();
  if (sm.bad == 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = threadIdx.x * kPer + j;
      if (i < n) first[i] = static_cast<int32_t>(before);
      before += fresh[j];
    }
    __syncthreads();
    auto entry = [&](int rank) {
      const int i = run_of(first, n, rank);
      return w.fresh + i * p.columns + (rank - first[i]);
    };
    const int want = static_cast<int>(need);
    const int got = take_free<kThreads>(p, want, sm, tile, [&](int rank, int32_t page) {
      *entry(rank) = page;
      p.refs[page] = 1;
    });
    __syncthreads();
    if (got < want) {
      for (int rank = threadIdx.x; rank < got; rank += kThreads) p.refs[*entry(rank)] = 0;
      raise(sm, KNN_PAGES_NONE_FREE);
    }
  }
  if (!plan_goes_on(p, sm) || !w.here) return;
  if constexpr (kThreads == kMoveThreads) {
    // what the sources are, before any of them may be a target
    for (int64_t i = 0; i < n; ++i) {
      const int64_t s = sources[i];
      const int32_t length = p.rows[s];
      if (threadIdx.x == 0) w.length[i] = length;
      for (int64_t c = threadIdx.x; c < pages_for(length, p.page_rows); c += kThreads)
        w.old[i * p.columns + c] = p.table[s * p.columns + c];
    }
    __syncthreads();
    for (int64_t i = 0; i < n; ++i) commit_target(p, sources, targets, w, i);
  }
}

// The kept rows of a chunk go to their places, piece by piece, four of a
// thread's under way at once.
template <class T>
__device__ __forceinline__ void gather_rows(T* pool, const int64_t* from, const int64_t* to,
                                            int kept, int64_t row_bytes) {
  const uint32_t pieces = static_cast<uint32_t>(row_bytes / sizeof(T));
  const uint32_t total = pieces * kept;
  // i / pieces by the reciprocal: it is at most `pieces` / 2^32 too large, and
  // i below kKeepChunk * pieces, so exact up to 4096 pieces
  const uint32_t over = 0xffffffffu / pieces + 1;
  const bool exact = pieces > 1 && pieces <= 4096;
  for (uint32_t i = threadIdx.x; i < total; i += 4 * kMoveThreads) {
    T v[4];
    int64_t at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t o = i + j * kMoveThreads;
      if (o >= total) continue;
      const uint32_t r = exact ? __umulhi(o, over) : o / pieces, c = o - r * pieces;
      at[j] = to[r] * pieces + c;
      v[j] = __ldcs(pool + from[r] * pieces + c);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * kMoveThreads < total) __stcs(pool + at[j], v[j]);
  }
}

__global__ void __launch_bounds__(kMoveThreads) compact_kernel(knn_pages p, const int32_t* sources,
                                                               const uint8_t* keep,
                                                               int64_t keep_stride,
                                                               CompactWork w) {
  __shared__ int64_t from[kKeepChunk], to[kKeepChunk];
  __shared__ int warp_kept[kKeepChunk / 32];
  wait_for_stream();
  if (!p.status[kStatusApplied]) return;
  const int64_t i = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks;
  const int64_t s = sources[i];
  const int64_t at = chunk * kKeepChunk + threadIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool kept = false;
  unsigned ballot = 0;
  if (threadIdx.x < kKeepChunk) {
    kept = at < (w.here ? w.length[i] : p.rows[s]) && keep[i * keep_stride + at] != 0;
    ballot = __ballot_sync(0xffffffffu, kept);
    if (lane == 0) warp_kept[warp] = __popc(ballot);
  }
  __syncthreads();
  int total = 0, before = 0;
#pragma unroll
  for (int j = 0; j < kKeepChunk / 32; ++j) {
    if (j < warp) before += warp_kept[j];
    total += warp_kept[j];
  }
  if (total == 0) return;
  if (kept) {
    const int slot = before + __popc(ballot & ((1u << lane) - 1));
    const Places old = {w.here ? w.old : p.table, p.columns, p.pages, p.page_rows};
    const Places now = {w.fresh, p.columns, p.pages, p.page_rows};
    const int64_t a = old.at(w.here ? i : s, at);
    from[slot] = a < 0 ? 0 : a;  // a table entry without a page: any row
    to[slot] = now.at(i, w.kept[i * w.chunks + chunk] + slot);
  }
  __syncthreads();
  for (int k = 0; k < p.n_pools; ++k) {
    const int64_t bytes = p.row_bytes[k];
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.pools[k]) | static_cast<uintptr_t>(bytes);
    if ((bits & 15) == 0) gather_rows(static_cast<uint4*>(p.pools[k]), from, to, total, bytes);
    else if ((bits & 3) == 0) gather_rows(static_cast<uint32_t*>(p.pools[k]), from, to, total, bytes);
    else gather_rows(static_cast<uint8_t*>(p.pools[k]), from, to, total, bytes);
  }
}

__global__ void __launch_bounds__(kMoveThreads) compact_commit_kernel(knn_pages p,
                                                                      const int32_t* sources,
                                                                      const int32_t* targets,
                                                                      CompactWork w) {
  wait_for_stream();
  if (!p.status[kStatusApplied]) return;
  commit_target(p, sources, targets, w, blockIdx.x);
}

// Work that a plan does itself rather than leave it to a second launch, which
// costs a small call more than one CTA takes for this: pieces of at most 16 KB
// or 1024 table entries, chunks of flags, table entries of a compaction.  Calls
// one after another, in one launch less (two for a compaction): 3 small pages
// copied in 5.5 us, not 7.5, 1000 rows forked in 9.2, not 11.5 (their freeing
// included), and compacted in 16, not 21; a call waited for is about as fast.
constexpr int64_t kHereItems = 8, kHereChunks = 64, kHerePages = 2048;

bool is_small(const knn_pages& p, int64_t n) { return n <= kFewList && p.pages <= kFewPages; }

constexpr int kPlanSmem = 200 * 1024;  // at most: a bitmap of 2^20 bits and lists of 2 x 4096

// Launches a plan kernel in its form for few or for many entries and pages.
template <class... P, class... A>
cudaError_t launch_plan(void (*few)(P...), void (*many)(P...), int64_t n, const knn_pages& p,
                        size_t smem, cudaStream_t stream, A&&... args) {
  const bool small = is_small(p, n);
  if (smem > 40 * 1024) {
    if (cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(small ? few : many),
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanSmem))
      return e;
  }
  return launch_after(small ? few : many, 1, small ? kFewThreads : kManyThreads, smem, stream,
                      args...);
}

int64_t move_chunks(const knn_pages& p) {
  int64_t chunks = 0;
  for (int k = 0; k < p.n_pools; ++k)
    chunks += (p.row_bytes[k] * p.page_rows + kMoveChunk - 1) / kMoveChunk;
  return chunks;
}

unsigned move_grid(int64_t items) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(items, 148 * 8)));
}

}  // namespace

cudaError_t launch_pages_grow(const knn_pages& p, const int32_t* seqs, const int32_t* counts,
                              int64_t n, int64_t total, cudaStream_t stream) {
  const size_t smem = 4 * (n + 1 + (p.sequences + 31) / 32);
  store_count_launches(1);
  return launch_plan(grow_kernel<kFewThreads>, grow_kernel<kManyThreads>, n, p, smem, stream, p,
                     seqs, counts, static_cast<int>(n), total);
}

cudaError_t launch_pages_free(const knn_pages& p, const int32_t* seqs, int64_t n,
                              cudaStream_t stream) {
  store_count_launches(1);
  return launch_after(free_kernel, static_cast<unsigned>(n), kMoveThreads, 0, stream, p, seqs,
                      static_cast<int>(n));
}

cudaError_t launch_pages_copy(const knn_pages& p, const int32_t* sources, const int32_t* targets,
                              int64_t n, cudaStream_t stream) {
  const size_t smem = 4 * ((p.pages + 31) / 32);
  const int64_t chunks = move_chunks(p);
  const bool here = is_small(p, n) && n * chunks <= kHereItems;
  store_count_launches(here ? 1 : 2);
  cudaError_t e = launch_plan(copy_plan_kernel<kFewThreads>, copy_plan_kernel<kManyThreads>, n, p,
                              smem, stream, p, sources, targets, n, chunks, here);
  if (e != cudaSuccess || here) return e;
  return launch_after(copy_kernel, move_grid(n * chunks), kMoveThreads, 0, stream, p, sources,
                      targets, n, chunks);
}

cudaError_t launch_pages_fork(const knn_pages& p, const int32_t* parents, const int32_t* children,
                              int64_t n, cudaStream_t stream) {
  const size_t smem = 4 * (2 * n + (p.sequences + 31) / 32);
  const int64_t shares = (p.columns + kShareChunk - 1) / kShareChunk, chunks = move_chunks(p);
  const bool here = is_small(p, n) && n * (shares + chunks) <= kHereItems;
  store_count_launches(here ? 1 : 2);
  cudaError_t e = launch_plan(fork_plan_kernel<kFewThreads>, fork_plan_kernel<kManyThreads>, n, p,
                              smem, stream, p, parents, children, static_cast<int>(n), shares,
                              chunks, here);
  if (e != cudaSuccess || here) return e;
  return launch_after(fork_kernel, move_grid(n * (shares + chunks)), kMoveThreads, 0, stream, p,
                      parents, children, n, shares, chunks);
}

int64_t pages_compact_words(const knn_pages& p, int64_t n, int64_t keep_columns) {
  const int64_t chunks = std::max<int64_t>(1, (keep_columns + kKeepChunk - 1) / kKeepChunk);
  return n * (chunks + 2 + 2 * p.columns);
}

cudaError_t launch_pages_compact(const knn_pages& p, const int32_t* sources,
                                 const int32_t* targets, int64_t n, const uint8_t* keep,
                                 int64_t keep_columns, int64_t keep_stride, int32_t* workspace,
                                 cudaStream_t stream) {
  CompactWork w;
  w.chunks = std::max<int64_t>(1, (keep_columns + kKeepChunk - 1) / kKeepChunk);
  w.kept = workspace;
  w.total = w.kept + n * w.chunks;
  w.fresh = w.total + n;
  w.length = w.fresh + n * p.columns;
  w.old = w.length + n;
  w.here = is_small(p, n) && n * w.chunks <= kHereChunks &&
           n * ((keep_columns + p.page_rows - 1) / p.page_rows) <= kHerePages;
  const size_t smem = 4 * (n + (p.sequences + 31) / 32);
  store_count_launches(w.here ? 2 : 4);
  const unsigned grid = static_cast<unsigned>(n * w.chunks);
  if (!w.here)
    if (cudaError_t e = launch_after(compact_count_kernel, grid, kKeepChunk, 0, stream, p, sources,
                                     keep, keep_columns, keep_stride, w))
      return e;
  if (cudaError_t e = launch_plan(compact_plan_kernel<kFewThreads>,
                                  compact_plan_kernel<kManyThreads>, n, p, smem, stream, p, sources,
                                  targets, static_cast<int>(n), keep, keep_columns, keep_stride, w))
    return e;
  cudaError_t e = launch_after(compact_kernel, grid, kMoveThreads, 0, stream, p, sources, keep,
                               keep_stride, w);
  if (e != cudaSuccess || w.here) return e;
  return launch_after(compact_commit_kernel, static_cast<unsigned>(n), kMoveThreads, 0, stream, p,
                      sources, targets, w);
}

}  // namespace knn
