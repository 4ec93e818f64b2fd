// knn_q4.cu -- rows in 4 bits with a scale (and a zero point) for every group
// of 32, 64 or 128 values: packing, reading, products and search.
//
//   value[i][j] = (code[i][j] - zero[i][g]) * scale[i][g],  g = j / group
//   y[b][i]     = sum_g scale[i][g] * sum_{j in g} (code[i][j] - zero[i][g]) * x[b][j]
//
// A value has at most 5 + 11 significant bits, so it is exact in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "knn_q4.h"

namespace knn {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kNoKey = 0xFFFFFFFFu;

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ float scale_of(const Q4View& v, int64_t row, int g) {
  const uint16_t bits = v.scales[row * v.groups + g];
  return v.scale_bf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16)
                      : __half2float(__ushort_as_half(bits));
}
__device__ __forceinline__ int zero_of(const Q4View& v, int64_t row, int g) {
  return v.zeros ? v.zeros[row * v.groups + g] : 8;
}

// The larger of two numbers, NaN where either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// --------------------------------------------------- rows of listed sequences
constexpr int kMaxList = KNN_PAGES_MAX_LIST;

struct ListSmem {
  int32_t before[kMaxList + 1];  // rows of the entries before entry i
  int32_t part[kWarps];
};

// Prefix sums of the counts.  False (for all threads) where the list breaks a
// rule: an index out of range, a count below 0 or above the sequence's
// length, counts whose sum is not the total.
__device__ bool open_list(const Q4List& l, ListSmem& sm) {
  if (!l.seqs) return true;
  constexpr int kPer = kMaxList / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool bad = false;
  long long mine = 0;
  for (int j = 0; j < kPer; ++j) {
    const int i = threadIdx.x * kPer + j;
    if (i >= l.n) break;
    const int32_t s = l.seqs[i], c = l.counts[i];
    bad |= s < 0 || s >= l.sequences || c < 0 || c > l.total || (s >= 0 && s < l.sequences && c > l.rows[s]);
    if (!bad) mine += c;
  }
  bad |= mine > l.total;
  bad = __syncthreads_or(bad);
  if (bad) return false;
  // sums fit 32 bits unless the list is bad: total < 2^31, every part <= total
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  const bool over = inc > l.total;
  if (lane == 31) sm.part[warp] = over ? 0 : static_cast<int32_t>(inc);
  if (__syncthreads_or(over)) return false;
  long long base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += sm.part[w];
    sum += sm.part[w];
  }
  if (sum != l.total) return false;
  long long at = base + inc - mine;
  for (int j = 0; j < kPer; ++j) {
    const int i = threadIdx.x * kPer + j;
    if (i >= l.n) break;
    sm.before[i] = static_cast<int32_t>(at);
    at += l.counts[i];
  }
  if (threadIdx.x == 0) sm.before[l.n] = static_cast<int32_t>(l.total);
  __syncthreads();
  return true;
}

// Row t of the list, as a row number in the pools (-1: no page).
__device__ __forceinline__ int64_t list_row(const Q4View& v, const Q4List& l, const ListSmem& sm,
                                            int64_t t) {
  if (!l.seqs) return l.first + t;
  int low = 0, high = l.n - 1;  // the last entry with before <= t
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (sm.before[mid] <= t) low = mid;
    else high = mid - 1;
  }
  const int64_t s = l.seqs[low];
  return v.places.at(s, static_cast<int64_t>(l.rows[s]) - l.counts[low] + (t - sm.before[low]));
}

// ------------------------------------------------------------------- pack
// q / t to the nearest whole number, ties to even, exactly: the quotient in
// fp32 can fall on a tie that the true one only comes near to, so the
// remainder (exact in one fma: q and t have at most 24 and 11 bits and the
// quotient 5) decides.
__device__ __forceinline__ float nearest(float q, float t) {
  float n = rintf(q / t);
  if (fabsf(n) > 64.0f) return n;  // clamped by the caller
  const float left = fmaf(-n, t, q), half = 0.5f * t;
  const bool odd = (static_cast<int>(n) & 1) != 0;
  if (left > half || (left == half && odd)) n += 1.0f;
  else if (left < -half || (left == -half && odd)) n -= 1.0f;
  return n;
}

// One warp a row; a lane holds 4 neighbouring values of each 128.  HBM bound:
// the values are read once, codes and scales written once.
template <class T>
__global__ void __launch_bounds__(kThreads) pack_kernel(Q4View v, Q4List l, const T* x, int64_t ld,
                                                        bool vec) {
  __shared__ ListSmem sm;
  wait_for_stream();
  if (l.seqs && !l.status[kStatusApplied]) return;
  if (!open_list(l, sm)) return;  // as the call that made room found it
  const int lane = threadIdx.x & 31;
  const int span = v.group / 4;  // lanes of a group
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < l.total;
       t += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = list_row(v, l, sm, t);
    if (row < 0) continue;
    const T* in = x + t * ld;
    float norm = 0.0f;
    for (int64_t base = 0; base < 2 * v.width; base += 128) {
      const int64_t j = base + 4 * lane;
      float a[4];
      if (vec && j + 4 <= v.dim) {
        if constexpr (sizeof(T) == 4) {
          const float4 f = *reinterpret_cast<const float4*>(in + j);
          a[0] = f.x, a[1] = f.y, a[2] = f.z, a[3] = f.w;
        } else {
          T h[4];
          *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(in + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = load_value(h + e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = j + e < v.dim ? load_value(in + j + e) : 0.0f;
      }
      float low, high;
      if (v.zeros) {
        high = max_nan(max_nan(max_nan(a[0], a[1]), max_nan(a[2], a[3])), 0.0f);
        low = -max_nan(max_nan(max_nan(-a[0], -a[1]), max_nan(-a[2], -a[3])), 0.0f);
      } else {
        high = max_nan(max_nan(fabsf(a[0]), fabsf(a[1])), max_nan(fabsf(a[2]), fabsf(a[3])));
        low = 0.0f;
      }
      for (int d = 1; d < span; d <<= 1) {
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, d));
        if (v.zeros) low = -max_nan(-low, -__shfl_xor_sync(0xffffffffu, low, d));
      }
      const float wide = v.zeros ? __fdiv_rn(high - low, 15.0f) : __fdiv_rn(high, 7.0f);
      uint16_t bits;
      float s;
      if (v.scale_bf16) {
        const __nv_bfloat16 h = __float2bfloat16_rn(wide);
        bits = __bfloat16_as_ushort(h);
        s = __bfloat162float(h);
      } else {
        const __half h = __float2half_rn(wide);
        bits = __half_as_ushort(h);
        s = __half2float(h);
      }
      const bool usable = s > 0.0f && s < __int_as_float(0x7f800000);
      float zero = 8.0f;
      if (v.zeros) zero = usable ? fminf(fmaxf(nearest(-low, s), 0.0f), 15.0f) : 0.0f;
      uint32_t packed = 0;
      int square = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float c = zero;
        if (usable) c = fminf(fmaxf(nearest(a[e], s) + zero, 0.0f), 15.0f);
        const int code = j + e < v.dim ? static_cast<int>(c) : 0;
        const int d = j + e < v.dim ? code - static_cast<int>(zero) : 0;
        square += d * d;
        packed |= static_cast<uint32_t>(code) << (4 * e);
      }
      norm += (s * s) * static_cast<float>(square);
      if (j < 2 * v.width)
        *reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(v.codes) + row * v.width + j / 2) =
            static_cast<uint16_t>(packed);
      if (lane % span == 0 && j < v.dim) {
        const int64_t g = row * v.groups + j / v.group;
        const_cast<uint16_t*>(v.scales)[g] = bits;
        if (v.zeros) const_cast<uint8_t*>(v.zeros)[g] = static_cast<uint8_t>(zero);
      }
    }
    if (v.norms) {
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, d);
      if (lane == 0) const_cast<float*>(v.norms)[row] = norm;
    }
  }
}

// ------------------------------------------------------------------- read
__global__ void __launch_bounds__(kThreads) read_kernel(Q4View v, Q4List l, float* out, int64_t ld,
                                                        bool vec) {
  __shared__ ListSmem sm;
  wait_for_stream();
  if (!open_list(l, sm)) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && l.status)
      atomicCAS(&l.status[kStatusError], 0, KNN_PAGES_BAD_COUNT);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < l.total;
       t += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = list_row(v, l, sm, t);
    for (int64_t j = 4 * lane; j < v.dim; j += 128) {
      float a[4];
      if (row < 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = __int_as_float(0x7fc00000);
      } else {
        const uint32_t packed = *reinterpret_cast<const uint16_t*>(v.codes + row * v.width + j / 2);
        const int g = static_cast<int>(j / v.group);
        const float s = scale_of(v, row, g);
        const int z = zero_of(v, row, g);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          a[e] = static_cast<float>(static_cast<int>((packed >> (4 * e)) & 15) - z) * s;
      }
      float* o = out + t * ld + j;
      if (vec && j + 4 <= v.dim) {
        *reinterpret_cast<float4*>(o) = make_float4(a[0], a[1], a[2], a[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < v.dim) o[e] = a[e];
      }
    }
  }
}

// --------------------------------------------------------------- products
// What becomes of a product: stored (in the output's type), or the key that a
// search orders rows by, |row|^2 - 2 q.row or -q.row (fp32; a row's place in
// the order does not depend on |q|^2).
enum { kStore = 0, kKeyL2 = 1, kKeyProduct = 2 };

struct Q4Out {
  void* y;
  int dtype;
  int64_t ld;
  int mode;
};

__device__ __forceinline__ void put(const Q4Out& o, int64_t b, int64_t i, float y, float norm) {
  if (o.mode == kKeyL2) y = norm - 2.0f * y;
  if (o.mode == kKeyProduct) y = -y;
  const int64_t at = b * o.ld + i;
  if (o.dtype == KNN_DTYPE_F32) static_cast<float*>(o.y)[at] = y;
  else if (o.dtype == KNN_DTYPE_F16) static_cast<__half*>(o.y)[at] = __float2half_rn(y);
  else static_cast<__nv_bfloat16*>(o.y)[at] = __float2bfloat16_rn(y);
}

// One warp a row, a lane 32 codes at a time.
template <class T>
__global__ void __launch_bounds__(kThreads) products_kernel(Q4View v, Q4Range r, const T* x,
                                                            int64_t batch, int64_t ldx, Q4Out o) {
  wait_for_stream();
  int64_t n = r.count;
  if (r.length) n = *r.length < n ? *r.length : n;
  const int lane = threadIdx.x & 31;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); i < r.count;
       i += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = i < n ? v.places.at(r.seq, i) : -1;
    for (int64_t b = 0; b < batch; ++b) {
      float sum = 0.0f;
      for (int c = lane; row >= 0 && c < v.width / 16; c += 32) {
        const uint4 w = *reinterpret_cast<const uint4*>(v.codes + row * v.width + 16 * c);
        const int g = 32 * c / v.group;
        const float z = static_cast<float>(zero_of(v, row, g));
        float part = 0.0f;
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int64_t j = 32 * c + e;
          if (j < v.dim)
            part += (static_cast<float>((words[e / 8] >> (4 * (e % 8))) & 15) - z) *
                    load_value(x + b * ldx + j);
        }
        sum += scale_of(v, row, g) * part;
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (row < 0) sum = i < n ? __int_as_float(0x7fc00000) : 0.0f;
      if (lane == 0) put(o, b, i, sum, o.mode == kKeyL2 && row >= 0 ? v.norms[row] : 0.0f);
    }
  }
}

// ----------------------------------------------------------------- search
constexpr int kGroupRows = 128;    // rows whose smallest key is kept
constexpr int kSelectThreads = 1024;
constexpr int kMoreCandidates = 16;  // scored again beyond the k asked for
constexpr int kMaxCandidates = KNN_MAX_K + kMoreCandidates;
constexpr int kGroupCap = 1024;
constexpr int kCandCap = 4096;

// Keys in an order that unsigned numbers have; a key that is +inf or NaN
// belongs to no neighbour.
__device__ __forceinline__ uint32_t ordered(float key) {
  if (!(key < __int_as_float(0x7f800000))) return kNoKey;
  const uint32_t b = __float_as_uint(key);
  return (b >> 31) ? ~b : b | 0x80000000u;
}

// The smallest key of every kGroupRows rows.
__global__ void __launch_bounds__(kThreads) group_min_kernel(Q4Range r, const float* keys,
                                                             int64_t ld, uint32_t* minima,
                                                             int64_t groups) {
  wait_for_stream();
  int64_t n = r.count;
  if (r.length) n = *r.length < n ? *r.length : n;
  const int lane = threadIdx.x & 31;
  const int64_t b = blockIdx.y;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (g >= groups) return;
  uint32_t m = kNoKey;
#pragma unroll
  for (int j = 0; j < kGroupRows / 32; ++j) {
    const int64_t i = g * kGroupRows + j * 32 + lane;
    if (i < n) m = min(m, ordered(keys[b * ld + i]));
  }
  m = __reduce_min_sync(0xffffffffu, m);
  if (lane == 0) minima[b * groups + g] = m;
}

struct SelectSmem {
  uint64_t cand[kCandCap];
  uint64_t final_key[kMaxCandidates];
  uint32_t final_row[kMaxCandidates];
  uint32_t hist[256];
  int32_t group[kGroupCap];
  uint32_t count, groups;
  uint64_t prefix;
  int64_t rank;
};

// The value of rank `rank` (from 0) among load(0 .. n - 1), by 8 bits a pass
// from the top; kBits 32 or 64.
template <int kBits, class Load>
__device__ uint64_t nth(int64_t n, int64_t rank, SelectSmem& sm, Load load) {
  uint64_t prefix = 0;
  for (int shift = kBits - 8; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) sm.hist[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t above = shift == kBits - 8 ? 0 : ~0ull << (shift + 8);
    for (int64_t base = 0; base < n; base += kSelectThreads) {
      const int64_t i = base + threadIdx.x;
      const uint64_t x = i < n ? load(i) : 0;
      const bool in = i < n && (x & above) == (prefix & above);
      const uint32_t bin = in ? static_cast<uint32_t>(x >> shift) & 255u : 256u;
      // keys share their leading bits: add up equal bins within the warp
      const uint32_t same = __match_any_sync(0xffffffffu, bin);
      if (in && (threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&sm.hist[bin], __popc(same));
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      uint32_t h[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += h[j] = sm.hist[8 * lane + j];
      uint32_t inc = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += up;
      }
      int64_t left = rank - static_cast<int64_t>(inc - sum);
      if (left >= 0 && left < static_cast<int64_t>(sum)) {
        int j = 0;
        while (left >= static_cast<int64_t>(h[j])) left -= h[j++];
        sm.prefix = prefix | (static_cast<uint64_t>(8 * lane + j) << shift);
        sm.rank = left;
      }
    }
    __syncthreads();
    prefix = sm.prefix;
    rank = sm.rank;
  }
  __syncthreads();
  return prefix;
}

// Sorts sm.cand[0 .. n) ascending, n a power of two.
__device__ void sort_candidates(SelectSmem& sm, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int p = threadIdx.x; p < n / 2; p += kSelectThreads) {
        const int lo = 2 * p - (p & (stride - 1)), hi = lo + stride;
        const uint64_t a = sm.cand[lo], b = sm.cand[hi];
        if ((a > b) == ((lo & size) == 0)) {
          sm.cand[lo] = b;
          sm.cand[hi] = a;
        }
      }
    }
  __syncthreads();
}

// One CTA a query: the k + 16 rows of smallest (key, index), their distances
// again in 64 bits, and the k first of those.
//
// The keys' sums are fp32 and rounded; near neighbours lie close together, so
// that order alone would depend on the order of the sums.  The distances of
// the candidates are summed again in 64 bits, which settles it.
//
// Candidates: with c wanted and tau the c-th smallest of the groups' minima,
// c rows lie at or below tau, so only keys <= tau are looked at, and they are
// in the groups whose minimum is <= tau: c groups, unless keys are equal.
template <class T>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(
    Q4View v, Q4Range r, const T* x, int64_t ldx, const float* keys, int64_t ld,
    const uint32_t* minima, int64_t groups, int k, int mode, int64_t* neighbors,
    float* distances) {
  extern __shared__ __align__(16) uint8_t raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(raw);
  wait_for_stream();
  const int64_t b = blockIdx.x;
  int64_t n = r.count;
  if (r.length) n = *r.length < n ? *r.length : n;
  keys += b * ld;
  minima += b * groups;
  const int wanted = k + kMoreCandidates;
  uint32_t tau = kNoKey - 1;
  if (groups > wanted) {
    tau = static_cast<uint32_t>(nth<32>(groups, wanted - 1, sm, [&](int64_t i) { return minima[i]; }));
    tau = min(tau, kNoKey - 1);
  }
  if (threadIdx.x == 0) sm.count = sm.groups = 0;
  __syncthreads();
  for (int64_t g = threadIdx.x; g < groups; g += kSelectThreads)
    if (minima[g] <= tau) {
      const uint32_t at = atomicAdd(&sm.groups, 1u);
      if (at < kGroupCap) sm.group[at] = static_cast<int32_t>(g);
    }
  __syncthreads();
  const uint32_t listed = sm.groups;
  if (listed <= kGroupCap) {
    for (uint32_t e = threadIdx.x; e < listed * kGroupRows; e += kSelectThreads) {
      const int64_t i = static_cast<int64_t>(sm.group[e / kGroupRows]) * kGroupRows + e % kGroupRows;
      const uint32_t key = i < n ? ordered(keys[i]) : kNoKey;
      if (key <= tau) {
        const uint32_t at = atomicAdd(&sm.count, 1u);
        if (at < kCandCap) sm.cand[at] = (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(i);
      }
    }
    __syncthreads();
  }
  int have;
  if (listed <= kGroupCap && sm.count <= kCandCap) {
    const int count = static_cast<int>(sm.count);
    int size = 2;
    while (size < count) size <<= 1;
    for (int e = count + threadIdx.x; e < size; e += kSelectThreads) sm.cand[e] = ~0ull;
    sort_candidates(sm, size);
    have = min(count, wanted);
  } else {
    // many equal keys: the row of rank wanted - 1 by (key, index), over all rows
    auto load = [&](int64_t i) {
      const uint32_t key = ordered(keys[i]);
      return (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(i);
    };
    const uint64_t last = n > wanted ? nth<64>(n, wanted - 1, sm, load) : ~0ull;
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < n; i += kSelectThreads) {
      const uint64_t c = load(i);
      if (c <= last && (c >> 32) != kNoKey) {
        const uint32_t at = atomicAdd(&sm.count, 1u);
        if (at < kCandCap) sm.cand[at] = c;  // at most `wanted`
      }
    }
    __syncthreads();
    have = min(static_cast<int>(sm.count), wanted);
  }
  // distances in 64 bits, a warp to a candidate
  const int lane = threadIdx.x & 31;
  const T* q = x + b * ldx;
  for (int e = threadIdx.x >> 5; e < have; e += kSelectThreads / 32) {
    const uint32_t i = static_cast<uint32_t>(sm.cand[e]);
    const int64_t row = v.places.at(r.seq, i);
    double sum = 0.0;
    for (int64_t j = lane; j < v.dim; j += 32) {
      const int g = static_cast<int>(j / v.group);
      const int code = (v.codes[row * v.width + j / 2] >> (4 * (j & 1))) & 15;
      const double value = static_cast<float>(code - zero_of(v, row, g)) * scale_of(v, row, g);
      const double qv = load_value(q + j);
      if (mode == kKeyL2) sum += (qv - value) * (qv - value);
      else sum -= qv * value;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) {
      if (sum != sum) sum = __longlong_as_double(0x7ff0000000000000ll);
      const uint64_t u = static_cast<uint64_t>(__double_as_longlong(sum + 0.0));
      sm.final_key[e] = (u >> 63) ? ~u : u | 0x8000000000000000ull;
      sm.final_row[e] = i;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < have; e += kSelectThreads) {
    const uint64_t key = sm.final_key[e];
    const uint32_t row = sm.final_row[e];
    int rank = 0;
    for (int o = 0; o < have; ++o)
      rank += sm.final_key[o] < key || (sm.final_key[o] == key && sm.final_row[o] < row);
    if (rank < k) {
      const uint64_t u = (key >> 63) ? key & 0x7fffffffffffffffull : ~key;
      const double d = __longlong_as_double(static_cast<long long>(u));
      neighbors[b * k + rank] = row;
      distances[b * k + rank] = static_cast<float>(mode == kKeyL2 ? d : -d);
    }
  }
  for (int e = have + threadIdx.x; e < k; e += kSelectThreads) {
    neighbors[b * k + e] = -1;
    distances[b * k + e] = __int_as_float(mode == kKeyL2 ? 0x7f800000 : 0xff800000);
  }
}

unsigned row_grid(int64_t rows) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>((rows + kWarps - 1) / kWarps, 148 * 8)));
}

template <class T>
cudaError_t products(const Q4View& v, const Q4Range& r, const void* x, int64_t batch, int64_t ldx,
                     const Q4Out& o, cudaStream_t stream) {
  store_count_launches(1);
  return launch_after(products_kernel<T>, row_grid(r.count), kThreads, 0, stream, v, r,
                      static_cast<const T*>(x), batch, ldx, o);
}

cudaError_t products_any(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                         int64_t batch, int64_t ldx, const Q4Out& o, cudaStream_t stream) {
  if (dtype == KNN_DTYPE_F32) return products<float>(v, r, x, batch, ldx, o, stream);
  if (dtype == KNN_DTYPE_F16) return products<__half>(v, r, x, batch, ldx, o, stream);
  return products<__nv_bfloat16>(v, r, x, batch, ldx, o, stream);
}

int64_t group_count(int64_t count) { return (count + kGroupRows - 1) / kGroupRows; }

template <class T>
cudaError_t select(const Q4View& v, const Q4Range& r, const void* x, int64_t batch, int64_t ldx,
                   const float* keys, int64_t ld, const uint32_t* minima, int k, int mode,
                   int64_t* neighbors, float* distances, cudaStream_t stream) {
  // above 48 KB only by leave, once per device and kernel
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(select_kernel<T>),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       sizeof(SelectSmem));
  if (e != cudaSuccess) return e;
  store_count_launches(1);
  return launch_after(select_kernel<T>, static_cast<unsigned>(batch), kSelectThreads,
                      sizeof(SelectSmem), stream, v, r, static_cast<const T*>(x), ldx, keys, ld,
                      minima, group_count(r.count), k, mode, neighbors, distances);
}

}  // namespace

cudaError_t launch_q4_pack(const Q4View& v, const Q4List& l, const void* rows, int dtype,
                           int64_t ld, cudaStream_t stream) {
  store_count_launches(1);
  const unsigned grid = row_grid(l.total);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(rows);
  if (dtype == KNN_DTYPE_F32)
    return launch_after(pack_kernel<float>, grid, kThreads, 0, stream, v, l,
                        static_cast<const float*>(rows), ld, ((bits | (ld * 4)) & 15) == 0);
  const bool vec = ((bits | (ld * 2)) & 7) == 0;
  if (dtype == KNN_DTYPE_F16)
    return launch_after(pack_kernel<__half>, grid, kThreads, 0, stream, v, l,
                        static_cast<const __half*>(rows), ld, vec);
  return launch_after(pack_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, v, l,
                      static_cast<const __nv_bfloat16*>(rows), ld, vec);
}

cudaError_t launch_q4_read(const Q4View& v, const Q4List& l, float* out, int64_t ld,
                           cudaStream_t stream) {
  store_count_launches(1);
  const bool vec = ((reinterpret_cast<uintptr_t>(out) | (ld * 4)) & 15) == 0;
  return launch_after(read_kernel, row_grid(l.total), kThreads, 0, stream, v, l, out, ld, vec);
}

cudaError_t launch_q4_products(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                               int64_t batch, int64_t ldx, void* out, int out_dtype, int64_t ldo,
                               cudaStream_t stream) {
  return products_any(v, r, x, dtype, batch, ldx, Q4Out{out, out_dtype, ldo, kStore}, stream);
}

int64_t q4_search_bytes(int64_t count) {
  return kQ4SearchBatch * 4 * (group_count(count) * (kGroupRows + 1));
}

cudaError_t launch_q4_search(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                             int64_t batch, int64_t ldx, int k, int metric, int64_t* neighbors,
                             float* distances, void* workspace, cudaStream_t stream) {
  const int mode = metric == KNN_METRIC_L2_EXPANDED ? kKeyL2 : kKeyProduct;
  const int64_t groups = group_count(r.count), ld = groups * kGroupRows;
  float* keys = static_cast<float*>(workspace);
  uint32_t* minima = static_cast<uint32_t*>(workspace) + kQ4SearchBatch * ld;
  const int64_t size = dtype == KNN_DTYPE_F32 ? 4 : 2;
  for (int64_t b = 0; b < batch; b += kQ4SearchBatch) {
    const int64_t m = std::min<int64_t>(kQ4SearchBatch, batch - b);
    const void* q = static_cast<const char*>(x) + b * ldx * size;
    if (r.count > 0) {
      if (cudaError_t e = products_any(v, r, q, dtype, m, ldx,
                                       Q4Out{keys, KNN_DTYPE_F32, ld, mode}, stream))
        return e;
      store_count_launches(1);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>((groups + kWarps - 1) / kWarps),
                         static_cast<unsigned>(m));
      cfg.blockDim = dim3(kThreads);
      cfg.stream = stream;
      if (cudaError_t e = cudaLaunchKernelEx(&cfg, group_min_kernel, r,
                                             static_cast<const float*>(keys), ld, minima, groups))
        return e;
    }
    cudaError_t e;
    if (dtype == KNN_DTYPE_F32)
      e = select<float>(v, r, q, m, ldx, keys, ld, minima, k, mode, neighbors + b * k,
                        distances + b * k, stream);
    else if (dtype == KNN_DTYPE_F16)
      e = select<__half>(v, r, q, m, ldx, keys, ld, minima, k, mode, neighbors + b * k,
                         distances + b * k, stream);
    else
      e = select<__nv_bfloat16>(v, r, q, m, ldx, keys, ld, minima, k, mode, neighbors + b * k,
                                distances + b * k, stream);
    if (e) return e;
  }
  return cudaSuccess;
}

}  // namespace knn
