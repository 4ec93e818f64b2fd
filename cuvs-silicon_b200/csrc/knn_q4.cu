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
#include <type_traits>

#include "knn_q4.h"

namespace knn {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kNoKey = 0xFFFFFFFFu;

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

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
// v / s to the nearest whole number, ties to even, exactly, for s > 0.  The
// quotient in fp32 can fall on a tie that the true one only comes near to; the
// remainder (exact in one fma where the quotient is below 32) tells.
__device__ float nearest(float v, float s) {
  float n = rintf(__fdiv_rn(v, s));
  if (!(fabsf(n) < 32.0f)) return n;  // clamped by the caller
  // bf16 scales can be so small that half of one is no longer exact
  const float up = s < 0x1p-100f ? 0x1p100f : 1.0f;
  const float left = fmaf(-n, s * up, v * up), half = 0.5f * (s * up);
  const bool odd = (static_cast<int>(n) & 1) != 0;
  if (fabsf(left) > half || (fabsf(left) == half && odd)) n += copysignf(1.0f, left);
  return n;
}

// a / kBy, rounded as IEEE asks: a product with the rounded reciprocal, and one
// correction by its exact remainder (Markstein's theorem; it needs the
// remainder not to underflow).
template <int kBy>
__device__ __forceinline__ float divided(float a) {
  constexpr float kOver = 1.0f / kBy;
  const float q = a * kOver, fine = fmaf(fmaf(-q, static_cast<float>(kBy), a), kOver, q);
  return a > 1e-30f && a < 1e38f ? fine : __fdiv_rn(a, static_cast<float>(kBy));
}

// The codes of 8 values of a group, and the sum of their squares in units of
// the scale.  Multiplying by 1 / s and adding 1.5 * 2^23 (and 8) leaves the
// rounded quotient in the lowest bits of the sum; the remainders show whether
// a quotient came so near to a tie that this may be wrong, and then, or where
// the scale was rounded so far that codes have to be clamped (it is
// subnormal), they are computed again with `nearest`.
template <bool kZeros>
__device__ __forceinline__ uint32_t codes_of(const float (&a)[8], float s, bool usable, float most,
                                             float zero, float* square) {
  const float shift = kZeros ? zero : 8.0f;
  const float whole = 12582912.0f + shift, over = __fdividef(1.0f, s), half = 0.5f * s;
  const float cap = 15.0f - shift;
  float worst = 0.0f, sum = 0.0f;
  uint32_t packed = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = __fmaf_rn(a[e], over, whole);
    float n = __fadd_rn(t, -whole);
    worst = fmaxf(worst, fabsf(fmaf(-n, s, a[e])));
    uint32_t bits = __float_as_uint(t);
    if (kZeros) {
      n = fminf(n, cap);
      bits = __float_as_uint(__fadd_rn(n, whole));
    }
    sum = fmaf(n, n, sum);
    packed += bits << (4 * e);
  }
  // each word added was 0x4b400000 + code; of the eight, three reach the end
  packed -= 0x4b400000u + 0xb4000000u + 0x40000000u;
  if (!usable || !(worst < half) || !(most * over < (kZeros ? 15.5f : 7.5f)) || s < 0x1p-100f) {
    packed = 0;
    sum = 0.0f;
    for (int e = 0; e < 8; ++e) {
      float n = 0.0f;
      if (usable) n = fminf(fmaxf(nearest(a[e], s), -shift), cap);
      sum = fmaf(n, n, sum);
      packed |= static_cast<uint32_t>(static_cast<int>(n + shift)) << (4 * e);
    }
  }
  *square = sum;
  return packed;
}

// One warp a row; a lane holds 8 neighbouring values of each 256, so that its
// codes are one word, and asks for 4 such pieces before it works on the first.
// HBM bound in principle: values are read once, codes and scales written once.
// Measured: 78,000 fp16 rows of 1024 values 91 us (200 MB, 31 us at the copy
// bandwidth); issuing bounds it, at some 200 instructions for 256 values.
template <class T, bool kZeros>
__global__ void __launch_bounds__(kThreads) pack_kernel(Q4View v, Q4List l, const T* x, int64_t ld,
                                                        bool vec) {
  constexpr int kAhead = 4, kPieces = sizeof(T) / 2;
  __shared__ ListSmem sm;
  wait_for_stream();
  if (l.seqs && !l.status[kStatusApplied]) return;
  if (!open_list(l, sm)) return;  // as the call that made room found it
  const int lane = threadIdx.x & 31;
  const int span = v.group / 8;  // lanes of a group
  const int dim = static_cast<int>(v.dim), padded = 2 * v.width;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < l.total;
       t += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = list_row(v, l, sm, t);
    if (row < 0) continue;
    const T* in = x + t * ld;
    uint32_t* codes = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(v.codes) + row * v.width);
    uint16_t* scales = const_cast<uint16_t*>(v.scales) + row * v.groups;
    uint8_t* zeros = const_cast<uint8_t*>(v.zeros) + (kZeros ? row * v.groups : 0);
    float norm = 0.0f;
    for (int base = 0; base < padded; base += 256 * kAhead) {
      uint4 raw[kAhead][kPieces];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = base + 256 * u + 8 * lane;
        if (vec && j + 8 <= dim) {
#pragma unroll
          for (int e = 0; e < kPieces; ++e) raw[u][e] = __ldcs(reinterpret_cast<const uint4*>(in + j) + e);
        } else {
          __align__(16) T h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = j + e < dim ? in[j + e] : T(0.0f);
#pragma unroll
          for (int e = 0; e < kPieces; ++e) raw[u][e] = reinterpret_cast<const uint4*>(h)[e];
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (base + 256 * u >= padded) break;
        const int j = base + 256 * u + 8 * lane;
        float a[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = load_value(reinterpret_cast<const T*>(raw[u]) + e);
        float low = 0.0f, high = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          high = max_nan(high, kZeros ? a[e] : fabsf(a[e]));
          if (kZeros) low = max_nan(low, -a[e]);
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          if (d >= span) continue;
          high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, d));
          if (kZeros) low = max_nan(low, __shfl_xor_sync(0xffffffffu, low, d));
        }
        const float wide = kZeros ? divided<15>(high + low) : divided<7>(high);
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
        // a scale of 0, or one that is no finite number: all values at the zero point
        const bool usable = s > 0.0f && s < __int_as_float(0x7f800000);
        float zero = 8.0f, square;
        if (kZeros) zero = usable ? fminf(nearest(low, s), 15.0f) : 0.0f;
        const uint32_t packed = codes_of<kZeros>(a, s, usable, kZeros ? low : high, zero, &square);
        // a scale that is no finite number makes the norm NaN, as the values are
        norm = fmaf(s * s, square, norm);
        if (j < padded) codes[j >> 3] = packed;
        if ((lane & (span - 1)) == 0 && j < dim) {
          scales[j >> v.group_shift] = bits;
          if (kZeros) zeros[j >> v.group_shift] = static_cast<uint8_t>(zero);
        }
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
// One warp a row; a lane turns 4 codes of each 128 into 16 bytes, and asks for
// 8 such pieces before it works on the first.  HBM bound: 4 bytes are written
// for half a byte that is read.  Measured: 78,000 rows of 1024 values 70 us
// (360 MB, 56 us at the copy bandwidth).
template <bool kZeros>
__global__ void __launch_bounds__(kThreads) read_kernel(Q4View v, Q4List l, float* out, int64_t ld,
                                                        bool vec) {
  constexpr int kAhead = 8;
  __shared__ ListSmem sm;
  wait_for_stream();
  if (!open_list(l, sm)) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && l.status)
      atomicCAS(&l.status[kStatusError], 0, KNN_PAGES_BAD_COUNT);
    return;
  }
  const int lane = threadIdx.x & 31, dim = static_cast<int>(v.dim), shift = v.group_shift;
  const bool bf16 = v.scale_bf16;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < l.total;
       t += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = list_row(v, l, sm, t);
    const int64_t from = row < 0 ? 0 : row;
    const uint8_t* codes = v.codes + from * v.width;
    const uint16_t* scales = v.scales + from * v.groups;
    const uint8_t* zeros = v.zeros + (kZeros ? from * v.groups : 0);
    float* to = out + t * ld;
    for (int base = 4 * lane; base < dim; base += 128 * kAhead) {
      uint32_t packed[kAhead], bits[kAhead], zero[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = base + 128 * u;
        if (j >= dim) continue;
        packed[u] = *reinterpret_cast<const uint16_t*>(codes + (j >> 1));
        bits[u] = scales[j >> shift];
        if (kZeros) zero[u] = zeros[j >> shift] & 15u;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = base + 128 * u;
        if (j >= dim) continue;
        float s = __half2float(__ushort_as_half(static_cast<unsigned short>(bits[u])));
        if (bf16) s = __uint_as_float(bits[u] << 16);
        if (row < 0) s = __int_as_float(0x7fc00000);  // no page: NaN
        // 2^23 + code less 2^23 + zero
        const float z = __uint_as_float(0xcb000000u + (kZeros ? zero[u] : 8u));
        float a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          a[e] = __fadd_rn(__uint_as_float(((packed[u] >> (4 * e)) & 15u) | 0x4b000000u), z) * s;
        if (vec && j + 4 <= dim) {
          __stcs(reinterpret_cast<float4*>(to + j), make_float4(a[0], a[1], a[2], a[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + e < dim) to[j + e] = a[e];
        }
      }
    }
  }
}

// --------------------------------------------------------------- products
// What becomes of a product: stored (in the output's type), or the key that a
// search orders rows by, |row|^2 - 2 q.row or -q.row (fp32; a row's place in
// the order does not depend on |q|^2), less a bound of its error.
enum { kStore = 0, kKeyL2 = 1, kKeyProduct = 2 };

// Keys in an order that unsigned numbers have; a key that is no finite number
// belongs to no neighbour.
__device__ __forceinline__ uint32_t ordered(float key) {
  if (!(fabsf(key) < __int_as_float(0x7f800000))) return kNoKey;
  const uint32_t b = __float_as_uint(key);
  return (b >> 31) ? ~b : b | 0x80000000u;
}

struct Q4Out {
  void* y;
  int dtype;
  int64_t ld;
  int mode;
  uint32_t* minima;  // [vectors][minima_ld]: smallest key of each tile of 32 rows
  int64_t minima_ld;
  // keys: a key's error over |x| |row| (products: over sum |x_j| and the row's
  // largest scale), and over |row|^2
  float slack, norm_slack;
};

__device__ __forceinline__ float root(float a) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}

// A lower bound of the true key.  It is the key less what the sums can be off
// by: with steps = 2 group + groups + 32, at most
//   steps 2^-23 sum_j |x_j row_j|
// (a group's values pass through group / 16 matrix instructions that cut 17
// numbers each at 2^-23 of their magnitudes or better, the groups' sums
// through one rounding for each group that follows; the vector's own rounding,
// the splits' adding up and the key's arithmetic are in the 32), and for L2
// what |row|^2 is off by as it is held.  The sum is at most |x| |row|, and for
// products, which need no norms, at most sum |x_j| times 15 (8 without zero
// points) times the row's largest scale.  `size` is |row| or that scale,
// `reach` what it is multiplied by.  2^-126 stands for what subnormal numbers
// lose (2^13 sums of squares up to 1800 in units of 2^-150).
__device__ __forceinline__ float lowest_key(const Q4Out& o, float y, float norm, float reach, float size) {
  constexpr float kMost = 3.402823466e38f, kTiny = 0x1p-126f;
  const float key = o.mode == kKeyL2 ? norm - 2.0f * y : -y;
  const float extra = o.mode == kKeyL2 ? fmaf(o.norm_slack, norm, kTiny) : kTiny;
  const float low = fmaxf(key - fminf(fmaf(reach, size, extra), kMost), -kMost);
  return fabsf(key) <= kMost ? low : __int_as_float(0x7fc00000);
}

// Stores a product or a key.
__device__ __forceinline__ void put(const Q4Out& o, int64_t b, int64_t i, float y) {
  const int64_t at = b * o.ld + i;
  if (o.dtype == KNN_DTYPE_F32) static_cast<float*>(o.y)[at] = y;
  else if (o.dtype == KNN_DTYPE_F16) static_cast<__half*>(o.y)[at] = __float2half_rn(y);
  else static_cast<__nv_bfloat16*>(o.y)[at] = __float2bfloat16_rn(y);
}

// The products run on the warp's own matrix instructions (mma.sync, fp16 in,
// fp32 sums): a row's partial sums have to be scaled after every 32 to 128
// values, which in registers is one multiply-add to a sum, while sums in
// tensor memory would have to be read out and scaled that often (a form that
// was not built, so not measured), and scales multiplied into the weights
// would no longer be exact in 16 bits.  A code
// less its zero point is a whole number of at most 5 bits, so every product
// in the matrix unit is exact, and the rounding is that of fp32 sums.
//
// Vectors become fp16 on the way into shared memory.  fp16 ones are taken as
// they are; bf16 and fp32 ones are first scaled, each vector by a power of
// two of its own that brings its largest finite magnitude to 2^14 .. 2^15,
// and fp32 ones split into two fp16 parts (columns of their own, added up
// at the group's end): high, and what is left, at most 8, times 2^12, so that it
// has 11 bits too where the value is small.  Two parts of 11 bits and a sign
// hold a value to 2^-23 of it; fp16's smallest step, 2^-24, is 2^-50 of the
// largest value in the low part, so x is off by at most 2^-23 |x| + 2^-51
// max|x|: a value has fewer bits only where it is 2^28 below its vector's
// largest, which the sums of a row that is zero at the large ones can show.  A
// bf16 value has 8 bits, and is exact but for 2^-39 max|x|.  Small vectors
// are scaled up, and a bf16 scale can be so large that only the product comes
// down again: such a group's sum is first scaled back by up to 2^-40, which is
// exact and keeps 2^19 values of any size in range.
//
// A warp takes tiles of 32 rows and runs down their codes in stages of 256,
// which it copies ahead into a ring of its own in shared memory (cp.async, no
// barrier between warps); the ring also hands the codes of a group to the
// lanes that the matrix instruction wants them in.  The order of the values
// within a group is free as long as codes and vector agree, so codes are
// unpacked where they lie, by the published way of placing whole numbers in
// the fraction of fp16's 1024 (Kim, Henry, Fahim and Hassan Awadalla, "Who says
// elephants can't run", 2022):
//   word of 8 codes, & 0x000f000f | 0x64006400 = (1024 + c0, 1024 + c4) in
//   fp16, & 0x00f000f0 likewise (1024 + 16 c1, 1024 + 16 c5), and both again
//   8 bits further; one fp16 instruction takes off 1024 + zero (and the 16).
// Rows are few where the matrix is small or wide: the codes of a tile are
// then split over 2 to 16 warps of the block (`split`) and their sums added
// up through shared memory, in order.
//
// Measured (B200; rows of 1024 values in groups of 64, a million of them):
// 1 to 8 fp16 vectors 112 us, 16 of them 146 us (0.64 of the copy bandwidth
// that the 608 MB would allow), 16 fp32 ones 218 us; 1 fp32 vector x 10,000
// rows 9 us, the call included; bf16 scales with bf16 or fp32 vectors 4 to 7% more
// than fp16 ones.  Copying alone, without the products, takes 92 us.  No unit is
// busy all the time: with 4 warps a scheduler (128 registers a thread, one
// block a multiprocessor) an instruction is issued in 56% of the cycles, and
// warps mostly wait for a math pipe (1.4 cycles an instruction) or for the fixed
// latency of the instruction before (1.3); the matrix unit is busy 41% of the
// time, the integer pipe 37%, DRAM 43%.  32 rows x 128 codes are 350
// instructions, of which unpacking is 144, the matrix unit's 32, scaling 32; 12
// warps take as long as 16.  Unpacking by ANDs alone, with the zero points taken
// off by one more matrix product a group, has 64 fewer but was 6% slower.
constexpr int kMmaWarps = 16;
constexpr int kMmaThreads = 32 * kMmaWarps;
constexpr int kTileRows4 = 32;    // rows of a tile
constexpr int kStageCodes = 256;  // codes of a row in a stage: two halves
constexpr int kStageBytes4 = kTileRows4 * kStageCodes / 2;
static_assert(kMmaWarps == kQ4SearchBatch, "a warp to a vector");
constexpr int kRing = 2;          // the stage at hand and the next
constexpr float kLowUp = 4096.0f;  // what an fp32 vector's low part is multiplied by
constexpr int kSumStride = 36;    // floats from column to column of a tile's sums: no bank twice

struct MmaPlan {
  int64_t tiles;
  int32_t iterations;    // tiles that a warp's slot goes through, at most
  int32_t stages;        // of 256 codes in a row
  int32_t chunk_stages;  // stages whose share of the vectors fits in shared memory
  int32_t chunks;
  int32_t split;  // warps that share a tile
};

// Dynamic shared memory: ring[warp][kRing][kStageBytes4], then scales[warp][2]
// [groups of a stage][32 rows], then (split > 1) sums[warp][vector]
// [kSumStride] and for keys of products largest[warp][kSumStride], then the
// vectors.  Before the ring is used, mosts[vector][warp] and sizes[vector][warp]
// lie in its place.
struct MmaShared {
  // a vector's power of two, and its inverse in two steps: taken off a group's
  // sum before the scale multiplies it (bf16 scales), and off the product
  float factor[kQ4SearchBatch], early[kQ4SearchBatch], inverse[kQ4SearchBatch];
  float reach[kQ4SearchBatch];  // of a vector's keys
  // rows of the tiles that a warp is at, by iteration: it copies ahead by up
  // to two stages, so by as many tiles
  int32_t rows[kMmaWarps][4][kTileRows4];
};

__device__ __forceinline__ void copy_ahead(void* to, const void* from, bool valid) {
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  const int size = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(from),
               "r"(size)
               : "memory");
}
__device__ __forceinline__ void copy_close() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// d = a b + c
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                          float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// (a & b) | c in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t sixteenth2(uint32_t a, uint32_t c) {
  const uint32_t s = 0x2c002c00u;  // 1/16
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<const __half2*>(&s),
                            *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Which 16 bytes of a row's 128 in a stage lie where: rows 0 .. 7 put them at
// piece ^ swizzle(row), the row's bits in reverse, so that the three ways below
// to read them (4, 8 or 16 bytes a lane) meet no bank twice.
__device__ __forceinline__ int swizzle(int row) {
  return ((row & 1) << 2) | (row & 2) | ((row >> 2) & 1);
}

// The stages of a chunk that fall to a warp.
__device__ __forceinline__ void part_of(const MmaPlan& p, int chunk, int part, int* first, int* end) {
  const int start = chunk * p.chunk_stages;
  int len = p.stages - start;
  if (len > p.chunk_stages) len = p.chunk_stages;
  *first = start + part * len / p.split;
  *end = start + (part + 1) * len / p.split;
}

// The scales and zero points of a stage's groups in one row, as they are held.
template <int kGroups>
struct HeldScales {
  uint32_t s[kGroups];            // two scales each
  uint32_t z[(kGroups + 1) / 2];  // four zero points each (kGroups = 1: two)
};

// kCols: columns of the matrix instruction in tiles of 8 (kTiles of them);
// kParts: fp16 parts of a vector.  With kTiles = 1 and two parts, columns 0-3
// hold the high parts of 4 vectors and 4-7 the low ones; otherwise the tiles'
// first half holds the high parts.  kGroups: groups in half a stage (128 / group).
// kKeyed: keys (o.mode says which), not products to store.
template <class T, int kTiles, int kParts, int kGroups, bool kZeros, bool kKeyed>
__global__ void __launch_bounds__(kMmaThreads, 1)
    products_kernel(Q4View v, Q4Range r, const T* x, int batch, int64_t ldx, Q4Out o, MmaPlan p) {
  constexpr bool kPacked = kTiles == 1 && kParts == 2;
  constexpr int kOutTiles = kPacked ? 1 : kTiles / kParts;
  constexpr int kPerGroup = 4 / kGroups;  // words of 8 codes a lane has in a group
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ MmaShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = raw + warp * (kRing * kStageBytes4);
  constexpr int kScales = 2 * kGroups * kTileRows4;  // words of a stage's scales
  uint32_t* scales = reinterpret_cast<uint32_t*>(raw + kMmaWarps * kRing * kStageBytes4) +
                     warp * (2 * kScales);
  float* sums = reinterpret_cast<float*>(raw + kMmaWarps * (kRing * kStageBytes4 + 2 * kScales * 4));
  const int sum_words = batch * kSumStride;  // of a warp
  float* largest = sums + kMmaWarps * sum_words;
  uint4* vectors = reinterpret_cast<uint4*>(
      p.split == 1 ? sums : largest + (kKeyed && o.mode == kKeyProduct ? kMmaWarps * kSumStride : 0));
  const int slots = kMmaWarps / p.split, slot = warp / p.split, part = warp % p.split;

  wait_for_stream();
  int64_t n = r.count;
  if (r.length) n = *r.length < n ? *r.length : n;

  auto tile_of = [&](int iteration) {
    return (static_cast<int64_t>(iteration) * slots + slot) * gridDim.x + blockIdx.x;
  };
  const int64_t stride = static_cast<int64_t>(slots) * gridDim.x;
  const int mine = static_cast<int>((p.tiles - tile_of(0) + stride - 1) / stride);  // this slot's tiles
  // this lane's row of a tile, as a row number in the pools; -1: none
  auto row_of = [&](int iteration) -> int32_t {
    const int64_t i = tile_of(iteration) * kTileRows4 + lane;
    return i < n ? static_cast<int32_t>(v.places.at(r.seq, i)) : -1;
  };

  // ---- copying codes ahead, and the scales with them.  Lane (g, t) copies 16
  // bytes of rows g, g + 8, g + 16 and g + 24, and holds the scales of row
  // g + 8 t.  A row that does not exist is read as the tile's first that does;
  // what comes of it is replaced in the end.  (Reading row 0 instead made
  // every warp that had run out of rows ask for the same few lines: a million
  // rows took 208 us instead of 131.)  A tile without rows copies nothing.
  int next_iteration = 0, next_chunk = 0, next_stage, next_end;
  part_of(p, 0, part, &next_stage, &next_end);
  int32_t row_after = row_of(0);
  const uint8_t* from[4];
  int64_t scales_at = 0;
  bool some = false;  // the tile has rows
  const bool together = v.groups % (2 * kGroups) == 0 &&
                        reinterpret_cast<uintptr_t>(v.scales) % (4 * kGroups) == 0 &&
                        (!kZeros || reinterpret_cast<uintptr_t>(v.zeros) % (2 * kGroups) == 0);
  auto enter_tile = [&]() {
    const int32_t row = row_after;
    sh.rows[warp][next_iteration & 3][lane] = row;
    row_after = row_of(next_iteration + 1);
    const uint32_t exist = __ballot_sync(0xffffffffu, row >= 0);
    some = exist != 0;
    const int32_t first = __shfl_sync(0xffffffffu, row, some ? __ffs(exist) - 1 : 0);
    const int32_t read = row >= 0 ? row : some ? first : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      from[i] = v.codes + static_cast<int64_t>(__shfl_sync(0xffffffffu, read, g + 8 * i)) * v.width;
    scales_at = static_cast<int64_t>(__shfl_sync(0xffffffffu, read, g + 8 * t)) * v.groups;
  };
  enter_tile();
  const int quarters = v.width >> 4;  // 16-byte pieces of a row
  const int to_lane = g * 128 + ((t ^ swizzle(g)) << 4);
  HeldScales<kGroups> held;
  auto send = [&](uint8_t* to) {
    if (next_iteration < mine) {
      const uint32_t ahead = 128u * next_stage + 16u * t;
      const bool near = some && 8 * next_stage + t < quarters;
      const bool far = some && 8 * next_stage + 4 + t < quarters;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // of what lies behind the row nothing is read, and zeros are written
        copy_ahead(to + to_lane + i * 1024, from[i] + (near ? ahead : 0u), near);
        copy_ahead(to + (to_lane ^ 64) + i * 1024, from[i] + (far ? ahead + 64u : 0u), far);
      }
      const int64_t j = scales_at + 2 * kGroups * next_stage;
      held = {};
      if (!some) {
      } else if (together) {
        if constexpr (kGroups == 1) held.s[0] = *reinterpret_cast<const uint32_t*>(v.scales + j);
        if constexpr (kGroups == 2)
          *reinterpret_cast<uint2*>(held.s) = *reinterpret_cast<const uint2*>(v.scales + j);
        if constexpr (kGroups == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(v.scales + j);
          held.s[0] = u.x, held.s[1] = u.y, held.s[2] = u.z, held.s[3] = u.w;
        }
        if constexpr (kZeros && kGroups == 1) held.z[0] = *reinterpret_cast<const uint16_t*>(v.zeros + j);
        if constexpr (kZeros && kGroups == 2) held.z[0] = *reinterpret_cast<const uint32_t*>(v.zeros + j);
        if constexpr (kZeros && kGroups == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(v.zeros + j);
          held.z[0] = u.x, held.z[1] = u.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2 * kGroups; ++e)
          if (2 * kGroups * next_stage + e < v.groups) {
            held.s[e >> 1] |= static_cast<uint32_t>(v.scales[j + e]) << (16 * (e & 1));
            if (kZeros) held.z[e >> 2] |= static_cast<uint32_t>(v.zeros[j + e]) << (8 * (e & 3));
          }
      }
      if (++next_stage == next_end) {
        do {
          if (++next_chunk == p.chunks) {
            next_chunk = 0;
            if (++next_iteration < mine) enter_tile();
          }
          part_of(p, next_chunk, part, &next_stage, &next_end);
        } while (next_stage == next_end);
      }
    }
    copy_close();
  };
  // Puts the scales that came with the last stage sent where every lane of the
  // warp finds those of its four rows side by side: as fp32, or with zero
  // points as they are held, below 1024 + zero in fp16.
  auto put_scales = [&](uint32_t* to) {
    to += lane;
    if constexpr (kZeros) {
#pragma unroll
      for (int j = 0; j < 2 * kGroups; ++j)
        to[j * kTileRows4] = ((held.s[j >> 1] >> (16 * (j & 1))) & 0xffffu) |
                             ((held.z[j >> 2] >> (8 * (j & 3))) & 15u) << 16 | 0x64000000u;
    } else if (v.scale_bf16) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        to[2 * j * kTileRows4] = held.s[j] << 16;
        to[(2 * j + 1) * kTileRows4] = held.s[j] & 0xffff0000u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&held.s[j]));
        to[2 * j * kTileRows4] = __float_as_uint(two.x);
        to[(2 * j + 1) * kTileRows4] = __float_as_uint(two.y);
      }
    }
  };
  // ---- the vectors' powers of two, and what their keys can be off by: 16 /
  // batch warps read a vector, and a warp adds up what they found
  constexpr bool kAsHeld = std::is_same<T, __half>::value;
  if constexpr (!kAsHeld || kKeyed) {
    uint32_t* mosts = reinterpret_cast<uint32_t*>(raw);
    float* sizes = reinterpret_cast<float*>(raw) + kMmaWarps * kQ4SearchBatch;
    int shift = 4;
    while ((batch << shift) > kMmaWarps) --shift;
    const int each = 1 << shift, part = warp & (each - 1), from_vector = warp >> shift;
    if (from_vector < batch) {
      uint32_t most = 0;
      float size = 0.0f;
      for (int base = 32 * part + lane; base < static_cast<int>(v.dim); base += 128 << shift) {
        float a[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = base + (u << (shift + 5));
          a[u] = j < static_cast<int>(v.dim) ? load_value(x + from_vector * ldx + j) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t bits = __float_as_uint(a[u]) & 0x7fffffffu;
          if (!kAsHeld && bits < 0x7f800000u && bits > most) most = bits;
          if constexpr (kKeyed) size = o.mode == kKeyL2 ? fmaf(a[u], a[u], size) : size + fabsf(a[u]);
        }
      }
      if constexpr (!kAsHeld) most = __reduce_max_sync(0xffffffffu, most);
      if constexpr (kKeyed) {
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) size += __shfl_xor_sync(0xffffffffu, size, d);
      }
      if (lane == 0) {
        mosts[from_vector * kMmaWarps + part] = most;
        sizes[from_vector * kMmaWarps + part] = size;
      }
    }
    __syncthreads();
    const bool mine_too = warp < batch && lane < each;
    const uint32_t most = __reduce_max_sync(0xffffffffu, mine_too ? mosts[warp * kMmaWarps + lane] : 0);
    float size = mine_too ? sizes[warp * kMmaWarps + lane] : 0.0f;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) size += __shfl_xor_sync(0xffffffffu, size, d);
    if (lane == 0) {
      int e = most ? 14 - (static_cast<int>(most >> 23) - 127) : 0;
      if (e > 126) e = 126;
      const int first = v.scale_bf16 && e > 0 ? (e < 40 ? e : 40) : 0;
      sh.factor[warp] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      sh.early[warp] = __uint_as_float(static_cast<uint32_t>(127 - first) << 23);
      sh.inverse[warp] = __uint_as_float(static_cast<uint32_t>(127 - e + first) << 23);
      // squares below 2^-149 are lost: 2^-66 is what 2^16 of them can come to
      if (kKeyed && o.mode == kKeyL2) size = root(size) + 0x1p-66f;
      if constexpr (kKeyed) sh.reach[warp] = o.slack * size;
    }
  } else if (threadIdx.x < kQ4SearchBatch) {
    sh.factor[threadIdx.x] = sh.early[threadIdx.x] = sh.inverse[threadIdx.x] = 1.0f;
  }
  __syncthreads();

  // ---- a chunk of the vectors, as the matrix instruction takes them
  const bool wide = ((reinterpret_cast<uintptr_t>(x) | (ldx * sizeof(T))) & 15) == 0;
  auto stage_vectors = [&](int chunk) {
    const int first = chunk * p.chunk_stages;
    int len = p.stages - first;
    if (len > p.chunk_stages) len = p.chunk_stages;
    for (int item = threadIdx.x; item < len * 8 * kTiles * 32; item += kMmaThreads) {
      const int l = item & 31, tile = (item >> 5) % kTiles, word = (item >> 5) / kTiles;
      const int w = word & 3, column = l >> 2, q = l & 3;
      int b, low;
      if constexpr (kPacked) {
        b = column & 3, low = column >> 2;
      } else {
        b = (tile % kOutTiles) * 8 + column, low = tile / kOutTiles;
      }
      int k = kStageCodes * first + 128 * (word >> 2);
      if constexpr (kGroups == 4) k += 32 * w + 8 * q;
      else if constexpr (kGroups == 2) k += 64 * (w >> 1) + 16 * q + 8 * (w & 1);
      else k += 32 * q + 8 * w;
      float a[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = 0.0f;
      if (b < batch && k < v.dim) {
        const T* from = x + b * ldx + k;
        if (wide && k + 8 <= v.dim) {
          __align__(16) T h[8];
#pragma unroll
          for (int e = 0; e < static_cast<int>(sizeof(T)) / 2; ++e)
            reinterpret_cast<uint4*>(h)[e] = reinterpret_cast<const uint4*>(from)[e];
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = load_value(h + e);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k + e < v.dim) a[e] = load_value(from + e);
        }
      }
      const float f = b < batch ? sh.factor[b] : 1.0f;
      __half h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float scaled = a[e] * f;
        h[e] = __float2half_rn(scaled);
        if (kParts == 2 && low) {
          const float high = __half2float(h[e]);
          h[e] = __float2half_rn(fabsf(high) <= 65504.0f ? (scaled - high) * kLowUp : 0.0f);
        }
      }
      uint4 out;
      out.x = __half_as_ushort(h[0]) | static_cast<uint32_t>(__half_as_ushort(h[4])) << 16;
      out.y = __half_as_ushort(h[1]) | static_cast<uint32_t>(__half_as_ushort(h[5])) << 16;
      out.z = __half_as_ushort(h[2]) | static_cast<uint32_t>(__half_as_ushort(h[6])) << 16;
      out.w = __half_as_ushort(h[3]) | static_cast<uint32_t>(__half_as_ushort(h[7])) << 16;
      vectors[item] = out;
    }
  };
  stage_vectors(0);
  send(ring);
  put_scales(scales);
  send(ring + kStageBytes4);

  __syncthreads();

  uint32_t ring_at = 0;     // bytes into the ring
  uint32_t scales_now = 0;  // words into the scales
  for (int iteration = 0; iteration < p.iterations; ++iteration) {
    float total[2][kOutTiles][4] = {};
    float most_scale[4] = {};  // of rows g + 8 i, for keys of products
    for (int chunk = 0; chunk < p.chunks; ++chunk) {
      if (p.chunks > 1 && (iteration > 0 || chunk > 0)) {
        __syncthreads();
        stage_vectors(chunk);
        __syncthreads();
      }
      int stage, end;
      part_of(p, chunk, part, &stage, &end);
      if (iteration >= mine) end = stage;
      const uint4* vec = vectors + (stage - chunk * p.chunk_stages) * (8 * kTiles * 32) + lane;
#pragma unroll 1
      for (; stage < end; ++stage, vec += 8 * kTiles * 32) {
        copy_wait<1>();
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t* codes = ring + ring_at + g * 128;
          uint32_t words[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* c = codes + i * 1024;
            if constexpr (kGroups == 4) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                words[i][j] = *reinterpret_cast<const uint32_t*>(
                    c + (((4 * half + j) ^ swizzle(g)) << 4) + 4 * t);
            } else if constexpr (kGroups == 2) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint2 u = *reinterpret_cast<const uint2*>(
                    c + (((4 * half + 2 * j + (t >> 1)) ^ swizzle(g)) << 4) + 8 * (t & 1));
                words[i][2 * j] = u.x;
                words[i][2 * j + 1] = u.y;
              }
            } else {
              const uint4 u = *reinterpret_cast<const uint4*>(c + (((4 * half + t) ^ swizzle(g)) << 4));
              words[i][0] = u.x, words[i][1] = u.y, words[i][2] = u.z, words[i][3] = u.w;
            }
          }
          const uint32_t* scale_row = scales + scales_now + half * (kGroups * kTileRows4) + 4 * g;
          if (half == 1) {
            // the codes of this stage are in registers: the one after the next
            // takes their place
            __syncwarp();
            scales_now ^= kScales;
            put_scales(scales + scales_now);
            send(ring + ring_at);
            ring_at ^= kStageBytes4;
            if (kStageCodes * stage + 128 >= v.dim) continue;
          }
#pragma unroll
          for (int j = 0; j < kGroups; ++j) {
            float acc[2][kTiles][4], scale[4];
            uint32_t one[4], sixteen[4];
            const uint4 s4 = *reinterpret_cast<const uint4*>(scale_row + j * kTileRows4);
            const uint32_t held4[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (kZeros) {
                scale[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(held4[i])));
                if (v.scale_bf16) scale[i] = __uint_as_float(held4[i] << 16);
                one[i] = __byte_perm(held4[i], 0, 0x3232);                     // 1024 + zero
                sixteen[i] = ((one[i] & 0x000f000fu) << 4) | 0xd400d400u;      // -(64 + zero)
              } else {
                scale[i] = __uint_as_float(held4[i]);
                one[i] = 0x64086408u;
                sixteen[i] = 0xd480d480u;
              }
            }
            if constexpr (kKeyed) {  // for both keys: a branch costs more
#pragma unroll
              for (int i = 0; i < 4; ++i) most_scale[i] = fmaxf(most_scale[i], fabsf(scale[i]));
            }
#pragma unroll
            for (int w = j * kPerGroup; w < (j + 1) * kPerGroup; ++w) {
              uint32_t a[4][4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t u = words[i][w], far = u >> 8;
                a[i][0] = sub2(and_or(u, 0x000f000fu, 0x64006400u), one[i]);
                a[i][1] = sixteenth2(and_or(u, 0x00f000f0u, 0x64006400u), sixteen[i]);
                a[i][2] = sub2(and_or(far, 0x000f000fu, 0x64006400u), one[i]);
                a[i][3] = sixteenth2(and_or(far, 0x00f000f0u, 0x64006400u), sixteen[i]);
              }
#pragma unroll
              for (int c = 0; c < kTiles; ++c) {
                const uint4 b = vec[((4 * half + w) * kTiles + c) * 32];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                  float(&d)[4] = acc[m][c];
                  if (w == j * kPerGroup)
                    mma_16816(d, a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b.x,
                              b.y, 0.0f, 0.0f, 0.0f, 0.0f);
                  else
                    mma_16816(d, a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b.x,
                              b.y, d[0], d[1], d[2], d[3]);
                  mma_16816(d, a[2 * m][2], a[2 * m + 1][2], a[2 * m][3], a[2 * m + 1][3], b.z, b.w,
                            d[0], d[1], d[2], d[3]);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int m = i >> 1, h = 2 * (i & 1);
#pragma unroll
              for (int c = 0; c < kOutTiles; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float sum = acc[m][c][h + e];
                  if constexpr (!kPacked && kParts == 2)
                    sum = fmaf(acc[m][c + kOutTiles][h + e], 1.0f / kLowUp, sum);
                  if constexpr (!std::is_same<T, __half>::value)
                    if (v.scale_bf16) sum *= sh.early[kPacked ? (2 * t + e) & 3 : 8 * c + 2 * t + e];
                  total[m][c][h + e] = fmaf(scale[i], sum, total[m][c][h + e]);
                }
            }
          }
        }
      }
    }
    if constexpr (kPacked) {  // the low parts' columns are two lanes on
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          total[m][0][e] =
              fmaf(__shfl_xor_sync(0xffffffffu, total[m][0][e], 2), 1.0f / kLowUp, total[m][0][e]);
    }
    const int64_t first = tile_of(iteration) * kTileRows4;
    if (p.split == 1) {
      if (iteration >= mine) continue;
      int32_t rows[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = sh.rows[warp][iteration & 3][g + 8 * i];
      const bool whole = __all_sync(0xffffffffu, (rows[0] | rows[1] | rows[2] | rows[3]) >= 0);
      if (whole) {  // all but the last tile: no tests of single rows
        [[maybe_unused]] float norm[4], size[4];
#pragma unroll
        for (int i = 0; kKeyed && i < 4; ++i) {
          norm[i] = o.mode == kKeyL2 ? v.norms[rows[i]] : 0.0f;
          size[i] = o.mode == kKeyL2 ? root(norm[i]) : most_scale[i];
        }
#pragma unroll
        for (int c = 0; c < kOutTiles; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (8 * c + e >= batch) continue;  // no lane has a vector
            const int b = 8 * c + 2 * t + e;
            const bool real = b < batch && (!kPacked || t < 2);
            const float f = real ? sh.inverse[b] : 0.0f;
            [[maybe_unused]] const float reach = kKeyed && real ? sh.reach[b] : 0.0f;
            const int64_t at = b * o.ld + first + g;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y[i] = total[i >> 1][c][2 * (i & 1) + e] * f;
              if constexpr (kKeyed) y[i] = lowest_key(o, y[i], norm[i], reach, size[i]);
            }
            if (real) {
              if (kKeyed || o.dtype == KNN_DTYPE_F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) static_cast<float*>(o.y)[at + 8 * i] = y[i];
              } else if (o.dtype == KNN_DTYPE_F16) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  static_cast<__half*>(o.y)[at + 8 * i] = __float2half_rn(y[i]);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  static_cast<__nv_bfloat16*>(o.y)[at + 8 * i] = __float2bfloat16_rn(y[i]);
              }
            }
            if constexpr (kKeyed) {
              uint32_t least = min(min(ordered(y[0]), ordered(y[1])), min(ordered(y[2]), ordered(y[3])));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1)
                least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
              if (g == 0 && real) o.minima[b * o.minima_ld + first / kTileRows4] = least;
            }
          }
        continue;
      }
#pragma unroll
      for (int c = 0; c < kOutTiles; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int b = 8 * c + 2 * t + e;
          const bool mine_too = b < batch && (!kPacked || t < 2);
          uint32_t least = kNoKey;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t at = first + g + 8 * i;
            if (!mine_too || at >= r.count) continue;
            float y = total[i >> 1][c][2 * (i & 1) + e] * sh.inverse[b];
            if (rows[i] < 0) y = at < n ? __int_as_float(0x7fc00000) : 0.0f;
            if constexpr (kKeyed) {
              const float norm = o.mode == kKeyL2 && rows[i] >= 0 ? v.norms[rows[i]] : 0.0f;
              y = lowest_key(o, y, norm, sh.reach[b], o.mode == kKeyL2 ? root(norm) : most_scale[i]);
            }
            put(o, b, at, y);
            if (at < n) least = min(least, ordered(y));
          }
          if constexpr (kKeyed) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
              least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
            if (g == 0 && mine_too) o.minima[b * o.minima_ld + first / kTileRows4] = least;
          }
        }
    } else {
      float* own = sums + warp * sum_words;
#pragma unroll
      for (int c = 0; c < kOutTiles; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int b = 8 * c + 2 * t + e;
          if (b >= batch || (kPacked && t >= 2)) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            own[b * kSumStride + g + 8 * i] = total[i >> 1][c][2 * (i & 1) + e];
        }
      if (kKeyed && o.mode == kKeyProduct && t == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) largest[warp * kSumStride + g + 8 * i] = most_scale[i];
      }
      __syncthreads();
      // a warp to a tile and vector, a lane to a row
      for (int item = warp; item < slots * batch; item += kMmaWarps) {
        const int s = item / batch, b = item - s * batch;
        const int64_t tile = (static_cast<int64_t>(iteration) * slots + s) * gridDim.x + blockIdx.x;
        if (tile >= p.tiles) continue;
        const int64_t at = tile * kTileRows4 + lane;
        float y = 0.0f;
        for (int q = 0; q < p.split; ++q)
          y += sums[(s * p.split + q) * sum_words + b * kSumStride + lane];
        y *= sh.inverse[b];
        const int32_t at_row = sh.rows[s * p.split][iteration & 3][lane];
        if (at_row < 0) y = at < n ? __int_as_float(0x7fc00000) : 0.0f;
        uint32_t least = kNoKey;
        if (at < r.count) {
          if constexpr (kKeyed) {
            const float norm = o.mode == kKeyL2 && at_row >= 0 ? v.norms[at_row] : 0.0f;
            float size = root(norm);
            if (o.mode == kKeyProduct)
              for (int q = 0; q < p.split; ++q)
                size = fmaxf(size, largest[(s * p.split + q) * kSumStride + lane]);
            y = lowest_key(o, y, norm, sh.reach[b], size);
          }
          put(o, b, at, y);
          if (at < n) least = ordered(y);
        }
        if constexpr (kKeyed) {
          least = __reduce_min_sync(0xffffffffu, least);
          if (lane == 0) o.minima[b * o.minima_ld + tile] = least;
        }
      }
      __syncthreads();
    }
  }
  copy_wait<0>();
}

// ----------------------------------------------------------------- search
constexpr int kGroupRows = kTileRows4;  // rows whose smallest key is kept
constexpr int kSelectThreads = 1024;
constexpr int kMoreCandidates = 16;  // scored again beyond the k asked for
constexpr int kScoreCap = 1024;      // rows that are scored at a time
constexpr int kGroupCap = 1024;  // kSelectThreads at least: one group a thread is listed at a time
constexpr int kCandCap = 4096;
static_assert(kGroupCap >= kSelectThreads && kScoreCap <= 32 * 32 && kScoreCap >= KNN_MAX_K + 2 * kMoreCandidates);
constexpr int kRankCap = 512;  // candidates that are ranked by counting, not sorted

constexpr int kBins = 2048;
constexpr int kQueryHeld = 8192;  // values up to which a query is kept in shared memory

struct SelectSmem {
  // values 8 i + 2 f and 8 i + 2 f + 1 in [f][i]: lanes take values 8 apart, and
  // 64 bytes apart they would meet in the banks (42 us a search's end, not 35)
  double2 query[4][kQueryHeld / 8];  // zeros behind the last value
  uint64_t cand[kCandCap];
  uint32_t pick[kScoreCap];  // rows to score again
  // the nearest so far, and those just scored
  uint64_t final_key[KNN_MAX_K + kScoreCap];
  uint32_t final_row[KNN_MAX_K + kScoreCap];
  uint64_t best_key[KNN_MAX_K];
  uint32_t best_row[KNN_MAX_K];
  float squared;    // |q|^2 from below
  uint32_t fresh;   // rows just scored that are among the nearest so far
  uint32_t hist[kBins];
  uint32_t part[32];
  int32_t group[kGroupCap];
  uint32_t count, groups;
  uint64_t prefix, last;
  int64_t rank;
  int64_t inside;  // values in the bin
};

// Adds one to the bin of each thread that has one (bin < kBins).  Keys share
// their leading bits: a warp adds up equal bins first.
__device__ __forceinline__ void count_bin(SelectSmem& sm, uint32_t bin) {
  const uint32_t same = __match_any_sync(0xffffffffu, bin);
  if (bin < kBins && (threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&sm.hist[bin], __popc(same));
}

// The bin that the value of rank `rank` falls in, (in sm.rank) its rank there
// and (in sm.inside) how many there are.  All threads; the bins are cleared for
// the next count.
__device__ uint32_t find_bin(SelectSmem& sm, int64_t rank) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kPer = kBins / kSelectThreads;
  __syncthreads();
  uint32_t h[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    sum += h[j] = sm.hist[kPer * threadIdx.x + j];
    sm.hist[kPer * threadIdx.x + j] = 0;
  }
  uint32_t inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 31) sm.part[warp] = inc;
  __syncthreads();
  uint32_t before = sm.part[lane], all = before;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, all, d);
    if (lane >= d) all += up;
  }
  const uint32_t first = __shfl_sync(0xffffffffu, all - before, warp);
  int64_t left = rank - static_cast<int64_t>(first + inc - sum);
  if (left >= 0 && left < static_cast<int64_t>(sum)) {
    int j = 0;
    while (left >= static_cast<int64_t>(h[j])) left -= h[j++];
    sm.prefix = static_cast<uint64_t>(kPer * threadIdx.x + j);
    sm.rank = left;
    sm.inside = h[j];
  }
  __syncthreads();
  return static_cast<uint32_t>(sm.prefix);
}

// The 64-bit value of rank `rank` (from 0) among load(0 .. n - 1), 11 bits a
// pass from the top.
template <class Load>
__device__ uint64_t nth(int64_t n, int64_t rank, SelectSmem& sm, Load load) {
  uint64_t prefix = 0;
  for (int top = 64; top > 0;) {
    const int shift = top > 11 ? top - 11 : 0;
    const uint64_t above = top == 64 ? 0 : ~0ull << top;
    const uint32_t mask = (1u << (top - shift)) - 1;
    for (int64_t base = 0; base < n; base += kSelectThreads) {
      const int64_t i = base + threadIdx.x;
      const uint64_t x = i < n ? load(i) : 0;
      const bool in = i < n && (x & above) == prefix;
      count_bin(sm, in ? static_cast<uint32_t>(x >> shift) & mask : static_cast<uint32_t>(kBins));
    }
    prefix |= static_cast<uint64_t>(find_bin(sm, rank)) << shift;
    rank = sm.rank;
    top = shift;
  }
  __syncthreads();
  return prefix;
}

// A bound that at least `wanted` of the minima lie at or below, and hardly
// more: the range of the minima is cut into 2048 equal bins of their ordered
// form, the bin of the wanted rank again, until few enough lie at or below its
// end.  Equal bins of the range that there is, not of a number's bits: minima
// share those, and atomics on one bin run one after another.  Where fewer groups
// than wanted have a key at all (a sequence much shorter than the count, pages
// missing), the bound is above every key: nothing says how many rows lie at or
// below the largest minimum.
__device__ uint32_t minima_bound(const uint32_t* minima, int64_t groups, int wanted,
                                 SelectSmem& sm) {
  auto each = [&](auto&& f) {
#pragma unroll 4
    for (int64_t i = 4 * threadIdx.x; i < groups; i += 4 * kSelectThreads) {
      const uint4 u = *reinterpret_cast<const uint4*>(minima + i);
      f(u.x);
      if (i + 1 < groups) f(u.y);
      if (i + 2 < groups) f(u.z);
      if (i + 3 < groups) f(u.w);
    }
  };
  uint32_t low = kNoKey, high = 0;
  each([&](uint32_t x) {
    if (x != kNoKey) low = min(low, x), high = max(high, x);
  });
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (threadIdx.x == 0) sm.count = kNoKey, sm.groups = 0;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&sm.count, low);
    atomicMax(&sm.groups, high);
  }
  __syncthreads();
  low = sm.count, high = sm.groups;
  if (low > high) return kNoKey - 1;  // no keys at all
  int64_t rank = wanted - 1;          // counted from low
  int64_t below = 0;                  // minima below low
  while (true) {
    // bins of 2^shift, 2048 of which reach over the range
    const int bits = 32 - __clz(high - low);
    const int shift = bits > 11 ? bits - 11 : 0;
    each([&](uint32_t x) {
      if (x != kNoKey && x >= low && x <= high) atomicAdd(&sm.hist[(x - low) >> shift], 1u);
    });
    if (threadIdx.x == 0) sm.rank = -1;
    const uint32_t bin = find_bin(sm, rank);
    if (sm.rank < 0) return kNoKey - 1;  // fewer keys than wanted
    const uint32_t first = low + (bin << shift);
    const uint32_t last = min(high, first + ((1u << shift) - 1u));
    const int64_t inside = sm.inside;
    below += rank - sm.rank;
    if (shift == 0 || below + inside <= wanted + wanted / 2 + 32) return last;
    rank = sm.rank;
    low = first;
    high = last;
    __syncthreads();
  }
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

// One CTA a query: the k + 16 rows of smallest (key, index), or a few more, their
// distances again in 64 bits, and the k first of those.
//
// The keys' sums are fp32 and rounded; near neighbours lie close together, so
// that order alone would depend on the order of the sums.  The distances of
// the candidates are summed again in 64 bits, which settles it.  A candidate
// whose distance is no finite number in fp32 is dropped then (its key may be:
// |q|^2 is not in it).  A query that is not finite makes no key that is.
//
// Keys are lower bounds, so a row is no neighbour if its key is above the k-th
// distance (less |q|^2).  Mostly that holds for every row that is no
// candidate.  Where it does not (near copies of one row, rows whose sums
// cancel), the other rows with keys up to that distance are scored too, up to
// 1024 at a time, while the k-th distance comes down: the result is the exact
// one always, and such a search takes longer the more rows there are that
// fp32 cannot tell apart (a million rows of 1024 values, one query, k = 10: 0.15
// ms, with 1000 copies of the nearest 0.25, with 10,000 of them 3.0, most of it
// the pass over all keys, with 100,000 10).
//
// Candidates: with c wanted and tau the c-th smallest of the groups' minima,
// c rows lie at or below tau, so only keys <= tau are looked at, and they are
// in the groups whose minimum is <= tau: c groups, unless keys are equal.
//
// A latency: one CTA goes through it for each query.  Measured: 12 us for the
// 10 nearest of 125,000 rows of 1024 values, 31 us for the 100 nearest of a
// million for each of 16 queries, about half of it the scoring.
template <class T, int kMode, bool kWide>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(
    Q4View v, Q4Range r, const T* x, int64_t ldx, const float* keys, int64_t ld,
    const uint32_t* minima, int64_t groups, int k, int64_t* neighbors, float* distances) {
  extern __shared__ __align__(16) uint8_t raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(raw);
  wait_for_stream();
  const int64_t b = blockIdx.x;
  int64_t n = r.count;
  if (r.length) n = *r.length < n ? *r.length : n;
  keys += b * ld;
  minima += b * ((groups + 3) / 4 * 4);  // 16-byte aligned
  const int wanted = k + kMoreCandidates;
  uint32_t tau = kNoKey - 1;
  for (int i = threadIdx.x; i < kBins; i += kSelectThreads) sm.hist[i] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int j = threadIdx.x; !kWide && j < ((v.dim + 255) & ~255ll); j += kSelectThreads) {
    const double value = j < v.dim ? static_cast<double>(load_value(x + b * ldx + j)) : 0.0;
    double2& pair = sm.query[(j & 7) >> 1][j >> 3];
    (j & 1 ? pair.y : pair.x) = value;
  }
  if (threadIdx.x == 0) sm.fresh = 0;
  __syncthreads();
  if (groups > wanted) tau = min(minima_bound(minima, groups, wanted, sm), kNoKey - 1);
  __syncthreads();
  if (threadIdx.x == 0) sm.count = sm.groups = 0;
  __syncthreads();
#pragma unroll 4
  for (int64_t g = 4 * threadIdx.x; g < groups; g += 4 * kSelectThreads) {
    const uint4 u = *reinterpret_cast<const uint4*>(minima + g);
    const uint32_t least[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (g + j < groups && least[j] <= tau) {
        const uint32_t at = atomicAdd(&sm.groups, 1u);
        if (at < kGroupCap) sm.group[at] = static_cast<int32_t>(g + j);
      }
  }
  __syncthreads();
  const uint32_t listed = sm.groups;
  if (listed <= kGroupCap) {
#pragma unroll 4
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
  constexpr int kSelectWarps = kSelectThreads / 32;
  int have;
  uint64_t last;  // (key, index) of the last candidate, all ones where there are no other rows
  if (listed <= kGroupCap && sm.count <= kCandCap) {
    const int count = static_cast<int>(sm.count);
    have = min(count, wanted);
    if (count <= wanted + kMoreCandidates) {  // a few more do no harm
      have = count;
      last = tau == kNoKey - 1 ? ~0ull : static_cast<uint64_t>(tau) << 32 | 0xffffffffu;
      for (int e = threadIdx.x; e < count; e += kSelectThreads)
        sm.pick[e] = static_cast<uint32_t>(sm.cand[e]);
    } else if (count <= kRankCap) {
      // the place of each among all, a warp to a candidate
      for (int e = warp; e < count; e += kSelectWarps) {
        const uint64_t c = sm.cand[e];
        int before = 0;
        for (int o = lane; o < count; o += 32) before += sm.cand[o] < c;
        before = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0 && before < wanted) sm.pick[before] = static_cast<uint32_t>(c);
        if (lane == 0 && before == wanted - 1) sm.last = c;
      }
      __syncthreads();
      last = sm.last;
    } else {
      int size = 2;
      while (size < count) size <<= 1;
      for (int e = count + threadIdx.x; e < size; e += kSelectThreads) sm.cand[e] = ~0ull;
      sort_candidates(sm, size);
      for (int e = threadIdx.x; e < have; e += kSelectThreads)
        sm.pick[e] = static_cast<uint32_t>(sm.cand[e]);
      last = sm.cand[wanted - 1];
    }
  } else {
    // many equal keys: the row of rank wanted - 1 by (key, index), over all rows
    auto load = [&](int64_t i) {
      const uint32_t key = ordered(keys[i]);
      return (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(i);
    };
    last = n > wanted ? nth(n, wanted - 1, sm, load) : ~0ull;
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < n; i += kSelectThreads) {
      const uint64_t c = load(i);
      if (c <= last && (c >> 32) != kNoKey) {
        const uint32_t at = atomicAdd(&sm.count, 1u);
        if (at < kScoreCap) sm.pick[at] = static_cast<uint32_t>(i);  // at most `wanted`
      }
    }
    __syncthreads();
    have = min(static_cast<int>(sm.count), wanted);
    if ((last >> 32) == kNoKey) last = ~0ull;
  }
  __syncthreads();
  const T* q = x + b * ldx;
  const int dim = static_cast<int>(v.dim);
  int kept = 0;                 // the nearest so far, in order, at the start of sm.final_*
  int64_t next_block = 0;       // of 1024 groups
  uint32_t at_group = 0, in_block = 0;
  for (bool first_round = true;; first_round = false) {
    // distances in 64 bits, a warp to a candidate; its lanes look its rows up at once
    const int mine = have > warp ? (have - warp + kSelectWarps - 1) / kSelectWarps : 0;
    uint32_t my_index = 0;
    int32_t my_row = 0;
    if (lane < mine) {
      my_index = sm.pick[warp + kSelectWarps * lane];
      my_row = static_cast<int32_t>(v.places.at(r.seq, my_index));
    }
    constexpr int kAhead = 4;  // pieces of 256 codes that are asked for at once
    for (int c = 0; c < mine; ++c) {
      const int64_t row = __shfl_sync(0xffffffffu, my_row, c);
      const uint32_t i = __shfl_sync(0xffffffffu, my_index, c);
      const uint8_t* codes = v.codes + row * v.width;
      const uint16_t* scales = v.scales + row * v.groups;
      const uint8_t* zeros = v.zeros ? v.zeros + row * v.groups : nullptr;
      double sum[2] = {0.0, 0.0};
      for (int base = 0; base < dim; base += 256 * kAhead) {
        uint32_t packed[kAhead], bits[kAhead], zero[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int j = base + 256 * u + 8 * lane;
          packed[u] = 0, bits[u] = 0, zero[u] = 8;
          if (j < dim) {
            packed[u] = *reinterpret_cast<const uint32_t*>(codes + (j >> 1));
            bits[u] = scales[j >> v.group_shift];
            if (zeros) zero[u] = zeros[j >> v.group_shift] & 15u;
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int j = base + 256 * u + 8 * lane;
          if (base + 256 * u >= dim) break;
          const double s = v.scale_bf16
                               ? __uint_as_float(bits[u] << 16)
                               : __half2float(__ushort_as_half(static_cast<unsigned short>(bits[u])));
          // 2^52 + code less 2^52 + zero: no conversion, which runs at a quarter
          // of the rate
          const double minus = -__hiloint2double(0x43300000, static_cast<int>(zero[u]));
          // codes behind the last value: at the zero point, so that they count for nothing
          uint32_t word = packed[u];
          if (j + 8 > dim) {
            const uint32_t keep = j < dim ? (1u << (4 * (dim - j))) - 1u : 0u;
            word = (word & keep) | (zero[u] * 0x11111111u & ~keep);
          }
          double part[2] = {0.0, 0.0};
#pragma unroll
          for (int f = 0; f < 8; f += 2) {
            double2 pair;
            if constexpr (!kWide) {
              pair = sm.query[f >> 1][j >> 3];
            } else {
              pair.x = j + f < dim ? static_cast<double>(load_value(q + j + f)) : 0.0;
              pair.y = j + f + 1 < dim ? static_cast<double>(load_value(q + j + f + 1)) : 0.0;
            }
            const double x0 = __hiloint2double(0x43300000, (word >> (4 * f)) & 15) + minus;
            const double x1 = __hiloint2double(0x43300000, (word >> (4 * f + 4)) & 15) + minus;
            if constexpr (kMode == kKeyL2) {
              const double d0 = fma(-s, x0, pair.x), d1 = fma(-s, x1, pair.y);
              sum[0] = fma(d0, d0, sum[0]);
              sum[1] = fma(d1, d1, sum[1]);
            } else {
              part[0] = fma(pair.x, x0, part[0]);
              part[1] = fma(pair.y, x1, part[1]);
            }
          }
          if constexpr (kMode != kKeyL2) sum[u & 1] = fma(-s, part[0] + part[1], sum[u & 1]);
        }
      }
      double all = sum[0] + sum[1];
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
      if (lane == 0 && fabsf(static_cast<float>(all)) < __int_as_float(0x7f800000)) {
        const uint64_t u = static_cast<uint64_t>(__double_as_longlong(all + 0.0));
        const uint64_t key = (u >> 63) ? ~u : u | 0x8000000000000000ull;
        // of a later round only what comes before the k-th so far
        if (kept < k || key < sm.best_key[k - 1] || (key == sm.best_key[k - 1] && i < sm.best_row[k - 1])) {
          const uint32_t at = kept + atomicAdd(&sm.fresh, 1u);
          sm.final_key[at] = key;
          sm.final_row[at] = i;
        }
      }
    }
    if (kMode == kKeyL2 && first_round && warp == kSelectWarps - 1) {  // |q|^2, by the warp with least to score
      double square = 0.0;
#pragma unroll 4
      for (int j = 2 * lane; j < dim; j += 64) {
        double2 pair;
        if constexpr (!kWide) {
          pair = sm.query[(j & 7) >> 1][j >> 3];
        } else {
          pair.x = static_cast<double>(load_value(q + j));
          pair.y = j + 1 < dim ? static_cast<double>(load_value(q + j + 1)) : 0.0;
        }
        square = fma(pair.x, pair.x, fma(pair.y, pair.y, square));
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
      // from below: sums in 64 bits are off by less than 2^-30
      if (lane == 0) sm.squared = __double2float_rd(square * (1.0 - 0x1p-30));
    }
    __syncthreads();
    // the place of each among all, 8 lanes to a row
    const int fresh = static_cast<int>(sm.fresh), all_rows = kept + fresh;
    kept = min(k, all_rows);
    for (int base = 0; fresh > 0 && base < all_rows; base += kSelectThreads / 8) {
      const int e = base + (threadIdx.x >> 3);
      const uint64_t key = e < all_rows ? sm.final_key[e] : 0;
      const uint32_t index = e < all_rows ? sm.final_row[e] : 0;
      int rank = 0;
#pragma unroll 4
      for (int o = threadIdx.x & 7; o < all_rows; o += 8)
        rank += sm.final_key[o] < key || (sm.final_key[o] == key && sm.final_row[o] < index);
#pragma unroll
      for (int d = 4; d >= 1; d >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
      if ((threadIdx.x & 7) == 0 && e < all_rows && rank < kept) {
        const uint64_t u = (key >> 63) ? key & 0x7fffffffffffffffull : ~key;
        const double d = __longlong_as_double(static_cast<long long>(u));
        neighbors[b * k + rank] = index;
        distances[b * k + rank] = static_cast<float>(kMode == kKeyL2 ? d : -d);
        sm.best_key[rank] = key;
        sm.best_row[rank] = index;
      }
    }
    __syncthreads();
    if (first_round && last == ~0ull) break;
    // keys up to which other rows may be as near as the k-th
    uint32_t bound = kNoKey - 1;
    if (kept == k) {
      const uint64_t u = sm.best_key[k - 1];
      const double far = __longlong_as_double(static_cast<long long>((u >> 63) ? u & 0x7fffffffffffffffull : ~u));
      float up = __double2float_ru(far);
      if constexpr (kMode == kKeyL2) up = __fadd_ru(__fmul_ru(up, 1.0f + 0x1p-23f), -sm.squared);
      up += 0.0f;  // no negative zero
      if (up < __int_as_float(0x7f800000)) bound = ordered(up);
    }
    if (first_round && (static_cast<uint64_t>(bound) << 32 | 0xffffffffu) <= last) break;
    if (threadIdx.x < kept) {
      sm.final_key[threadIdx.x] = sm.best_key[threadIdx.x];
      sm.final_row[threadIdx.x] = sm.best_row[threadIdx.x];
    }
    if (threadIdx.x == 0) sm.count = sm.fresh = 0;
    __syncthreads();
    have = 0;
    while (have <= kScoreCap / 2) {
      if (at_group >= in_block) {  // the groups of the next 1024 that have such keys
        if (next_block >= groups) break;
        if (threadIdx.x == 0) sm.groups = 0;
        __syncthreads();
        const int64_t g = next_block + threadIdx.x;
        if (g < groups && minima[g] <= bound) sm.group[atomicAdd(&sm.groups, 1u)] = static_cast<int32_t>(g);
        __syncthreads();
        in_block = sm.groups;
        at_group = 0;
        next_block += kSelectThreads;
        __syncthreads();
        continue;
      }
      const uint32_t e = at_group + warp;
      if (warp < kScoreCap / 2 / kGroupRows && e < in_block) {
        const int64_t i = static_cast<int64_t>(sm.group[e]) * kGroupRows + lane;
        const uint32_t key = i < n ? ordered(keys[i]) : kNoKey;
        if (key <= bound && (static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(i)) > last)
          sm.pick[atomicAdd(&sm.count, 1u)] = static_cast<uint32_t>(i);
      }
      at_group += kScoreCap / 2 / kGroupRows;
      __syncthreads();
      have = static_cast<int>(sm.count);
      __syncthreads();
    }
    if (have == 0) break;
  }
  for (int e = kept + threadIdx.x; e < k; e += kSelectThreads) {
    neighbors[b * k + e] = -1;
    distances[b * k + e] = __int_as_float(kMode == kKeyL2 ? 0x7f800000 : 0xff800000);
  }
}

unsigned row_grid(int64_t rows) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>((rows + kWarps - 1) / kWarps, 148 * 8)));
}

// Shared memory of a block beside the vectors.
int64_t mma_fixed_bytes(int split, int batch, int groups, int mode) {
  return kMmaWarps * (kRing * kStageBytes4 + 2 * 2 * groups * kTileRows4 * 4) +
         (split > 1 ? kMmaWarps * (batch + (mode == kKeyProduct)) * kSumStride * 4 : 0);
}

// Warps that share a tile: the number with the least time of a block, in
// stages.  A tile that is shared costs about a stage more for adding up.
int mma_split(int64_t tiles, int stages, int sms) {
  int best = 1;
  double least = 0;
  for (int split = 1; split <= kMmaWarps && split <= stages; split *= 2) {
    const int64_t at_once = static_cast<int64_t>(sms) * (kMmaWarps / split);
    const double time = static_cast<double>((tiles + at_once - 1) / at_once) *
                        ((stages + split - 1) / split + (split > 1 ? 1.0 : 0.25));
    if (split == 1 || time < least) least = time, best = split;
  }
  return best;
}

template <class T, int kTiles, int kParts, int kGroups, bool kZeros, bool kKeyed>
cudaError_t products(const Q4View& v, const Q4Range& r, const T* x, int batch, int64_t ldx,
                     const Q4Out& o, cudaStream_t stream) {
  constexpr int64_t kMost = 232448 - sizeof(MmaShared) - 64;
  auto kernel = products_kernel<T, kTiles, kParts, kGroups, kZeros, kKeyed>;
  const int sms = store_sm_count();
  MmaPlan p;
  p.tiles = (r.count + kTileRows4 - 1) / kTileRows4;
  p.stages = static_cast<int32_t>((v.dim + kStageCodes - 1) / kStageCodes);
  p.split = mma_split(p.tiles, p.stages, sms);
  const int64_t room = (kMost - mma_fixed_bytes(p.split, batch, kGroups, o.mode)) / (8 * kTiles * 512);
  p.chunk_stages = static_cast<int32_t>(std::min<int64_t>(p.stages, room));
  while (p.split > p.chunk_stages) p.split /= 2;  // every warp has a stage of every full chunk
  p.chunks = (p.stages + p.chunk_stages - 1) / p.chunk_stages;
  const int64_t grid = std::min<int64_t>(p.tiles, sms);
  const int64_t slots = kMmaWarps / p.split;
  p.iterations = static_cast<int32_t>((p.tiles + grid * slots - 1) / (grid * slots));
  const size_t smem = mma_fixed_bytes(p.split, batch, kGroups, o.mode) + p.chunk_stages * (8 * kTiles * 512);
  static std::atomic<uint64_t> allowed{0};
  if (cudaError_t e = allow_smem(kernel, static_cast<int>(kMost), &allowed)) return e;
  store_count_launches(1);
  return launch_after(kernel, static_cast<unsigned>(grid), kMmaThreads, smem, stream, v, r, x,
                      batch, ldx, o, p);
}

template <class T, int kTiles, int kParts, bool kKeyed>
cudaError_t products_as(const Q4View& v, const Q4Range& r, const T* x, int batch, int64_t ldx,
                        const Q4Out& o, cudaStream_t stream) {
  if (v.group == 32)
    return v.zeros ? products<T, kTiles, kParts, 4, true, kKeyed>(v, r, x, batch, ldx, o, stream)
                   : products<T, kTiles, kParts, 4, false, kKeyed>(v, r, x, batch, ldx, o, stream);
  if (v.group == 64)
    return v.zeros ? products<T, kTiles, kParts, 2, true, kKeyed>(v, r, x, batch, ldx, o, stream)
                   : products<T, kTiles, kParts, 2, false, kKeyed>(v, r, x, batch, ldx, o, stream);
  return v.zeros ? products<T, kTiles, kParts, 1, true, kKeyed>(v, r, x, batch, ldx, o, stream)
                 : products<T, kTiles, kParts, 1, false, kKeyed>(v, r, x, batch, ldx, o, stream);
}

template <class T, int kTiles, int kParts>
cudaError_t products_of(const Q4View& v, const Q4Range& r, const T* x, int batch, int64_t ldx,
                        const Q4Out& o, cudaStream_t stream) {
  return o.mode == kStore ? products_as<T, kTiles, kParts, false>(v, r, x, batch, ldx, o, stream)
                          : products_as<T, kTiles, kParts, true>(v, r, x, batch, ldx, o, stream);
}

// Up to kQ4SearchBatch vectors in one pass over the rows.
cudaError_t products_any(const Q4View& v, const Q4Range& r, const void* x, int dtype, int batch,
                         int64_t ldx, const Q4Out& o, cudaStream_t stream) {
  if (dtype == KNN_DTYPE_F32) {
    const float* f = static_cast<const float*>(x);
    if (batch <= 4) return products_of<float, 1, 2>(v, r, f, batch, ldx, o, stream);
    if (batch <= 8) return products_of<float, 2, 2>(v, r, f, batch, ldx, o, stream);
    return products_of<float, 4, 2>(v, r, f, batch, ldx, o, stream);
  }
  if (dtype == KNN_DTYPE_F16) {
    const __half* f = static_cast<const __half*>(x);
    if (batch <= 8) return products_of<__half, 1, 1>(v, r, f, batch, ldx, o, stream);
    return products_of<__half, 2, 1>(v, r, f, batch, ldx, o, stream);
  }
  const __nv_bfloat16* f = static_cast<const __nv_bfloat16*>(x);
  if (batch <= 8) return products_of<__nv_bfloat16, 1, 1>(v, r, f, batch, ldx, o, stream);
  return products_of<__nv_bfloat16, 2, 1>(v, r, f, batch, ldx, o, stream);
}

int64_t group_count(int64_t count) { return (count + kGroupRows - 1) / kGroupRows; }
int64_t minima_ld(int64_t count) { return (group_count(count) + 3) / 4 * 4; }

template <class T, int kMode, bool kWide>
cudaError_t select_as(const Q4View& v, const Q4Range& r, const void* x, int64_t batch, int64_t ldx,
                      const float* keys, int64_t ld, const uint32_t* minima, int k,
                      int64_t* neighbors, float* distances, cudaStream_t stream) {
  auto kernel = select_kernel<T, kMode, kWide>;
  static std::atomic<uint64_t> allowed{0};
  if (cudaError_t e = allow_smem(kernel, sizeof(SelectSmem), &allowed)) return e;
  store_count_launches(1);
  return launch_after(kernel, static_cast<unsigned>(batch), kSelectThreads, sizeof(SelectSmem),
                      stream, v, r, static_cast<const T*>(x), ldx, keys, ld, minima,
                      group_count(r.count), k, neighbors, distances);
}

template <class T>
cudaError_t select(const Q4View& v, const Q4Range& r, const void* x, int64_t batch, int64_t ldx,
                   const float* keys, int64_t ld, const uint32_t* minima, int k, int mode,
                   int64_t* neighbors, float* distances, cudaStream_t stream) {
  const bool wide = v.dim > kQueryHeld;
  auto f = mode == kKeyL2 ? (wide ? select_as<T, kKeyL2, true> : select_as<T, kKeyL2, false>)
                          : (wide ? select_as<T, kKeyProduct, true> : select_as<T, kKeyProduct, false>);
  return f(v, r, x, batch, ldx, keys, ld, minima, k, neighbors, distances, stream);
}

}  // namespace

cudaError_t launch_q4_pack(const Q4View& v, const Q4List& l, const void* rows, int dtype,
                           int64_t ld, cudaStream_t stream) {
  store_count_launches(1);
  const unsigned grid = row_grid(l.total);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(rows);
  const bool vec = ((bits | (ld * (dtype == KNN_DTYPE_F32 ? 4 : 2))) & 15) == 0;
  if (dtype == KNN_DTYPE_F32)
    return launch_after(v.zeros ? pack_kernel<float, true> : pack_kernel<float, false>, grid,
                        kThreads, 0, stream, v, l, static_cast<const float*>(rows), ld, vec);
  if (dtype == KNN_DTYPE_F16)
    return launch_after(v.zeros ? pack_kernel<__half, true> : pack_kernel<__half, false>, grid,
                        kThreads, 0, stream, v, l, static_cast<const __half*>(rows), ld, vec);
  return launch_after(v.zeros ? pack_kernel<__nv_bfloat16, true> : pack_kernel<__nv_bfloat16, false>,
                      grid, kThreads, 0, stream, v, l, static_cast<const __nv_bfloat16*>(rows), ld,
                      vec);
}

cudaError_t launch_q4_read(const Q4View& v, const Q4List& l, float* out, int64_t ld,
                           cudaStream_t stream) {
  store_count_launches(1);
  const bool vec = ((reinterpret_cast<uintptr_t>(out) | (ld * 4)) & 15) == 0;
  return launch_after(v.zeros ? read_kernel<true> : read_kernel<false>, row_grid(l.total), kThreads,
                      0, stream, v, l, out, ld, vec);
}

cudaError_t launch_q4_products(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                               int64_t batch, int64_t ldx, void* out, int out_dtype, int64_t ldo,
                               cudaStream_t stream) {
  const int64_t size = dtype == KNN_DTYPE_F32 ? 4 : 2, out_size = out_dtype == KNN_DTYPE_F32 ? 4 : 2;
  for (int64_t b = 0; b < batch; b += kQ4SearchBatch) {
    const Q4Out o = {static_cast<char*>(out) + b * ldo * out_size, out_dtype, ldo, kStore, nullptr, 0, 0.0f, 0.0f};
    if (cudaError_t e = products_any(
            v, r, static_cast<const char*>(x) + b * ldx * size, dtype,
            static_cast<int>(std::min<int64_t>(kQ4SearchBatch, batch - b)), ldx, o, stream))
      return e;
  }
  return cudaSuccess;
}

int64_t q4_search_bytes(int64_t count, int64_t batch) {
  return std::min<int64_t>(batch, kQ4SearchBatch) * 4 *
         (group_count(count) * kGroupRows + minima_ld(count));
}

cudaError_t launch_q4_search(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                             int64_t batch, int64_t ldx, int k, int metric, int64_t* neighbors,
                             float* distances, void* workspace, cudaStream_t stream) {
  const int mode = metric == KNN_METRIC_L2_EXPANDED ? kKeyL2 : kKeyProduct;
  const int64_t groups = group_count(r.count), ld = groups * kGroupRows;
  float* keys = static_cast<float*>(workspace);
  uint32_t* minima =
      static_cast<uint32_t*>(workspace) + std::min<int64_t>(batch, kQ4SearchBatch) * ld;
  const int64_t size = dtype == KNN_DTYPE_F32 ? 4 : 2;
  for (int64_t b = 0; b < batch; b += kQ4SearchBatch) {
    const int64_t m = std::min<int64_t>(kQ4SearchBatch, batch - b);
    const void* q = static_cast<const char*>(x) + b * ldx * size;
    if (r.count > 0) {
      // see lowest_key; norms are held to (dim / 256 + 16) 2^-24 of them
      const float steps = static_cast<float>(2 * v.group + v.groups + 32) * 1.001f * 0x1p-23f;
      const Q4Out o = {keys, KNN_DTYPE_F32, ld, mode, minima, minima_ld(r.count),
                       steps * (mode == kKeyL2 ? 2.0f : v.zeros ? 15.0f : 8.0f),
                       static_cast<float>(v.dim / 256 + 32) * 0x1p-24f};
      if (cudaError_t e = products_any(v, r, q, dtype, static_cast<int>(m), ldx, o, stream)) return e;
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
