// knn_store.h -- declarations of the row store: pages of rows and rows in
// 4 bits (knn_pages.cu, knn_q4.cu, knn_store_capi.cu).
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#include "cuvs_b200.h"

namespace knn {

// Error text and kernel count of the C ABI (knn_capi.cu).
int store_fail(int status, const char* text);
void store_count_launches(int n);

// knn_pages::status: the first error of any call (sticky until the caller
// clears it), and whether the last call that changes the store was applied.
constexpr int kStatusError = 0;
constexpr int kStatusApplied = 1;

// A position of a sequence, as a row number in the pools, or -1 where the
// table holds no page for it.
struct Places {
  const int32_t* table;  // nullptr: rows lie one after another
  int64_t columns;
  int64_t pages;
  int32_t page_rows;
  // Positions are below 2^31, as a store's rows are: 32-bit division.
  __device__ __forceinline__ int64_t at(int64_t seq, int64_t position) const {
    if (!table) return position;
    const uint32_t p = static_cast<uint32_t>(position);
    const uint32_t column = p / static_cast<uint32_t>(page_rows);
    if (column >= columns) return -1;
    const int32_t page = table[seq * columns + column];
    if (page < 0 || page >= pages) return -1;
    return static_cast<int64_t>(page) * page_rows + (p - column * page_rows);
  }
};

// Launch of a kernel that may start while the one before it in the stream
// ends (every kernel of the store waits, griddepcontrol.wait, before it
// reads or writes memory).
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem,
                         cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Leave for a kernel to use `bytes` of dynamic shared memory on the current
// device, asked for once a device (`allowed` has a bit for each of the first 64).
template <class K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>* allowed) {
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device)) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (allowed->load(std::memory_order_relaxed) & bit) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) allowed->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Multiprocessors of the current device.
inline int store_sm_count() {
  static std::atomic<int> counts[64];
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 148;
  if (device < 64 && (sms = counts[device].load(std::memory_order_relaxed)) > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms < 1)
    return 148;
  if (device < 64) counts[device].store(sms, std::memory_order_relaxed);
  return sms;
}

__device__ __forceinline__ void wait_for_stream() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// knn_pages.cu: launchers of the page operators.  Each enqueues all of its
// kernels on `stream` and returns the first launch error.
cudaError_t launch_pages_grow(const knn_pages& p, const int32_t* seqs, const int32_t* counts,
                              int64_t n, int64_t total, cudaStream_t stream);
cudaError_t launch_pages_free(const knn_pages& p, const int32_t* seqs, int64_t n,
                              cudaStream_t stream);
cudaError_t launch_pages_copy(const knn_pages& p, const int32_t* sources, const int32_t* targets,
                              int64_t n, cudaStream_t stream);
cudaError_t launch_pages_fork(const knn_pages& p, const int32_t* parents, const int32_t* children,
                              int64_t n, cudaStream_t stream);
int64_t pages_compact_words(const knn_pages& p, int64_t n, int64_t keep_columns);
cudaError_t launch_pages_compact(const knn_pages& p, const int32_t* sources,
                                 const int32_t* targets, int64_t n, const uint8_t* keep,
                                 int64_t keep_columns, int64_t keep_stride, int32_t* workspace,
                                 cudaStream_t stream);

}  // namespace knn
