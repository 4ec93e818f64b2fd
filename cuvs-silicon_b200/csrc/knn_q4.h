// knn_q4.h -- rows in 4 bits: what the kernels of knn_q4.cu take.
#pragma once

#include "knn_store.h"

namespace knn {

// Rows in 4 bits, by their row number in the pools (dense rows: 0 .. n - 1).
struct Q4View {
  const uint8_t* codes;    // [rows][width], low nibble first
  const uint16_t* scales;  // [rows][groups], fp16 or bf16
  const uint8_t* zeros;    // [rows][groups], or nullptr: 8 throughout
  const float* norms;      // [rows], |row|^2, or nullptr
  int64_t dim;
  int32_t group, groups;
  int32_t group_shift;  // group = 1 << group_shift
  int32_t width;  // bytes of a row's codes, 16 * ceil(dim / 32)
  int32_t scale_bf16;
  Places places;
};

// Which rows a product or search runs over: positions 0 .. count - 1 of
// sequence seq, no further than its length where `length` is given.
struct Q4Range {
  int64_t seq;
  int64_t count;
  const int32_t* length;  // device word, or nullptr
};

// The rows of a list of sequences, one after another: the last counts[i] rows
// of sequence seqs[i].  seqs == nullptr: dense rows first .. first + total - 1.
struct Q4List {
  const int32_t* seqs;
  const int32_t* counts;
  int32_t n;
  int64_t total;
  int64_t first;
  const int32_t* rows;  // the store's lengths
  int64_t sequences;
  int32_t* status;
};

cudaError_t launch_q4_pack(const Q4View& v, const Q4List& list, const void* rows, int dtype,
                           int64_t ld, cudaStream_t stream);
cudaError_t launch_q4_read(const Q4View& v, const Q4List& list, float* out, int64_t ld,
                           cudaStream_t stream);
cudaError_t launch_q4_products(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                               int64_t batch, int64_t ldx, void* out, int out_dtype, int64_t ldo,
                               cudaStream_t stream);
// Queries that one pass of a search takes, and its workspace in bytes.
constexpr int kQ4SearchBatch = 16;
int64_t q4_search_bytes(int64_t count, int64_t batch);
cudaError_t launch_q4_search(const Q4View& v, const Q4Range& r, const void* x, int dtype,
                             int64_t batch, int64_t ldx, int k, int metric, int64_t* neighbors,
                             float* distances, void* workspace, cudaStream_t stream);

}  // namespace knn
