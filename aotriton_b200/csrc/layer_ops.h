// Host-side declarations of the operators that stand around attention in a layer (layer_ops.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include "common.cuh"

namespace ab200 {

constexpr int kMaxBorders = 127;      // buckets of one direction, less one

struct RelativeBias {
  View4 bias;                    // forward: (1, H, Sq, Sk), written; backward: (B, H, Sq, Sk), the gradient
  void* table;                   // (buckets, heads): the table, or its gradient
  int64_t table_stride[2];
  int32_t heads, sq, sk, batch, offset;
  int32_t per_direction, both;   // buckets of one direction; both: keys after the query's position take the second half
  int32_t borders[kMaxBorders];  // borders[k - 1]: the smallest distance whose bucket is k or more
  float* partial;                // backward: bucket sums of each CTA
  int32_t strips, bands, chunks, chunk_rows;
  int32_t unit, vec;             // the bias' elements are next to each other in its rows; and those start on 16-byte boundaries
};

struct Dropout {
  const void *x, *residual;
  void* out;
  int64_t rows, cols, sx, sr, so;      // strides between rows, in elements
  const uint64_t *seed_ptr, *offset_ptr;
  uint64_t seed, offset;               // added to what the pointers (may be null) say
  float scale;
  int32_t threshold, on;
  uint32_t keys[20];                   // of calls without pointers (dropout_keys)
};

cudaError_t launch_relative_bias(int dtype, int table_dtype, const RelativeBias& a, cudaStream_t st);
// How the backward is cut (strips, bands, chunks, chunk_rows), for `sms` SMs; returns the floats of workspace it needs.
int64_t plan_relative_bias_backward(int dtype, RelativeBias& a, int sms);
cudaError_t launch_relative_bias_backward(int dtype, int table_dtype, const RelativeBias& a, cudaStream_t st);
cudaError_t launch_dropout(int dtype, const Dropout& a, cudaStream_t st);

}  // namespace ab200
