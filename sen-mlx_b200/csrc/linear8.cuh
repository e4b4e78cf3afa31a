// linear8.cuh -- what the kernels of the products over 8-bit rows share.
#pragma once

#include <type_traits>

#include "linear.cuh"
#include "rows8.cuh"

namespace senmoe {

struct Quantize8Args {
  const void* x;
  int64_t x_stride;
  const void* preact;
  int64_t preact_stride;
  int64_t rows;
  int n, act, bf16;
  uint8_t* codes;
  int64_t codes_stride;
  uint8_t* scales;
  int64_t scales_stride;
};
cudaError_t launch_quantize8(const Quantize8Args& a, cudaStream_t st);

// One product, z = x W^T (+ bias), y = act(z) (+ residual); all row-major.
// offsets null: one group holding every row.
struct Linear8Args {
  const uint8_t *x, *x_scales, *w, *w_scales;
  int64_t x_stride, x_scales_stride;
  int64_t w_stride, w_group_stride, w_scales_stride, w_scales_group_stride;
  const int32_t* offsets;      // [groups + 1]
  int groups;
  int64_t rows;
  int n, k;                    // W's rows (gate and up: both) and columns
  int act, bf16;               // bf16: of bias, residual, y and preact; 0: fp16
  const void *bias, *residual;
  int64_t residual_stride;
  void* y;                     // 16 bits, or null: 8 bits
  int64_t y_stride;
  uint8_t *codes, *scales;
  int64_t codes_stride, scales_stride;
  void* preact;                // or null
  int64_t preact_stride;
};
// [begin, end) in k blocks (stages of linear8_tc.cu) of CTA `rank` of a K split
// over `split`; empty for some where there are fewer blocks than CTAs.
struct KRange {
  int begin, end;
};
__host__ __device__ inline KRange k_share(int blocks, int rank, int split) {
  return {static_cast<int>(static_cast<int64_t>(blocks) * rank / split),
          static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / split)};
}
// The units of two blocks in which their scales come; none without blocks.
__host__ __device__ inline KRange scale_units(int kb0, int kb1) {
  return {kb0 / 2, kb1 > kb0 ? (kb1 + 1) / 2 : kb0 / 2};
}
// Few rows (linear8_small.cu), in chunks of 8, 16, 32 or 64 by the mean group.
inline int linear8_small_chunk(const Linear8Args& a) {
  const int64_t mean = a.rows / a.groups;
  return mean <= 8 ? 8 : mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
}
bool linear8_small_supported(const Linear8Args& a);
cudaError_t launch_linear8_small(const Linear8Args& a, cudaStream_t st);
// tcgen05 (linear8_tc.cu); form: a LinearForm, kFormAuto by estimated time.
cudaError_t launch_linear8_tc(const Linear8Args& a, int form, cudaStream_t st);
// Where these kernels record their device error, on the current device (for linear_device_error).
cudaError_t linear8_error_word(int** word);

}  // namespace senmoe
