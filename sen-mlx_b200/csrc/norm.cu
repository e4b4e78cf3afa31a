// norm.cu -- RMS norm with the residual's addition, its output in 16 bits, in
// 8 bits with scales (rows8.cuh) or both, and its gradients.
//
//   h = x + residual                              rounded to 16 bits
//   y = h / sqrt(mean(h^2) + eps) * g             g = weight, or 1 + weight
//
//   dn = dy g,  r = 1 / sqrt(mean(h^2) + eps)
//   dx = r (dn - h r^2 mean(dn h)) + dh           (dx is also the residual's)
//   dweight = sum over the rows of dy h r
//
// Sums are fp32 in a fixed order; each output is rounded once.  The norm is
// taken of the rounded h, which is what the layers after it and the backward
// pass have.
//
// Bound by HBM.  A row takes 1 to 16 warps: enough that a lane holds at most
// four pieces of 16 bytes (backward, with its sums for dweight, two), and with
// few rows as many as shorten the one trip to memory and back that such a call
// is.  Rows are read once, each lane its own pieces with cp.async into its own
// places of shared memory, from where it takes them into registers: no barrier
// but the one of the row's sum, and with many rows a row's warps have the next
// rows' loads in flight, more bytes than registers would hold.

#include <cuda_runtime.h>

#include "checks.h"
#include "kernels.h"
#include "linear.cuh"
#include "rows8.cuh"

namespace senmoe {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormIter = 4;    // most pieces of 8 elements a lane holds
constexpr int kGradIter = 2;    // wanted at most in the backward pass: 8 sums for dweight a piece
constexpr int kNormWarps = 16;  // most warps of a row
constexpr int kOddIter = 16, kOddWide = kNormWarps * 32 * kOddIter;  // elements of a lane where rows are on no 16-byte grid
constexpr int kNormWide = kNormIter * kNormWarps * 32 * 8;  // longest row held in registers
// With many rows: rows of a row's warps in shared memory, and blocks of 256
// threads an SM.  32767 rows of 2816 fp16 (369 MB) forward 64.7 us with 2 rows,
// 66.2 with 3, 70.9 with 4; 80.7 us with 2 blocks, 79.2 with 3, 67.8 with 6.
// 32768 rows of 2048 backward (537 MB) 90 us with 2 rows, 104 with 3, 108 with
// 4; 158 us with 1 block, 110 with 3; 104 with 4 pieces a lane, 116 with 1.
constexpr int kDepth = 2, kNormBlocks = 4, kGradBlocks = 2, kOddBlocks = 4;

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t x_stride, residual_stride;
  void *h, *y;
  int64_t h_stride, y_stride;
  uint8_t *codes, *scales;
  int64_t codes_stride, scales_stride;
  int64_t rows;
  int hidden, weight_fp32, bf16;
  float eps, offset;  // offset: 0, or 1 for weights stored around zero
};

struct NormGradArgs {
  const void *dy, *h, *weight, *dh;
  int64_t dy_stride, h_stride, dh_stride;
  void* dx;
  int64_t dx_stride;
  void* dweight;       // the weight's type, or null
  float* partial;      // [blocks, hidden]
  int64_t rows;
  int hidden, weight_fp32, bf16, blocks;
  float eps, offset;
};

// 16 bytes global -> shared, past L1.
__device__ __forceinline__ void cp_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// g of 8 consecutive columns
template <bool BF16> __device__ __forceinline__ void gain8(const void* weight, int fp32, float offset, int c, float (&g)[8]) {
  if (fp32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(weight) + c);
    const float4 a = p[0], b = p[1];
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
    g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
  } else {
    unpack8<BF16>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(weight) + c), g);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] += offset;
}
template <bool BF16> __device__ __forceinline__ float gain(const void* weight, int fp32, float offset, int c) {
  return offset + (fp32 ? static_cast<const float*>(weight)[c] : to_f32<BF16>(static_cast<const uint16_t*>(weight)[c]));
}

// The sums of a row over its WARPS warps, in warp order; `slot` of s is this
// row's and alternates, so that one barrier a row is enough.
template <int WARPS, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float (*s)[N], int row, int warp) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[warp][i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(row + 1), "n"(WARPS * 32) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += s[w][i];
    }
  }
}

template <int WARPS> constexpr int norm_threads() { return WARPS * 32 > kNormThreads ? WARPS * 32 : kNormThreads; }

// Rows on their way: DEPTH slots of a row's STREAMS operands in shared memory,
// a lane's pieces in its own places.
template <int WARPS, int ITER, int DEPTH> struct RowRing {
  static constexpr int kThreads = norm_threads<WARPS>(), kLanes = WARPS * 32, kRows = kThreads / kLanes;
  uint4* mine;  // [DEPTH][streams][ITER][threads]
  int streams;
  __device__ __forceinline__ RowRing(unsigned char* smem, int n) : mine(reinterpret_cast<uint4*>(smem) + threadIdx.x), streams(n) {}
  __device__ __forceinline__ uint4* at(int slot, int stream, int i) const {
    return mine + ((slot * streams + stream) * ITER + i) * kThreads;
  }
  // row: one operand's row, or past the last one null
  __device__ __forceinline__ void fetch(int slot, int stream, const uint16_t* row, int hidden) const {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (threadIdx.x % kLanes + i * kLanes) * 8;
      if (row && c < hidden) cp_async_16(at(slot, stream, i), row + c);
    }
  }
};
constexpr size_t ring_bytes(int threads, int iter, int depth, int streams) { return size_t(threads) * iter * depth * streams * 16; }

template <bool BF16, int WARPS, int ITER, int DEPTH>
__global__ void __launch_bounds__(norm_threads<WARPS>(), 1024 / norm_threads<WARPS>())
    norm_kernel(const __grid_constant__ NormArgs a) {
  using Ring = RowRing<WARPS, ITER, DEPTH>;
  constexpr int kLanes = Ring::kLanes, kRows = Ring::kRows;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ float s_sum[2][kRows][WARPS][1];
  const int sub = threadIdx.x / kLanes, t = threadIdx.x % kLanes;
  const Ring ring(smem_raw, a.residual ? 2 : 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub;
  pdl_wait();
  pdl_launch_dependents();
  const auto fetch = [&](int64_t r, int slot) {
    if (r < a.rows) {
      ring.fetch(slot, 0, static_cast<const uint16_t*>(a.x) + r * a.x_stride, a.hidden);
      if (a.residual) ring.fetch(slot, 1, static_cast<const uint16_t*>(a.residual) + r * a.residual_stride, a.hidden);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(row + d * step, d);
  int slot = 0, turn = 0;
  for (; row < a.rows; row += step, turn ^= 1) {  // a row's warps together
    const int last = slot ? slot - 1 : DEPTH - 1;  // the slot of the row before, which its lanes have read
    fetch(row + (DEPTH - 1) * step, last);
    cp_async_wait<DEPTH - 1>();
    uint4 v[ITER];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (t + i * kLanes) * 8;
      v[i] = c < a.hidden ? *ring.at(slot, 0, i) : make_uint4(0, 0, 0, 0);
      float f[8];
      unpack8<BF16>(v[i], f);
      if (a.residual) {
        float g[8];
        unpack8<BF16>(c < a.hidden ? *ring.at(slot, 1, i) : make_uint4(0, 0, 0, 0), g);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += g[k];
        v[i] = pack8<BF16>(f);
        unpack8<BF16>(v[i], f);
      }
      if (a.h && c < a.hidden) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row * a.h_stride + c) = v[i];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[0] += f[k] * f[k];
    }
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
    row_sums<WARPS>(sum, s_sum[turn][sub], sub, t >> 5);
    const float rstd = rsqrtf(sum[0] / a.hidden + a.eps);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (t + i * kLanes) * 8;
      const bool in = c < a.hidden;
      float f[8], g[8];
      unpack8<BF16>(v[i], f);
      if (in) gain8<BF16>(a.weight, a.weight_fp32, a.offset, c, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = in ? f[k] * rstd * g[k] : 0.0f;
      if (a.y && in) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y) + row * a.y_stride + c) = pack8<BF16>(f);
      if (a.codes) {
        uint32_t byte;
        const uint2 q = pack8_lane(f, byte);
        if (in) {
          *reinterpret_cast<uint2*>(a.codes + row * a.codes_stride + c) = q;
          if ((t & 3) == 0) a.scales[row * a.scales_stride + c / kBlock8] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
}

// Rows on no 16-byte grid of at most 32 * kOddIter elements: a warp a row, an
// element a lane and load.
template <bool BF16> __global__ void __launch_bounds__(kNormThreads) norm_odd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kLanes = 32, kRows = kNormThreads / kLanes;
  const int sub = threadIdx.x / kLanes, t = threadIdx.x % kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub; row < a.rows; row += step) {
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.x_stride;
    const uint16_t* res = static_cast<const uint16_t*>(a.residual) + row * a.residual_stride;
    uint16_t v[kOddIter], r[kOddIter];
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      v[i] = c < a.hidden ? x[c] : uint16_t(0);
      r[i] = a.residual && c < a.hidden ? res[c] : uint16_t(0);
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      if (a.residual) v[i] = from_f32<BF16>(to_f32<BF16>(v[i]) + to_f32<BF16>(r[i]));
      if (a.h && c < a.hidden) (static_cast<uint16_t*>(a.h) + row * a.h_stride)[c] = v[i];
      const float f = to_f32<BF16>(v[i]);
      sum += f * f;
    }
    const float rstd = rsqrtf(warp_sum(sum) / a.hidden + a.eps);
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      if (c >= a.hidden) break;  // (8 bits: hidden is in whole blocks, a warp has one)
      const float f = to_f32<BF16>(v[i]) * rstd * gain<BF16>(a.weight, a.weight_fp32, a.offset, c);
      if (a.y) (static_cast<uint16_t*>(a.y) + row * a.y_stride)[c] = from_f32<BF16>(f);
      if (a.codes) {
        uint32_t byte;
        a.codes[row * a.codes_stride + c] = pack8_warp(f, byte);
        if (t == 0) a.scales[row * a.scales_stride + c / kBlock8] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// Any width, stride and alignment: a block a row, element by element, the row
// read twice (the second time mostly from L1).
template <bool BF16> __global__ void __launch_bounds__(kNormThreads) norm_any_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float s_sum[2][kNormThreads / 32][1];
  pdl_wait();
  pdl_launch_dependents();
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.x_stride;
    const uint16_t* res = static_cast<const uint16_t*>(a.residual) + row * a.residual_stride;
    uint16_t* h = static_cast<uint16_t*>(a.h) + row * a.h_stride;
    const auto value = [&](int c) { return a.residual ? from_f32<BF16>(to_f32<BF16>(x[c]) + to_f32<BF16>(res[c])) : x[c]; };
    float sum[1] = {0.0f};
    for (int c = threadIdx.x; c < a.hidden; c += kNormThreads) {
      const float f = to_f32<BF16>(value(c));
      sum[0] += f * f;
    }
    row_sums<kNormThreads / 32>(sum, s_sum[turn], 0, threadIdx.x >> 5);
    const float rstd = rsqrtf(sum[0] / a.hidden + a.eps);
    for (int c = threadIdx.x; c < a.hidden; c += kNormThreads) {  // (8 bits: hidden is in whole blocks, a warp has one)
      const uint16_t hc = value(c);
      const float v = to_f32<BF16>(hc) * rstd * gain<BF16>(a.weight, a.weight_fp32, a.offset, c);
      if (a.h) h[c] = hc;
      if (a.y) (static_cast<uint16_t*>(a.y) + row * a.y_stride)[c] = from_f32<BF16>(v);
      if (a.codes) {
        uint32_t byte;
        a.codes[row * a.codes_stride + c] = pack8_warp(v, byte);
        if ((threadIdx.x & 31) == 0) a.scales[row * a.scales_stride + c / kBlock8] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// Gradients.  Each row's warps of a block take rows in turn and keep their
// columns' part of dweight in registers; the block's parts meet in shared
// memory at the end and go to its line of `partial`, which norm_join_kernel
// adds in block order.
template <bool BF16, int WARPS, int ITER, int DEPTH>
__global__ void __launch_bounds__(norm_threads<WARPS>(), 512 / norm_threads<WARPS>())
    norm_grad_kernel(const __grid_constant__ NormGradArgs a) {
  using Ring = RowRing<WARPS, ITER, DEPTH>;
  constexpr int kLanes = Ring::kLanes, kRows = Ring::kRows;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ float s_sum[2][kRows][WARPS][2];
  __shared__ __align__(16) float s_part[kRows > 1 ? kLanes * 8 : 1];
  const int sub = threadIdx.x / kLanes, t = threadIdx.x % kLanes;
  const Ring ring(smem_raw, a.dh ? 3 : 2);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub;
  pdl_wait();
  pdl_launch_dependents();
  const auto fetch = [&](int64_t r, int slot) {
    if (r < a.rows) {
      ring.fetch(slot, 0, static_cast<const uint16_t*>(a.dy) + r * a.dy_stride, a.hidden);
      ring.fetch(slot, 1, static_cast<const uint16_t*>(a.h) + r * a.h_stride, a.hidden);
      if (a.dh) ring.fetch(slot, 2, static_cast<const uint16_t*>(a.dh) + r * a.dh_stride, a.hidden);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(row + d * step, d);
  float acc[ITER][8] = {};
  int slot = 0, turn = 0;
  for (; row < a.rows; row += step, turn ^= 1) {
    const int last = slot ? slot - 1 : DEPTH - 1;  // the slot of the row before, which its lanes have read
    fetch(row + (DEPTH - 1) * step, last);
    cp_async_wait<DEPTH - 1>();
    float sum[2] = {0.0f, 0.0f};
    uint4 y[ITER], h[ITER], d[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (t + i * kLanes) * 8;
      if (c < a.hidden) {
        y[i] = *ring.at(slot, 0, i);
        h[i] = *ring.at(slot, 1, i);
        d[i] = a.dh ? *ring.at(slot, 2, i) : make_uint4(0, 0, 0, 0);
        float fy[8], fh[8], g[8];
        unpack8<BF16>(y[i], fy);
        unpack8<BF16>(h[i], fh);
        gain8<BF16>(a.weight, a.weight_fp32, a.offset, c, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          sum[0] += fh[k] * fh[k];
          sum[1] += fy[k] * g[k] * fh[k];
        }
      }
    }
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
    row_sums<WARPS>(sum, s_sum[turn][sub], sub, t >> 5);
    const float r = rsqrtf(sum[0] / a.hidden + a.eps), m = r * r * (sum[1] / a.hidden);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (t + i * kLanes) * 8;
      if (c < a.hidden) {
        float fy[8], fh[8], fd[8], g[8];
        unpack8<BF16>(y[i], fy);
        unpack8<BF16>(h[i], fh);
        unpack8<BF16>(d[i], fd);
        gain8<BF16>(a.weight, a.weight_fp32, a.offset, c, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          acc[i][k] += fy[k] * (fh[k] * r);
          fd[k] += r * (fy[k] * g[k] - fh[k] * m);
        }
        if (a.dx) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dx) + row * a.dx_stride + c) = pack8<BF16>(fd);
      }
    }
  }
  if (!a.partial) return;
  float* part = a.partial + static_cast<int64_t>(blockIdx.x) * a.hidden;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (t + i * kLanes) * 8;
    if constexpr (kRows > 1) {  // row group by row group, one after the other
      for (int s = 0; s < kRows; ++s) {
        __syncthreads();
        if (sub == s) {
          float4* p = reinterpret_cast<float4*>(s_part + t * 8);
          float4 u = make_float4(0, 0, 0, 0), w = u;
          if (s > 0) {
            u = p[0];
            w = p[1];
          }
          p[0] = make_float4(u.x + acc[i][0], u.y + acc[i][1], u.z + acc[i][2], u.w + acc[i][3]);
          p[1] = make_float4(w.x + acc[i][4], w.y + acc[i][5], w.z + acc[i][6], w.w + acc[i][7]);
        }
      }
      if (sub == kRows - 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[i][k] = s_part[t * 8 + k];
      }
    }
    if (sub == kRows - 1 && c < a.hidden) {
      float4* p = reinterpret_cast<float4*>(part + c);
      p[0] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
      p[1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
    }
  }
}

// Rows on no 16-byte grid of at most kOddWide elements: an element a lane and load
// (14251 x 1467 with dh 94 us, with a block a row 266).
template <bool BF16, int WARPS>
__global__ void __launch_bounds__(norm_threads<WARPS>()) norm_grad_odd_kernel(const __grid_constant__ NormGradArgs a) {
  constexpr int kLanes = WARPS * 32, kRows = norm_threads<WARPS>() / kLanes;
  __shared__ float s_sum[2][kRows][WARPS][2];
  __shared__ float s_part[kRows > 1 ? kLanes : 1];
  const int sub = threadIdx.x / kLanes, t = threadIdx.x % kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  pdl_wait();
  pdl_launch_dependents();
  float acc[kOddIter] = {};
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub; row < a.rows; row += step, turn ^= 1) {
    const uint16_t* dy = static_cast<const uint16_t*>(a.dy) + row * a.dy_stride;
    const uint16_t* h = static_cast<const uint16_t*>(a.h) + row * a.h_stride;
    const uint16_t* dh = static_cast<const uint16_t*>(a.dh) + row * a.dh_stride;
    uint16_t y[kOddIter], v[kOddIter], d[kOddIter];
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      y[i] = c < a.hidden ? dy[c] : uint16_t(0);
      v[i] = c < a.hidden ? h[c] : uint16_t(0);
      d[i] = a.dh && c < a.hidden ? dh[c] : uint16_t(0);
    }
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      if (c >= a.hidden) break;
      const float fh = to_f32<BF16>(v[i]);
      sum[0] += fh * fh;
      sum[1] += to_f32<BF16>(y[i]) * gain<BF16>(a.weight, a.weight_fp32, a.offset, c) * fh;
    }
    row_sums<WARPS>(sum, s_sum[turn][sub], sub, t >> 5);
    const float r = rsqrtf(sum[0] / a.hidden + a.eps), m = r * r * (sum[1] / a.hidden);
#pragma unroll
    for (int i = 0; i < kOddIter; ++i) {
      const int c = t + i * kLanes;
      if (c >= a.hidden) break;
      const float fh = to_f32<BF16>(v[i]), fy = to_f32<BF16>(y[i]);
      acc[i] += fy * (fh * r);
      if (a.dx)
        (static_cast<uint16_t*>(a.dx) + row * a.dx_stride)[c] = from_f32<BF16>(
            to_f32<BF16>(d[i]) + r * (fy * gain<BF16>(a.weight, a.weight_fp32, a.offset, c) - fh * m));
    }
  }
  if (!a.partial) return;
  float* part = a.partial + static_cast<int64_t>(blockIdx.x) * a.hidden;
#pragma unroll
  for (int i = 0; i < kOddIter; ++i) {
    const int c = t + i * kLanes;
    if constexpr (kRows > 1) {  // row group by row group, one after the other
      for (int s = 0; s < kRows; ++s) {
        __syncthreads();
        if (sub == s) s_part[t] = acc[i] = (s > 0 ? s_part[t] : 0.0f) + acc[i];
      }
    }
    if (sub == kRows - 1 && c < a.hidden) part[c] = acc[i];
  }
}

// Any width, stride and alignment; a block adds to its line of `partial` row by row.
template <bool BF16>
__global__ void __launch_bounds__(kNormThreads) norm_grad_any_kernel(const __grid_constant__ NormGradArgs a) {
  __shared__ float s_sum[2][kNormThreads / 32][2];
  pdl_wait();
  pdl_launch_dependents();
  float* part = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * a.hidden : nullptr;
  if (part)
    for (int c = threadIdx.x; c < a.hidden; c += kNormThreads) part[c] = 0.0f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const uint16_t* dy = static_cast<const uint16_t*>(a.dy) + row * a.dy_stride;
    const uint16_t* h = static_cast<const uint16_t*>(a.h) + row * a.h_stride;
    const uint16_t* dh = static_cast<const uint16_t*>(a.dh) + row * a.dh_stride;
    float sum[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < a.hidden; c += kNormThreads) {
      const float fh = to_f32<BF16>(h[c]);
      sum[0] += fh * fh;
      sum[1] += to_f32<BF16>(dy[c]) * gain<BF16>(a.weight, a.weight_fp32, a.offset, c) * fh;
    }
    row_sums<kNormThreads / 32>(sum, s_sum[turn], 0, threadIdx.x >> 5);
    const float r = rsqrtf(sum[0] / a.hidden + a.eps), m = r * r * (sum[1] / a.hidden);
    for (int c = threadIdx.x; c < a.hidden; c += kNormThreads) {
      const float fh = to_f32<BF16>(h[c]), fy = to_f32<BF16>(dy[c]);
      if (part) part[c] += fy * (fh * r);
      const float d = (a.dh ? to_f32<BF16>(dh[c]) : 0.0f) +
                      r * (fy * gain<BF16>(a.weight, a.weight_fp32, a.offset, c) - fh * m);
      if (a.dx) (static_cast<uint16_t*>(a.dx) + row * a.dx_stride)[c] = from_f32<BF16>(d);
    }
  }
}

// dweight = the sum of the blocks' lines: 32 columns a block, its warps every
// 32nd line, all their loads in flight together, then the warps in order.
constexpr int kJoinWarps = 32;
template <bool BF16> __global__ void __launch_bounds__(kJoinWarps * 32) norm_join_kernel(const __grid_constant__ NormGradArgs a) {
  __shared__ float s_sum[kJoinWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_launch_dependents();
  float v = 0.0f;
  if (c < a.hidden) {
    const float* p = a.partial + c;
    for (int b = warp; b < a.blocks; b += 16 * kJoinWarps) {
      float t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        t[i] = b + i * kJoinWarps < a.blocks ? p[static_cast<int64_t>(b + i * kJoinWarps) * a.hidden] : 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) v += t[i];
    }
  }
  s_sum[warp][lane] = v;
  __syncthreads();
  v = warp_sum(s_sum[lane][warp]);  // a warp a column, the lines' 32 sums in its lanes
  const int col = blockIdx.x * 32 + warp;
  if (lane == 0 && col < a.hidden) {
    if (a.weight_fp32) static_cast<float*>(a.dweight)[col] = v;
    else static_cast<uint16_t*>(a.dweight)[col] = from_f32<BF16>(v);
  }
}

// ------------------------------------------------------------- host side
bool aligned16(const void* p, int64_t stride, int size = 2) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0;
}

// Warps of a row and pieces of a lane; iter 0: an element a lane and load; warps
// 0: a block a row.
struct NormPlan {
  int warps = 0, iter = 0;
};
// iter: pieces of a lane that are wanted at most; few: warps below which more take a row
NormPlan norm_plan(int64_t rows, int hidden, bool aligned, int iter, int64_t few) {
  NormPlan p;
  if (!aligned || hidden % 8 || hidden > kNormWide) {
    if (hidden <= kOddWide)
      for (p.warps = 1; p.warps * 32 * kOddIter < hidden;) p.warps *= 4;
    return p;
  }
  const int pieces = hidden / 8;
  p.warps = 1;
  while (p.warps < kNormWarps && p.warps * 32 * iter < pieces) p.warps *= 2;
  while (p.warps < kNormWarps && p.warps * 32 < pieces && rows * p.warps < few) p.warps *= 2;
  p.iter = (pieces + p.warps * 32 - 1) / (p.warps * 32);
  return p;
}

#define SENMOE_NORM_ODD(KERNEL, B) (p.warps == 1 ? KERNEL<B, 1> : p.warps == 4 ? KERNEL<B, 4> : KERNEL<B, 16>)
#define SENMOE_NORM_ITER(KERNEL, B, W, D) \
  (p.iter == 1 ? KERNEL<B, W, 1, D> : p.iter == 2 ? KERNEL<B, W, 2, D> : p.iter == 3 ? KERNEL<B, W, 3, D> : KERNEL<B, W, 4, D>)
#define SENMOE_NORM_PICK(KERNEL, B, D)                                                                 \
  (p.warps == 1 ? SENMOE_NORM_ITER(KERNEL, B, 1, D) : p.warps == 2 ? SENMOE_NORM_ITER(KERNEL, B, 2, D) \
   : p.warps == 4 ? SENMOE_NORM_ITER(KERNEL, B, 4, D) : p.warps == 8 ? SENMOE_NORM_ITER(KERNEL, B, 8, D) \
                                                      : SENMOE_NORM_ITER(KERNEL, B, 16, D))

int plan_threads(const NormPlan& p) { return p.warps * 32 > kNormThreads ? p.warps * 32 : kNormThreads; }
int plan_rows(const NormPlan& p) { return p.warps ? plan_threads(p) / (p.warps * 32) : 1; }

template <typename A>
cudaError_t launch_rows(void (*kern)(A), const NormPlan& p, int depth, int streams, int64_t grid, const A& a, cudaStream_t st) {
  const size_t smem = ring_bytes(plan_threads(p), p.iter, depth, streams);
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(plan_threads(p)), smem, st, a);
}

cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  const bool aligned = aligned16(a.x, a.x_stride) && (!a.residual || aligned16(a.residual, a.residual_stride)) &&
                       (!a.h || aligned16(a.h, a.h_stride)) && (!a.y || aligned16(a.y, a.y_stride)) &&
                       aligned16(a.weight, 0) && (!a.codes || aligned16(a.codes, a.codes_stride, 1));
  const int64_t sms = sm_count();
  const NormPlan p = norm_plan(a.rows, a.hidden, aligned, kNormIter, sms * 8);
  // on no grid: a warp a row, or a block (with a residual, a warp a row: 21461 x 223 17.6 us, a
  // block a row 42.9; 4 warps a row: 6191 x 820 50.7, a block a row 22.0)
  if (!p.warps || (!p.iter && p.warps > 1)) {
    const int64_t grid = a.rows < sms * 8 ? a.rows : sms * 8;
    return launch_pdl(a.bf16 ? norm_any_kernel<true> : norm_any_kernel<false>, dim3(static_cast<unsigned>(grid)),
                      dim3(kNormThreads), 0, st, a);
  }
  const int64_t blocks = (a.rows + plan_rows(p) - 1) / plan_rows(p), streams = a.residual ? 2 : 1;
  if (!p.iter)
    return launch_pdl(a.bf16 ? norm_odd_kernel<true> : norm_odd_kernel<false>,
                      dim3(static_cast<unsigned>(blocks < sms * 32 ? blocks : sms * 32)), dim3(plan_threads(p)), 0, st, a);
  // many rows: the blocks that are resident together
  const int64_t fit = 200 * 1024 / static_cast<int64_t>(ring_bytes(plan_threads(p), p.iter, kDepth, streams));
  const int64_t most = kNormBlocks * kNormThreads / plan_threads(p), resident = sms * (fit < most ? fit : most);
  if (blocks > 4 * resident)
    return launch_rows(a.bf16 ? SENMOE_NORM_PICK(norm_kernel, true, kDepth) : SENMOE_NORM_PICK(norm_kernel, false, kDepth), p,
                       kDepth, streams, resident, a, st);
  return launch_rows(a.bf16 ? SENMOE_NORM_PICK(norm_kernel, true, 1) : SENMOE_NORM_PICK(norm_kernel, false, 1), p, 1,
                     streams, blocks, a, st);
}

bool grad_aligned(const NormGradArgs& a) {
  return aligned16(a.dy, a.dy_stride) && aligned16(a.h, a.h_stride) && (!a.dh || aligned16(a.dh, a.dh_stride)) &&
         (!a.dx || aligned16(a.dx, a.dx_stride)) && aligned16(a.weight, 0);
}
// Blocks of a backward pass: as many as are resident together, at most one a
// row group; by the sizes alone, so that the same call adds in the same order.
int grad_blocks(const NormPlan& p, int64_t rows, int sms) {
  const int64_t groups = (rows + plan_rows(p) - 1) / plan_rows(p);
  const int resident = p.warps && !p.iter ? kOddBlocks : kGradBlocks;
  const int64_t most = static_cast<int64_t>(sms) * resident * kNormThreads / (p.warps ? plan_threads(p) : kNormThreads);
  return static_cast<int>(groups < most ? groups : most);
}

cudaError_t launch_norm_grad(NormGradArgs a, const NormPlan& p, cudaStream_t st) {
  if (a.rows > 0) {
    cudaError_t e;
    if (p.warps && !p.iter)
      e = launch_pdl(a.bf16 ? SENMOE_NORM_ODD(norm_grad_odd_kernel, true) : SENMOE_NORM_ODD(norm_grad_odd_kernel, false),
                     dim3(a.blocks), dim3(plan_threads(p)), 0, st, a);
    else if (!p.warps)
      e = launch_pdl(a.bf16 ? norm_grad_any_kernel<true> : norm_grad_any_kernel<false>, dim3(a.blocks),
                     dim3(kNormThreads), 0, st, a);
    else
      e = launch_rows(a.bf16 ? SENMOE_NORM_PICK(norm_grad_kernel, true, kDepth) : SENMOE_NORM_PICK(norm_grad_kernel, false, kDepth), p,
                      kDepth, a.dh ? 3 : 2, a.blocks, a, st);
    if (e != cudaSuccess || !a.dweight) return e;
  }
  if (!a.dweight) return cudaSuccess;
  return launch_pdl(a.bf16 ? norm_join_kernel<true> : norm_join_kernel<false>, dim3((a.hidden + 31) / 32),
                    dim3(kJoinWarps * 32), 0, st, a);
}

constexpr int64_t kMaxNormRows = (int64_t(1) << 31) - 1024;
constexpr int64_t kMaxHidden = int64_t(1) << 24;

int check_rows(const char* call, const char* name, const void* p, int64_t stride, int64_t cols, int64_t rows,
               int align) {
  if (!p) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is NULL", call, name);
  if (reinterpret_cast<uintptr_t>(p) & (align - 1))
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s is not %d-byte aligned", call, name, align);
  if ((stride < cols && rows > 1) || stride < 0 || stride > (int64_t(1) << 40))
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s row stride %lld for rows of %lld elements", call, name,
                  (long long)stride, (long long)cols);
  return SENMOE_OK;
}

int check_norm(const char* call, int32_t dtype, int32_t weight_fp32, int32_t unit_offset, float eps, int64_t rows,
               int64_t hidden, const void* weight) {
  if (dtype != SENMOE_BF16 && dtype != SENMOE_FP16)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are supported)", call, dtype);
  if ((weight_fp32 | unit_offset) & ~1)
    return reject(SENMOE_ERR_BAD_ARG, "%s: weight_fp32=%d unit_offset=%d", call, weight_fp32, unit_offset);
  if (!(eps >= 0.0f) || eps > 1e30f) return reject(SENMOE_ERR_BAD_ARG, "%s: eps=%g", call, eps);
  if (rows < 0 || rows > kMaxNormRows) return reject(SENMOE_ERR_BAD_ARG, "%s: rows=%lld", call, (long long)rows);
  if (hidden < 1 || hidden > kMaxHidden) return reject(SENMOE_ERR_BAD_ARG, "%s: hidden=%lld", call, (long long)hidden);
  if (reinterpret_cast<uintptr_t>(weight) & (weight_fp32 ? 3 : 1))
    return reject(SENMOE_ERR_BAD_ARG, "%s: weight is not aligned to its type", call);
  return SENMOE_OK;
}

// The arguments' checks, the kernels' form and the blocks of a backward call.
int plan_grad(const char* call, const SenMoeNormGrad* g, NormGradArgs* a, NormPlan* p) {
  if (!g) return reject(SENMOE_ERR_BAD_ARG, "%s: grad is NULL", call);
  const int rc = check_norm(call, g->dtype, g->weight_fp32, g->unit_offset, g->eps, g->rows, g->hidden, g->weight);
  if (rc) return rc;
  a->dy = g->dy;
  a->dy_stride = g->dy_stride;
  a->h = g->h;
  a->h_stride = g->h_stride;
  a->weight = g->weight;
  a->dh = g->dh;
  a->dh_stride = g->dh_stride;
  a->dx = g->dx;
  a->dx_stride = g->dx_stride;
  a->dweight = g->dweight;
  a->rows = g->rows;
  a->hidden = static_cast<int>(g->hidden);
  a->weight_fp32 = g->weight_fp32;
  a->bf16 = g->dtype == SENMOE_BF16;
  a->eps = g->eps;
  a->offset = g->unit_offset ? 1.0f : 0.0f;
  const int sms = sm_count();
  *p = norm_plan(g->rows, a->hidden, grad_aligned(*a), kGradIter, sms * 8);
  a->blocks = grad_blocks(*p, g->rows, sms);
  return SENMOE_OK;
}

}  // namespace
}  // namespace senmoe

using namespace senmoe;

extern "C" {

int senmoe_rms_norm(const SenMoeNorm* n, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "rms_norm";
  if (!n) return reject(SENMOE_ERR_BAD_ARG, "%s: norm is NULL", call);
  int rc = check_norm(call, n->dtype, n->weight_fp32, n->unit_offset, n->eps, n->rows, n->hidden, n->weight);
  if (rc) return rc;
  if (n->codes && n->hidden % kBlock8)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: hidden=%lld in 8 bits (a multiple of %d)", call, (long long)n->hidden, kBlock8);
  if (n->rows == 0) return SENMOE_OK;
  if (!n->y && !n->codes && !(n->residual && n->h)) return reject(SENMOE_ERR_BAD_ARG, "%s: no output", call);
  if (!n->weight) return reject(SENMOE_ERR_BAD_ARG, "%s: weight is NULL", call);
  if ((rc = check_rows(call, "x", n->x, n->x_stride, n->hidden, n->rows, 2))) return rc;
  if (n->residual && (rc = check_rows(call, "residual", n->residual, n->residual_stride, n->hidden, n->rows, 2))) return rc;
  if (n->h && (rc = check_rows(call, "h", n->h, n->h_stride, n->hidden, n->rows, 2))) return rc;
  if (n->y && (rc = check_rows(call, "y", n->y, n->y_stride, n->hidden, n->rows, 2))) return rc;
  if (n->codes) {
    if ((rc = check_rows(call, "codes", n->codes, n->codes_stride, n->hidden, n->rows, 1))) return rc;
    if ((rc = check_rows(call, "scales", n->scales, n->scales_stride, n->hidden / kBlock8, n->rows, 1))) return rc;
  }
  NormArgs a{};
  a.x = n->x;
  a.x_stride = n->x_stride;
  a.residual = n->residual;
  a.residual_stride = n->residual_stride;
  a.weight = n->weight;
  a.h = n->h;
  a.h_stride = n->h_stride;
  a.y = n->y;
  a.y_stride = n->y_stride;
  a.codes = static_cast<uint8_t*>(n->codes);
  a.codes_stride = n->codes_stride;
  a.scales = static_cast<uint8_t*>(n->scales);
  a.scales_stride = n->scales_stride;
  a.rows = n->rows;
  a.hidden = static_cast<int>(n->hidden);
  a.weight_fp32 = n->weight_fp32;
  a.bf16 = n->dtype == SENMOE_BF16;
  a.eps = n->eps;
  a.offset = n->unit_offset ? 1.0f : 0.0f;
  return cuda_status(call, launch_norm(a, stream));
}

int64_t senmoe_rms_norm_backward_workspace(const SenMoeNormGrad* g) {
  clear_failure();
  NormGradArgs a{};
  NormPlan p;
  const int rc = plan_grad("rms_norm_backward", g, &a, &p);
  return rc ? -int64_t(rc) : g->dweight ? int64_t(4) * a.blocks * a.hidden : 0;
}

int senmoe_rms_norm_backward(const SenMoeNormGrad* g, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "rms_norm_backward";
  NormGradArgs a{};
  NormPlan p;
  int rc = plan_grad(call, g, &a, &p);
  if (rc) return rc;
  if (g->rows > 0) {
    if (!g->weight) return reject(SENMOE_ERR_BAD_ARG, "%s: weight is NULL", call);
    if ((rc = check_rows(call, "dy", g->dy, g->dy_stride, g->hidden, g->rows, 2))) return rc;
    if ((rc = check_rows(call, "h", g->h, g->h_stride, g->hidden, g->rows, 2))) return rc;
    if (g->dh && (rc = check_rows(call, "dh", g->dh, g->dh_stride, g->hidden, g->rows, 2))) return rc;
    if (g->dx && (rc = check_rows(call, "dx", g->dx, g->dx_stride, g->hidden, g->rows, 2))) return rc;
  }
  if (reinterpret_cast<uintptr_t>(g->dweight) & (g->weight_fp32 ? 3 : 1))
    return reject(SENMOE_ERR_BAD_ARG, "%s: dweight is not aligned to its type", call);
  if (!g->dx && !g->dweight) return SENMOE_OK;
  if (g->dweight) {
    const int64_t need = int64_t(4) * a.blocks * a.hidden;
    if (need > 0 && (!g->workspace || g->workspace_bytes < need))
      return reject(SENMOE_ERR_BAD_ARG, "%s: workspace of %lld bytes, %lld needed", call,
                    g->workspace ? (long long)g->workspace_bytes : 0ll, (long long)need);
    if (reinterpret_cast<uintptr_t>(g->workspace) & 15)
      return reject(SENMOE_ERR_BAD_ARG, "%s: workspace is not 16-byte aligned", call);
    a.partial = static_cast<float*>(g->workspace);
  }
  return cuda_status(call, launch_norm_grad(a, p, stream));
}

}  // extern "C"
