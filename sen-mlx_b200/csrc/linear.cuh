// linear.cuh -- what the 16-bit linear product kernels share: their
// arguments, the epilogue's activations with their derivatives, and the table
// of row groups.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace senmoe {

// Values of SenMoeEpilogue (include/senmoe.h).
enum LinearAct : int {
  kActNone = 0,
  kActRelu = 1,
  kActSilu = 2,
  kActGelu = 3,      // z * Phi(z)
  kActGeluTanh = 4,  // its tanh form
  kActSwiglu = 5,    // silu(gate) * up
  kActGeglu = 6,     // tanh-form gelu(gate) * up
};
inline __host__ __device__ bool act_gated(int act) { return act >= kActSwiglu; }

// The three products of a linear map, each C[i, j] = sum_k A(i, k) B(j, k):
//   kProdForward  i = row of x,   j = row of W,    k = input feature
//   kProdInput    i = row of dz,  j = input feature, k = row of W     (dx)
//   kProdWeight   i = row of W,   j = input feature, k = row of the group (dW)
enum LinearProduct : int { kProdForward = 0, kProdInput = 1, kProdWeight = 2 };

constexpr int kMaxGroups = 1024;

// One product.  a is x (forward) or dz; b is W (forward, dx) or x (dW); all
// row-major with the given element strides between rows.  offsets null: one
// group holding every row.
struct LinearArgs {
  const void* a;
  const void* b;
  int64_t a_stride, b_stride, b_group_stride;  // b_group_stride: W's, forward and dx
  const int32_t* offsets;                      // [groups + 1]
  int groups;
  int64_t rows;                                // of x and dz
  int n, k;                                    // W's rows (gate and up: both) and columns
  int act;                                     // forward only
  const void* bias;                            // [groups, n] or null
  const void* residual;
  int64_t residual_stride;
  void* out;                                   // y, dx or dW
  int64_t out_stride, out_group_stride;        // out_group_stride: dW's
  void* preact;                                // forward: z before the activation, or null
  int64_t preact_stride;
  int bf16;                                    // 1: bf16, 0: fp16
  const unsigned* dz_max;                      // dx, dW: the groups' scales of an fp16 dz (dz_exponent), or null
};

// fp16 holds 2^-14 to 65504 in full precision, less than |dy u act'(z)| may
// span.  So an fp16 dz is stored times 2^-x, with x from its group's largest
// finite |dz| (as the bits of a float), and the gradients' epilogues multiply
// by 2^x: 0 where that is between 2^-6 and 65504, so that the terms that
// decide a sum are in range as they are, otherwise the x that takes it into
// [2^14, 2^15).  Elements under 2^-39 of a group's largest are lost.
__host__ __device__ inline int dz_exponent(unsigned max_bits) {
  const int x = static_cast<int>(max_bits >> 23) - 127;
  if (max_bits == 0 || (x >= -6 && max_bits <= 0x477fe000u)) return 0;
  return (x > -100 ? x : -100) - 14;
}
__device__ __forceinline__ float power_of_two(int x) { return __int_as_float((x + 127) << 23); }

// 16-bit values by their bit patterns.
template <bool BF16> __device__ __forceinline__ float to_f32(uint16_t v) {
  if constexpr (BF16) return bf16_bits_to_f32(v);
  else return __half2float(__ushort_as_half(v));
}
template <bool BF16> __device__ __forceinline__ uint16_t from_f32(float v) {
  if constexpr (BF16) return f32_to_bf16_bits(v);
  else return __half_as_ushort(__float2half_rn(v));
}
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

template <bool BF16> __device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = to_f32<BF16>(static_cast<uint16_t>(w[i]));
    f[2 * i + 1] = to_f32<BF16>(static_cast<uint16_t>(w[i] >> 16));
  }
}
template <bool BF16> __device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
}

// Activations in fp32, rounded once, to 16 bits or (FINE) to 8.  The intrinsics'
// error (a few units in the last place, __expf one more for every unit of its
// argument: below 2^-15 of the value down to z = -12) is far below a 16-bit unit.
// In 8 bits it decides which side of a border a value next to one falls on: of
// silu's and gelu's tanh form, and of their slopes, as many fall on the other side
// as with exact exponentials and divisions (2, 3 and 9 against 3, 5 and 10 of 1.4,
// 12.6 and 8.4 million slopes); gelu's Phi is fitted closer there.  Where its
// exponential nears overflow (z < -87, gelu's tanh form z < -10), a value under
// 1e-35 comes out as 0.
// gelu's tanh form 0.5 z (1 + tanh(a)) equals z / (1 + exp(-2a)), which has
// one exponential and keeps its relative precision in the lower tail.
__device__ __forceinline__ float logistic(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
__device__ __forceinline__ float gelu_arg2(float z) {  // 2a, a = sqrt(2/pi) (z + 0.044715 z^3)
  return 1.5957691216057308f * (z + 0.044715f * z * z * z);
}
// Phi(z), e = exp(-z^2 / 2): 1/2 erfc(a) = e t P(t) for a = |z| / sqrt 2,
// t = 1 / (1 + 0.365 |z|), the form of Hastings' approximations (Abramowitz and
// Stegun, 7.1.26), which bound the absolute error only.  P is fitted for the
// least maximum of the *relative* error over |z| <= 15 (linear program over
// 4000 points), 1.3e-6 in fp32, so that the lower tail is as exact as the rest.
// FINE: two degrees more, 1e-8, in fp32 4e-7 and 7e-8 on average (gelu's slopes in
// 8 bits: 240 of 8.4 million were on the other side of a border, now none; 8192 x
// 2048 -> 8192 gelu to 8 bits 155.4 -> 158.0 us, the slopes' kernel the same).
template <bool FINE> __device__ __forceinline__ float normal_cdf(float z, float e) {
  if constexpr (FINE) {
    const float t = __fdividef(1.0f, 1.0f + 0.35f * fabsf(z));
    const float p = 0.139619693f + t * (0.139894828f + t * (0.119570084f + t * (0.106644519f + t * (-0.0260373186f + t * (0.163785264f +
                    t * (-0.260060489f + t * (0.146217644f + t * -0.0296342336f)))))));
    const float q = t * p * e;
    return z < 0.0f ? q : 1.0f - q;
  }
  const float t = __fdividef(1.0f, 1.0f + 0.365f * fabsf(z));
  const float p = 0.14567815f + t * (0.14424385f + t * (0.13795274f + t * (0.03523802f +
                  t * (0.16542687f + t * (-0.17671363f + t * 0.04817444f)))));
  const float q = t * p * e;
  return z < 0.0f ? q : 1.0f - q;
}
template <bool FINE = false> __device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
    case kActSilu: case kActSwiglu: return __fdividef(z, 1.0f + __expf(-z));
    case kActGelu: return z * normal_cdf<FINE>(z, __expf(-0.5f * z * z));
    case kActGeluTanh: case kActGeglu: return __fdividef(z, 1.0f + __expf(-gelu_arg2(z)));
    default: return z;
  }
}
// act'(z), and act(z) in `value` (the two share their exponential).
template <bool FINE = false> __device__ __forceinline__ float act_both(int act, float z, float& value) {
  switch (act) {
    case kActRelu:
      value = z > 0.0f ? z : 0.0f;
      return z > 0.0f ? 1.0f : 0.0f;
    case kActSilu: case kActSwiglu: {
      const float s = logistic(z);
      value = z * s;
      return s * (1.0f + z * (1.0f - s));
    }
    case kActGelu: {  // Phi(z) + z phi(z)
      const float e = __expf(-0.5f * z * z), c = normal_cdf<FINE>(z, e);
      value = z * c;
      return c + z * 0.3989422804014327f * e;
    }
    case kActGeluTanh: case kActGeglu: {  // s = (1 + tanh a) / 2: s + 2 z s (1 - s) a'
      const float s = logistic(gelu_arg2(z));
      value = z * s;
      return s + z * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * z * z);
    }
    default:
      value = z;
      return 1.0f;
  }
}

// Row range of every group, made monotone and clamped to [0, rows] (whatever
// offsets holds, no access leaves the operands), and the prefix sums of the
// groups' chunks of `chunk` rows.  s_off and s_pre: groups + 1 ints of shared
// memory each; s_tot: 64 ints.  Every thread of the block calls it; it ends
// with __syncthreads.
__device__ __forceinline__ void group_table(const int32_t* __restrict__ offsets, int groups, int64_t rows, int chunk,
                                            int* s_off, int* s_pre, int* s_tot) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = (blockDim.x + 31) >> 5;
  if (!offsets) {
    if (tid == 0) {
      s_off[0] = s_pre[0] = 0;
      s_off[1] = static_cast<int>(rows);
      s_pre[1] = static_cast<int>((rows + chunk - 1) / chunk);
    }
    __syncthreads();
    return;
  }
  // one pass for the running maximum of the offsets, one for the chunk sums
  const int n = groups + 1, per = (n + blockDim.x - 1) / blockDim.x;
  const int first = min(tid * per, n), last = min(first + per, n);
  const int cap = static_cast<int>(rows);
  int m = 0;
  for (int i = first; i < last; ++i) {
    m = max(m, min(max(offsets[i], 0), cap));
    s_off[i] = m;
  }
  int v = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  if (lane == 31) s_tot[warp] = v;
  int before = __shfl_up_sync(0xffffffffu, v, 1);
  if (lane == 0) before = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = max(before, s_tot[w]);
  for (int i = first; i < last; ++i) s_off[i] = max(s_off[i], before);
  __syncthreads();
  int sum = 0;
  for (int i = first; i < last; ++i) {
    s_pre[i] = sum;  // chunks of this thread's groups before i
    if (i < groups) sum += (s_off[i + 1] - s_off[i] + chunk - 1) / chunk;
  }
  v = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_tot[32 + warp] = v;
  int base = v - sum;
  __syncthreads();
  for (int w = 0; w < warp && w < nw; ++w) base += s_tot[32 + w];
  for (int i = first; i < last; ++i) s_pre[i] += base;
  __syncthreads();
}

// The group whose chunks include chunk c: the last e with s_pre[e] <= c and chunks of its own.
__device__ __forceinline__ int group_of(const int* s_pre, int groups, int c) {
  int lo = 0, hi = groups;  // s_pre[lo] <= c < s_pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_pre[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Rows that no group holds (before the first offset, after the last) are
// zero.  All threads of block `block` of `blocks`.
__device__ __forceinline__ void zero_uncovered(const int* s_off, int groups, int64_t rows, uint16_t* out,
                                               int64_t stride, int cols, int block, int blocks) {
  const int64_t head = s_off[0], tail = s_off[groups];
  const int64_t n = head + (rows - tail);
  for (int64_t i = block; i < n; i += blocks) {
    uint16_t* row = out + (i < head ? i : tail + (i - head)) * stride;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) row[c] = 0;
  }
}

// ------------------------------------------------------------ launchers
// Any strides and alignments (linear_any.cu).
cudaError_t launch_linear_any(const LinearArgs& a, LinearProduct p, cudaStream_t st);
// Few rows, forward (linear_small.cu): 16-byte aligned rows of a multiple of 8 elements.
bool linear_small_supported(const LinearArgs& a);
cudaError_t launch_linear_small(const LinearArgs& a, cudaStream_t st);
// tcgen05 (linear_tc.cu): operands that TMA can read, see linear_tc_supported.
bool linear_tc_supported(const LinearArgs& a, LinearProduct p);
// form: of the tiles, kFormAuto by estimated time.  bias (dW only, or null):
// also the bias gradient, from its parts, or without parts as the column sums
// of dz where this form can take them; *summed says whether it does.
struct BiasJoin;
enum LinearForm : int { kFormAuto = 0, kFormOne = 1, kFormPair = 2, kFormSplit = 3 };
cudaError_t launch_linear_tc(const LinearArgs& a, LinearProduct p, int form, const BiasJoin* bias, bool* summed,
                             cudaStream_t st);
// Waits for `st`, returns and clears the device error that the tcgen05
// kernels recorded on the current device (DeviceError), here or at `also`.
cudaError_t linear_device_error(cudaStream_t st, int* error, int* also);
// A kernel whose only wait runs out (about 2 s) and is recorded.
cudaError_t selftest_linear_wait(cudaStream_t st);

// dz = dy * act'(z) in 16 bits, and its column sums over each group (the bias
// gradient) from the fp32 values; see linear_grad.cu.
struct LinearGradArgs {
  const void* dy;
  int64_t dy_stride;
  const void* preact;       // not read for kActNone
  int64_t preact_stride;
  const int32_t* offsets;
  int groups;
  int64_t rows;
  int n;                    // columns of dz (gate and up: both)
  int act;                  // kActNone: dz is dy and is not stored
  void* dz;                 // [rows, dz_stride]
  int64_t dz_stride;
  void* dbias;              // [groups, n] or null
  float* partial;           // [dz_slots, n]: the sums' parts; null where there is one run
  int run;                  // dz_run's
  unsigned* dz_max;         // fp16: [groups], the largest finite |dz| (see dz_exponent); null: dz is not scaled
  int bf16;
};
// Rows of a run, and the slots that the sums of all runs and groups take (0:
// the one run of a dense product goes straight to dbias).
constexpr int dz_run_rows(bool gated) { return gated ? 2 : 4; }  // of one warp
int dz_run(int64_t rows, bool grouped, int act);
int64_t dz_slots(int64_t rows, int groups, bool grouped, int run);
cudaError_t launch_dz(const LinearGradArgs& a, cudaStream_t st);

// dbias[e] = the sum of group e's slots.
struct BiasJoin {
  const float* partial;     // [dz_slots, n]
  const int32_t* offsets;
  int groups, run, n;
  int64_t rows;
  void* dbias;              // [groups, n]
};
// A warp takes 32 columns of a group or, where groups have many runs, 8
// columns whose four lanes take every fourth slot.
__host__ __device__ inline int bias_join_cols(const BiasJoin& j) { return j.rows / j.groups > 16 * j.run ? 8 : 32; }
__host__ __device__ inline int64_t bias_join_items(const BiasJoin& j) {
  const int w = bias_join_cols(j);
  return static_cast<int64_t>(j.groups) * ((j.n + w - 1) / w);
}
// Warp `warp` of `warps`; every lane calls it.
template <bool BF16> __device__ __forceinline__ void join_bias(const BiasJoin& j, int warp, int warps) {
  const int rows = static_cast<int>(j.rows), lane = threadIdx.x & 31;
  const int width = bias_join_cols(j), slices = 32 / width, slice = lane / width, col_blocks = (j.n + width - 1) / width;
  const int64_t items = bias_join_items(j);
  for (int64_t it = warp; it < items; it += warps) {
    const int e = static_cast<int>(it / col_blocks);
    const int c = static_cast<int>(it - static_cast<int64_t>(e) * col_blocks) * width + lane % width;
    float v = 0.0f;
    if (c < j.n) {
      const int o0 = j.offsets ? min(max(j.offsets[e], 0), rows) : 0;
      const int o1 = j.offsets ? min(max(j.offsets[e + 1], 0), rows) : rows;
      const float* p = j.partial + static_cast<int64_t>(e) * j.n + c;
      const int last = o1 > o0 ? (o1 - 1) / j.run : -1;
      for (int run = o0 / j.run + slice; run <= last; run += 8 * slices) {  // eight loads in flight, none waits for an add
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = run + i * slices <= last ? p[static_cast<int64_t>(run + i * slices) * j.n] : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += t[i];
      }
    }
    if (slices > 1) {
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
    }
    if (slice == 0 && c < j.n) static_cast<uint16_t*>(j.dbias)[static_cast<int64_t>(e) * j.n + c] = from_f32<BF16>(v);
  }
}
cudaError_t launch_bias_join(const BiasJoin& j, bool bf16, cudaStream_t st);

}  // namespace senmoe
