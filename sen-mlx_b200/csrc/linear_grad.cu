// linear_grad.cu -- the elementwise and column-sum parts of the linear
// products' backward pass.
//
// act_backward: dz = dy * act'(z) (gated: dg = dy * u * act'(g), du = dy *
// act(g)), evaluated in fp32 and rounded once to the operands' 16-bit type,
// because dz is an operand of both gradient products on the 16-bit tensor
// cores.  The rounding (at most 2^-8 of the value in bf16, 2^-11 in fp16) is
// independent from element to element and so adds to a gradient about as much
// as the gradient's own rounding does: 0.0023 of a gradient's norm in bf16
// against 0.0017 for fp32 sums of an unrounded dz.  Over some 10,000 random
// sizes the ratio was 1.4, and up to 1.8 where a few large elements decide
// (a handful of rows, short bias gradients).  Carrying dz in two 16-bit parts
// would bring it to 1 for twice the products.
//
// bias_grad: db[e] = sum of dz's rows of group e, in fp32 and in a fixed
// order (rows strided over 8 warps, then warps, then splits), so repeated
// calls agree bit for bit.

#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kActThreads = 256;

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

// A warp a piece of a row (kUnroll steps), V columns a lane and step: 8 (16-byte accesses) where every
// row starts on a 16-byte boundary, else 1.  The loads of kUnroll steps are in
// flight together.  Bound by HBM: dy and z read once, dz written once; 36 us
// for 32768 rows of 2 x 768 (252 MB, 7.0 TB/s with part of the writes still in
// L2; 82 us with a thread an element group and a division each).
template <bool BF16, int V, int ACT>
__global__ void __launch_bounds__(kActThreads) act_backward_kernel(const LinearGradArgs a) {
  constexpr bool kGated = ACT >= kActSwiglu;
  constexpr int kUnroll = V == 8 ? 3 : 1;
  pdl_wait();
  pdl_launch_dependents();
  const int cols = kGated ? a.n / 2 : a.n;
  const int lane = threadIdx.x & 31;
  const unsigned pieces = (cols + 32 * V * kUnroll - 1) / (32 * V * kUnroll);
  const int64_t items = a.rows * pieces, warps = gridDim.x * (kActThreads / 32);
  for (int64_t it = blockIdx.x * (kActThreads / 32) + (threadIdx.x >> 5); it < items; it += warps) {
    const int64_t r = it < 0xffffffffll ? static_cast<unsigned>(it) / pieces : it / pieces;
    const uint16_t* py = static_cast<const uint16_t*>(a.dy) + r * a.dy_stride;
    const uint16_t* pz = static_cast<const uint16_t*>(a.preact) + r * a.preact_stride;
    uint16_t* po = static_cast<uint16_t*>(a.dz) + r * a.dz_stride;
    const int c0 = static_cast<int>(it - r * pieces) * 32 * V * kUnroll + lane * V;
    uint4 vy[kUnroll], vz[kUnroll], vu[kUnroll];
    if constexpr (V == 8) {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        const int c = c0 + j * 256;
        if (c < cols) {
          vy[j] = *reinterpret_cast<const uint4*>(py + c);
          vz[j] = *reinterpret_cast<const uint4*>(pz + c);
          if constexpr (kGated) vu[j] = *reinterpret_cast<const uint4*>(pz + cols + c);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int c = c0 + j * 32 * V;
      if (c >= cols) break;
      float d[V], z[V], u[V], g[V];
      if constexpr (V == 8) {
        unpack8<BF16>(vy[j], d);
        unpack8<BF16>(vz[j], z);
        if constexpr (kGated) unpack8<BF16>(vu[j], u);
      } else {
        d[0] = to_f32<BF16>(py[c]);
        z[0] = to_f32<BF16>(pz[c]);
        if constexpr (kGated) u[0] = to_f32<BF16>(pz[cols + c]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float value;
        const float slope = act_both(ACT, z[i], value);
        g[i] = d[i] * slope;
        if constexpr (kGated) {
          g[i] *= u[i];
          u[i] = d[i] * value;
        }
      }
      if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(po + c) = pack8<BF16>(g);
        if constexpr (kGated) *reinterpret_cast<uint4*>(po + cols + c) = pack8<BF16>(u);
      } else {
        po[c] = from_f32<BF16>(g[0]);
        if constexpr (kGated) po[cols + c] = from_f32<BF16>(u[0]);
      }
    }
  }
}

template <bool BF16, int V> auto act_backward_for(int act) {
  switch (act) {
    case kActRelu: return act_backward_kernel<BF16, V, kActRelu>;
    case kActSilu: return act_backward_kernel<BF16, V, kActSilu>;
    case kActGelu: return act_backward_kernel<BF16, V, kActGelu>;
    case kActGeluTanh: return act_backward_kernel<BF16, V, kActGeluTanh>;
    case kActSwiglu: return act_backward_kernel<BF16, V, kActSwiglu>;
    case kActGeglu: return act_backward_kernel<BF16, V, kActGeglu>;
    default: return act_backward_kernel<BF16, V, kActNone>;
  }
}

constexpr int kSumCols = 256;  // columns of a block: eight a lane

// vec: every row starts on a 16-byte boundary.
template <bool BF16>
__global__ void __launch_bounds__(256) bias_grad_kernel(const LinearGradArgs a, const uint16_t* src, int64_t stride,
                                                        bool vec) {
  __shared__ int s_off[kMaxGroups + 1], s_pre[kMaxGroups + 1], s_tot[64];
  __shared__ float s_sum[8][kSumCols];
  pdl_wait();
  pdl_launch_dependents();
  group_table(a.offsets, a.groups, a.rows, 1, s_off, s_pre, s_tot);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col_blocks = (a.n + kSumCols - 1) / kSumCols;
  const int64_t items = static_cast<int64_t>(a.groups) * a.splits * col_blocks;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int cb = static_cast<int>(it % col_blocks);
    const int es = static_cast<int>(it / col_blocks), e = es / a.splits, sp = es - e * a.splits;
    const int cnt = s_off[e + 1] - s_off[e], per = (cnt + a.splits - 1) / a.splits;
    const int r0 = min(sp * per, cnt), r1 = min(r0 + per, cnt);
    const int c = cb * kSumCols + 8 * lane;
    float x[8] = {};
    const uint16_t* p = src + static_cast<int64_t>(s_off[e]) * stride + c;
    if (vec && c + 8 <= a.n) {
#pragma unroll 4
      for (int r = r0 + warp; r < r1; r += 8) {
        float f[8];
        unpack8<BF16>(*reinterpret_cast<const uint4*>(p + r * stride), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += f[i];
      }
    } else {
      for (int r = r0 + warp; r < r1; r += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < a.n) x[i] += to_f32<BF16>(p[r * stride + i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_sum[warp][8 * lane + i] = x[i];
    __syncthreads();
    const int col = cb * kSumCols + threadIdx.x;
    if (col < a.n) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += s_sum[w][threadIdx.x];
      if (a.splits > 1)
        a.partial[static_cast<int64_t>(es) * a.n + col] = v;
      else
        static_cast<uint16_t*>(a.dbias)[static_cast<int64_t>(e) * a.n + col] = from_f32<BF16>(v);
    }
    __syncthreads();
  }
}

template <bool BF16> __global__ void __launch_bounds__(256) bias_join_kernel(const LinearGradArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t total = static_cast<int64_t>(a.groups) * a.n;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t e = i / a.n, c = i - e * a.n;
    float v = 0.0f;
    for (int s = 0; s < a.splits; ++s) v += a.partial[(e * a.splits + s) * a.n + c];
    static_cast<uint16_t*>(a.dbias)[i] = from_f32<BF16>(v);
  }
}

bool on16(const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; }

unsigned grid_for(int64_t items, int64_t cap) {
  const int64_t g = items < cap ? items : cap;
  return static_cast<unsigned>(g < 1 ? 1 : g);
}

}  // namespace

cudaError_t launch_act_backward(const LinearGradArgs& a, cudaStream_t st) {
  const int cols = act_gated(a.act) ? a.n / 2 : a.n;
  const bool wide = cols % 8 == 0 && on16(a.dy, a.dy_stride) && on16(a.preact, a.preact_stride) &&
                    on16(a.dz, a.dz_stride);
  const int64_t items = a.rows * ((cols + (wide ? 767 : 31)) / (wide ? 768 : 32));
  const dim3 grid(grid_for((items + kActThreads / 32 - 1) / (kActThreads / 32), 148 * 16)), block(kActThreads);
  auto kern = a.bf16 ? (wide ? act_backward_for<true, 8>(a.act) : act_backward_for<true, 1>(a.act))
                     : (wide ? act_backward_for<false, 8>(a.act) : act_backward_for<false, 1>(a.act));
  return launch_pdl(kern, grid, block, 0, st, a);
}

cudaError_t launch_bias_grad(const LinearGradArgs& a, cudaStream_t st) {
  const uint16_t* src = static_cast<const uint16_t*>(a.preact ? a.dz : a.dy);
  const int64_t stride = a.preact ? a.dz_stride : a.dy_stride;
  const int64_t items = static_cast<int64_t>(a.groups) * a.splits * ((a.n + kSumCols - 1) / kSumCols);
  auto kern = a.bf16 ? bias_grad_kernel<true> : bias_grad_kernel<false>;
  cudaError_t e = launch_pdl(kern, dim3(grid_for(items, 148 * 8)), dim3(256), 0, st, a, src, stride, on16(src, stride));
  if (e != cudaSuccess || a.splits <= 1) return e;
  auto join = a.bf16 ? bias_join_kernel<true> : bias_join_kernel<false>;
  return launch_pdl(join, dim3(grid_for((static_cast<int64_t>(a.groups) * a.n + 255) / 256, 148 * 8)), dim3(256), 0,
                    st, a);
}

}  // namespace senmoe
