// quantize8.cu -- 16-bit rows into 8 bits with scales (rows8.cuh): x itself,
// or dz = dy act'(z), the operand of an input gradient in 8 bits.
//
// dz is evaluated in fp32 and goes to its 8 bits from there, without a 16-bit
// rounding between, so that an fp16 dz needs no range of its own either.

#include "rows8.cuh"

#include "linear8.cuh"

namespace senmoe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;


// One row's V columns (gated: the gate's and the up's) as loaded, and the
// values to store of them; lanes without columns hold zeros.
template <bool BF16, int V, int ACT> struct Piece {
  static constexpr bool kGated = ACT >= kActSwiglu;
  using Raw = std::conditional_t<V == 8, uint4, uint16_t>;
  Raw y = {}, z = {}, u = {};
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[V]) {
    if constexpr (V == 8) unpack8<BF16>(v, f);
    else f[0] = to_f32<BF16>(v);
  }
  __device__ __forceinline__ void load(const uint16_t* x, const uint16_t* pre, int cols) {
    y = *reinterpret_cast<const Raw*>(x);
    if constexpr (ACT != kActNone) z = *reinterpret_cast<const Raw*>(pre);
    if constexpr (kGated) u = *reinterpret_cast<const Raw*>(pre + cols);
  }
  __device__ __forceinline__ void values(float (&g)[V], float (&up)[V]) const {
    unpack(y, g);
    if constexpr (ACT != kActNone) {
      float zf[V];
      unpack(z, zf);
      if constexpr (kGated) unpack(u, up);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float value;
        const float d = g[i];
        g[i] = d * act_both<true>(ACT, zf[i], value);
        if constexpr (kGated) {
          g[i] *= up[i];
          up[i] = d * value;
        }
      }
    }
  }
};

template <int V> __device__ __forceinline__ void store8(const float (&f)[V], uint8_t* codes, uint8_t* scales, int c,
                                                        bool in, int lane) {
  uint32_t byte;
  if constexpr (V == 8) {
    const uint2 q = pack8_lane(f, byte);
    if (in) *reinterpret_cast<uint2*>(codes + c) = q;
    if (in && (lane & 3) == 0) scales[c / kBlock8] = static_cast<uint8_t>(byte);
  } else {
    const uint8_t q = pack8_warp(f[0], byte);
    if (in) codes[c] = q;
    if (in && lane == 0) scales[c / kBlock8] = static_cast<uint8_t>(byte);
  }
}

// A warp takes a piece of a row (kUnroll steps, their loads in flight
// together), V columns a lane and step: 8 where rows start on a 16-byte grid,
// else 1.  Bound by HBM.
template <bool BF16, int V, int ACT>
__global__ void __launch_bounds__(kThreads) quantize8_kernel(const __grid_constant__ Quantize8Args a) {
  using P = Piece<BF16, V, ACT>;
  constexpr int kUnroll = V == 8 ? (P::kGated ? 3 : 4) : 1;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const unsigned pieces = (a.n + 32 * V * kUnroll - 1) / (32 * V * kUnroll);
  const int64_t items = a.rows * pieces, warps = static_cast<int64_t>(gridDim.x) * kWarps;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); it < items; it += warps) {
    const int64_t r = it < 0xffffffffll ? static_cast<unsigned>(it) / pieces : it / pieces;
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + r * a.x_stride;
    const uint16_t* pre = static_cast<const uint16_t*>(a.preact) + r * a.preact_stride;
    uint8_t *codes = a.codes + r * a.codes_stride, *scales = a.scales + r * a.scales_stride;
    const int c0 = static_cast<int>(it - r * pieces) * 32 * V * kUnroll + lane * V;
    P piece[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (c0 + j * 32 * V < a.n) piece[j].load(x + c0 + j * 32 * V, pre + c0 + j * 32 * V, a.n);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int c = c0 + j * 32 * V;
      float g[V], up[V];
      piece[j].values(g, up);
      store8<V>(g, codes, scales, c, c < a.n, lane);
      if constexpr (P::kGated) store8<V>(up, codes + a.n, scales + a.n / kBlock8, c, c < a.n, lane);
    }
  }
}

template <bool BF16, int V, int ACT> cudaError_t launch_t(const Quantize8Args& a, cudaStream_t st) {
  constexpr int kCols = 32 * V * (V == 8 ? (ACT >= kActSwiglu ? 3 : 4) : 1);
  const int64_t items = a.rows * ((a.n + kCols - 1) / kCols), blocks = (items + kWarps - 1) / kWarps;
  return launch_pdl(quantize8_kernel<BF16, V, ACT>, dim3(static_cast<unsigned>(blocks < 148 * 64 ? blocks : 148 * 64)),
                    dim3(kThreads), 0, st, a);
}
template <bool BF16, int V> cudaError_t launch_v(const Quantize8Args& a, cudaStream_t st) {
  switch (a.act) {
    case kActRelu: return launch_t<BF16, V, kActRelu>(a, st);
    case kActSilu: return launch_t<BF16, V, kActSilu>(a, st);
    case kActGelu: return launch_t<BF16, V, kActGelu>(a, st);
    case kActGeluTanh: return launch_t<BF16, V, kActGeluTanh>(a, st);
    case kActSwiglu: return launch_t<BF16, V, kActSwiglu>(a, st);
    case kActGeglu: return launch_t<BF16, V, kActGeglu>(a, st);
    default: return launch_t<BF16, V, kActNone>(a, st);
  }
}

}  // namespace

cudaError_t launch_quantize8(const Quantize8Args& a, cudaStream_t st) {
  const auto on16 = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0;
  };
  const bool wide = on16(a.x, a.x_stride) && (a.act == kActNone || on16(a.preact, a.preact_stride)) &&
                    (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0 && a.codes_stride % 8 == 0;
  if (wide) return a.bf16 ? launch_v<true, 8>(a, st) : launch_v<false, 8>(a, st);
  return a.bf16 ? launch_v<true, 1>(a, st) : launch_v<false, 1>(a, st);
}

}  // namespace senmoe
