// linear8_small.cu -- products over 8-bit rows for few rows (decode): the
// weights stream once from global memory into the registers of warp-level
// MMAs, as in linear_small.cu.
//
// A block computes TILES tiles of 16 rows of W (a gated pair: 8 features' gate
// rows over their 8 up rows) for one chunk of up to 8 * NT rows of one group;
// KWARPS warps a tile take runs of kSteps scale blocks (32 k each) in turn.
// Of a block, thread 4g + t of a warp loads 8 consecutive columns, 8t .. 8t + 7,
// of W's rows g and g + 8 and of the chunk's rows g, g + 8, ...; as fp16, which
// holds e4m3, they are the fragments of two m16n8k16 MMAs, since a contraction
// does not depend on the order of k.  (The m16n8k32 MMA of e4m3 itself took
// longer: one token's 8 experts 18.3 us against 13.6.)  A scale block's sums
// start from zero and are added times 2^(sw + sx), in fp32.  The warps' sums
// meet in shared memory and are added in warp order: the same bits every time.
//
// With an 8-bit output a block has 32 features, one scale block of a row of y.

#include "linear8.cuh"

namespace senmoe {
namespace {

// 4 e4m3 as 2 x 2 fp16 (exact)
__device__ __forceinline__ void to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(v)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(v >> 16)));
}
// D += A B, fp16 x fp16, fp32 sums
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 bytes at p, or zeros; W is read once and passes L1 by.
__device__ __forceinline__ uint2 load_w(const uint8_t* p, bool live) {
  uint2 v = make_uint2(0, 0);
  if (live) asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_x(const uint8_t* p, bool live) {
  return live ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
}
// N scales (4 or 2) from block b on, `have` blocks in all, one a byte; words: rows
// lie on a 4-byte grid and are whole words.
template <int N> __device__ __forceinline__ uint32_t load_scales(const uint8_t* p, int b, int have, bool words, bool live,
                                                                 const uint8_t* begin, const uint8_t* end) {
  if (!live || b >= have) return 0x7f7f7f7fu;
  if (words) return N == 4 ? *reinterpret_cast<const uint32_t*>(p + b) : *reinterpret_cast<const uint16_t*>(p + b);
  uint32_t v[1];
  scale_words<1>(p + b, min(N, have - b), begin, end, v);
  return v[0];
}
// d times two scales 2^(w - 127), 2^(x - 127), given by their bytes (up to 254).
// The scales' product can leave fp32 where the result is in range, or zero.  So d
// is multiplied by 2^(floor(s / 2) - 127), then by 2^(ceil(s / 2) - 127), s = w + x:
// within a factor of two of one another, they leave fp32 only with the result.
// (The first is 0 in place of 2^-127, where the result is under 2^-229.)
__device__ __forceinline__ float scaled(float d, uint32_t w, uint32_t x) {
  const uint32_t s = w + x, half = s << 22 & 0x7f800000u;
  return d * __uint_as_float(half) * __uint_as_float((s << 23) - half);
}
__device__ __forceinline__ uint32_t scale_of(uint32_t word, int i) { return word >> 8 * i & 0xffu; }

template <bool BF16, bool GATED, bool EIGHT, int NT> struct Shape {
  static constexpr int kTiles = !EIGHT ? 1 : GATED ? 4 : 2;
  static constexpr int kWarpsK = EIGHT && GATED ? 4 : 8;
  static constexpr int kThreads = 32 * kTiles * kWarpsK;
  static constexpr int kFeat = 16 * kTiles / (GATED ? 2 : 1);  // features of a block
  static constexpr int kSteps = NT > 4 ? 2 : 4;  // scale blocks whose loads are in flight together
  static constexpr int kBlocks = NT > 1 ? 1 : 2;  // an SM, at least
};

template <bool BF16, bool GATED, bool EIGHT, int NT>
__global__ void __launch_bounds__(Shape<BF16, GATED, EIGHT, NT>::kThreads, Shape<BF16, GATED, EIGHT, NT>::kBlocks)
    linear8_small_kernel(const __grid_constant__ Linear8Args a, const bool words) {
  using S = Shape<BF16, GATED, EIGHT, NT>;
  constexpr int kWarps = S::kThreads / 32, kFeat = S::kFeat, kSteps = S::kSteps, kChunk = 8 * NT;
  __shared__ float s_part[S::kWarpsK / 2][16 * S::kTiles][kChunk + 1];
  __shared__ int s_sum[kWarps], s_tile[3];  // group, first row, rows
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int features = GATED ? a.n / 2 : a.n, f0 = blockIdx.x * kFeat, want = blockIdx.y;
  uint16_t *out = static_cast<uint16_t*>(a.y), *pre = static_cast<uint16_t*>(a.preact);
  pdl_wait();
  pdl_launch_dependents();

  // ---- this block's rows: chunk `want` of the groups' chunks
  int e = 0, row0 = want * kChunk, rows;
  if (a.offsets) {
    const int cap = static_cast<int>(a.rows), per = (a.groups + S::kThreads - 1) / S::kThreads;
    const int first = min(tid * per, a.groups), last = min(first + per, a.groups);
    int mine = 0;
    auto range = [&](int i, int& lo, int& cnt) {  // clamped: no row outside the operands whatever offsets holds
      lo = min(max(a.offsets[i], 0), cap);
      cnt = max(min(a.offsets[i + 1], cap) - lo, 0);
    };
    for (int i = first; i < last; ++i) {
      int lo, cnt;
      range(i, lo, cnt);
      mine += (cnt + kChunk - 1) / kChunk;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    if (tid == 0) s_tile[2] = 0;
    __syncthreads();
    int before = incl - mine;
    for (int w = 0; w < warp; ++w) before += s_sum[w];
    if (want >= before && want < before + mine) {
      int at = before;
      for (int i = first; i < last; ++i) {
        int lo, cnt;
        range(i, lo, cnt);
        const int n = (cnt + kChunk - 1) / kChunk;
        if (want < at + n) {
          s_tile[0] = i;
          s_tile[1] = lo + (want - at) * kChunk;
          s_tile[2] = min(kChunk, cnt - (want - at) * kChunk);
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    e = s_tile[0];
    row0 = s_tile[1];
    rows = s_tile[2];
    // rows of no group: zero, this block's features of every gridDim.y-th
    const int head = min(max(a.offsets[0], 0), cap), tail = max(min(a.offsets[a.groups], cap), head);
    const int n = head + (cap - tail), fi = tid % kFeat, f = f0 + fi;
    for (int i = want + gridDim.y * (tid / kFeat); i < n; i += gridDim.y * (S::kThreads / kFeat)) {
      const int64_t r = i < head ? i : tail + (i - head);
      if (f < features) {
        if constexpr (EIGHT) {
          a.codes[r * a.codes_stride + f] = 0;
          if (fi == 0) a.scales[r * a.scales_stride + f / kBlock8] = 0;
        } else {
          out[r * a.y_stride + f] = 0;
        }
        if (pre) pre[r * a.preact_stride + f] = 0;
        if (GATED && pre) pre[r * a.preact_stride + features + f] = 0;
      }
    }
    if (rows == 0) return;
  } else {
    rows = static_cast<int>(min(static_cast<int64_t>(kChunk), a.rows - row0));
  }

  // ---- the products: warp (tile, kw) takes runs kw, kw + KWARPS, ... of kSteps blocks
  const int tile = warp / S::kWarpsK, kw = warp % S::kWarpsK;
  // W's rows g and g + 8 of the tile: two features, or one feature's gate and up
  const int ft = f0 + tile * (GATED ? 8 : 16) + g;
  const bool live0 = ft < features, live1 = GATED ? live0 : ft + 8 < features;
  const int64_t r0 = live0 ? ft : 0, r1 = live1 ? ft + (GATED ? features : 8) : 0;
  const uint8_t* w0 = a.w + e * a.w_group_stride + r0 * a.w_stride + 8 * t4;
  const uint8_t* w1 = a.w + e * a.w_group_stride + r1 * a.w_stride + 8 * t4;
  const uint8_t* sw0 = a.w_scales + e * a.w_scales_group_stride + r0 * a.w_scales_stride;
  const uint8_t* sw1 = a.w_scales + e * a.w_scales_group_stride + r1 * a.w_scales_stride;
  const uint8_t* x0 = a.x + static_cast<int64_t>(row0 + g) * a.x_stride + 8 * t4;
  const uint8_t* sx0 = a.x_scales + static_cast<int64_t>(row0 + 2 * t4) * a.x_scales_stride;
  const int blocks = a.k / kBlock8;
  const uint8_t* const w_end = a.w_scales + (a.groups - 1) * a.w_scales_group_stride + (a.n - 1) * a.w_scales_stride + blocks;
  const uint8_t* const x_end = a.x_scales + (a.rows - 1) * a.x_scales_stride + blocks;
  float acc[NT][4] = {};
  for (int b = kw * kSteps; b < blocks; b += S::kWarpsK * kSteps) {
    uint2 wa[kSteps][2], xb[kSteps][NT];
    uint32_t sw[2], sx[NT][2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = (b + s) * kBlock8;
      const bool in = b + s < blocks;
      wa[s][0] = load_w(w0 + c, live0 && in);
      wa[s][1] = load_w(w1 + c, live1 && in);
    }
    sw[0] = load_scales<kSteps>(sw0, b, blocks, words, live0, a.w_scales, w_end);
    sw[1] = load_scales<kSteps>(sw1, b, blocks, words, live1, a.w_scales, w_end);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        xb[s][n] = load_x(x0 + n * 8 * a.x_stride + (b + s) * kBlock8, n * 8 + g < rows && b + s < blocks);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        sx[n][j] = load_scales<kSteps>(sx0 + (n * 8 + j) * a.x_scales_stride, b, blocks, words, n * 8 + 2 * t4 + j < rows,
                                       a.x_scales, x_end);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (b + s >= blocks) break;
      const uint32_t v0 = scale_of(sw[0], s), v1 = scale_of(sw[1], s);
      uint32_t a0[4], a1[4];  // rows g and g + 8, in fp16 pairs
      to_f16(wa[s][0].x, a0[0], a0[1]);
      to_f16(wa[s][0].y, a0[2], a0[3]);
      to_f16(wa[s][1].x, a1[0], a1[1]);
      to_f16(wa[s][1].y, a1[2], a1[3]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t x[4];
        to_f16(xb[s][n].x, x[0], x[1]);
        to_f16(xb[s][n].y, x[2], x[3]);
        float d[4] = {};
        mma16816(d, a0[0], a1[0], a0[1], a1[1], x[0], x[1]);
        mma16816(d, a0[2], a1[2], a0[3], a1[3], x[2], x[3]);
        const uint32_t u0 = scale_of(sx[n][0], s), u1 = scale_of(sx[n][1], s);
        acc[n][0] += scaled(d[0], v0, u0);
        acc[n][1] += scaled(d[1], v0, u1);
        acc[n][2] += scaled(d[2], v1, u0);
        acc[n][3] += scaled(d[3], v1, u1);
        if (max(max(v0, v1), max(u0, u1)) == 255u) {  // a scale that is NaN: so are its rows' sums, from here on
          const float nan = __uint_as_float(0x7fc00000u);
          if (max(v0, u0) == 255u) acc[n][0] = nan;
          if (max(v0, u1) == 255u) acc[n][1] = nan;
          if (max(v1, u0) == 255u) acc[n][2] = nan;
          if (max(v1, u1) == 255u) acc[n][3] = nan;
        }
      }
    }
  }

  // ---- partial sums: the upper half of a tile's warps hand over to the lower, then those are added
  constexpr int kHalf = S::kWarpsK / 2;
  auto each = [&](auto&& f) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        f(acc[n][q], s_part[kw % kHalf][tile * 16 + g + (q >> 1) * 8][n * 8 + 2 * t4 + (q & 1)]);
  };
  if (kw >= kHalf) each([](float& v, float& s) { s = v; });
  __syncthreads();
  if (kw < kHalf) each([](float& v, float& s) { s += v; });
  __syncthreads();

  // ---- epilogue: the block's features of a row at a time (8 bits: a warp a row)
  const uint16_t *bias = static_cast<const uint16_t*>(a.bias), *res = static_cast<const uint16_t*>(a.residual);
  const int fi = tid % kFeat, f = f0 + fi;
  if (f >= features) return;  // (8 bits: features are whole blocks, none is)
  const int i0 = GATED ? (fi >> 3) * 16 + (fi & 7) : fi;  // its row in the tiles; a gated pair's up is 8 on
  const float b0 = bias ? to_f32<BF16>(bias[static_cast<int64_t>(e) * a.n + f]) : 0.0f;
  const float b1 = GATED && bias ? to_f32<BF16>(bias[static_cast<int64_t>(e) * a.n + features + f]) : 0.0f;
  for (int r = tid / kFeat; r < rows; r += S::kThreads / kFeat) {
    const int64_t row = row0 + r;
    float z = b0;
#pragma unroll
    for (int w = 0; w < kHalf; ++w) z += s_part[w][i0][r];
    if (pre) pre[row * a.preact_stride + f] = from_f32<BF16>(z);
    float y = act_value<EIGHT>(a.act, z);
    if constexpr (GATED) {
      float u = b1;
#pragma unroll
      for (int w = 0; w < kHalf; ++w) u += s_part[w][i0 + 8][r];
      if (pre) pre[row * a.preact_stride + features + f] = from_f32<BF16>(u);
      y *= u;
    }
    if (res) y += to_f32<BF16>(res[row * a.residual_stride + f]);
    if constexpr (EIGHT) {
      uint32_t byte;
      a.codes[row * a.codes_stride + f] = pack8_warp(y, byte);
      if (lane == 0) a.scales[row * a.scales_stride + f / kBlock8] = static_cast<uint8_t>(byte);
    } else {
      out[row * a.y_stride + f] = from_f32<BF16>(y);
    }
  }
}

template <bool BF16, bool GATED, bool EIGHT, int NT> cudaError_t launch_t(const Linear8Args& a, bool words, cudaStream_t st) {
  using S = Shape<BF16, GATED, EIGHT, NT>;
  const int64_t most = (a.rows + 8 * NT - 1) / (8 * NT) + (a.offsets ? a.groups : 0);
  const int features = GATED ? a.n / 2 : a.n;
  const dim3 grid((features + S::kFeat - 1) / S::kFeat, static_cast<unsigned>(most < a.rows ? most : a.rows));
  return launch_pdl(linear8_small_kernel<BF16, GATED, EIGHT, NT>, grid, dim3(S::kThreads), 0, st, a, words);
}
template <bool BF16, bool GATED, bool EIGHT> cudaError_t launch_n(const Linear8Args& a, bool words, cudaStream_t st) {
  switch (linear8_small_chunk(a)) {
    case 8: return launch_t<BF16, GATED, EIGHT, 1>(a, words, st);
    case 16: return launch_t<BF16, GATED, EIGHT, 2>(a, words, st);
    case 32: return launch_t<BF16, GATED, EIGHT, 4>(a, words, st);
    default: return launch_t<BF16, GATED, EIGHT, 8>(a, words, st);
  }
}
template <bool EIGHT> cudaError_t launch_e(const Linear8Args& a, bool words, cudaStream_t st) {
  if (act_gated(a.act)) return a.bf16 ? launch_n<true, true, EIGHT>(a, words, st) : launch_n<false, true, EIGHT>(a, words, st);
  return a.bf16 ? launch_n<true, false, EIGHT>(a, words, st) : launch_n<false, false, EIGHT>(a, words, st);
}

}  // namespace

bool linear8_small_supported(const Linear8Args& a) { return (a.rows + 7) / 8 + a.groups <= 65535; }

cudaError_t launch_linear8_small(const Linear8Args& a, cudaStream_t st) {
  const auto whole = [](const void* p, int64_t stride, int64_t group) {
    return ((reinterpret_cast<uintptr_t>(p) | stride | group) & 3) == 0;
  };
  // scales four at a time: rows on a 4-byte grid, of whole words
  const bool words = a.k / kBlock8 % 4 == 0 && whole(a.x_scales, a.x_scales_stride, 0) &&
                     whole(a.w_scales, a.w_scales_stride, a.groups > 1 ? a.w_scales_group_stride : 0);
  return a.codes ? launch_e<true>(a, words, st) : launch_e<false>(a, words, st);
}

}  // namespace senmoe
