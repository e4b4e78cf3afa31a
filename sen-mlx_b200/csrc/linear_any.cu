// linear_any.cu -- the linear products for operands of any strides and
// alignments: C[i, j] = sum_k A(i, k) B(j, k) over 64 x 64 tiles, warp-level
// MMA with fp32 accumulation.
//
// Each block copies 64 x 32 blocks of A and B element by element into shared
// memory with k innermost, whichever way they lie in global memory, and four
// warps take a 32 x 32 quarter each.  Elements past a group's rows, or past
// the matrices' edges, are zeroed on the way in and never read.  A gated pair
// keeps a second accumulator over B's rows `half` further on, so the
// activation needs no exchange.  Bound by its copies (two bytes a load): 53
// TFLOP/s at 8192 x 2048 x 8192, 750 GB/s on 64 tokens over 128 experts; it
// serves the operands that TMA cannot read, where being right for every
// stride comes before speed.

#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kT = 64, kKB = 32, kPad = 8;  // tile, k block, padding against bank conflicts
constexpr int kThreads = 128;

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A 64 x 32 block of M(i, k) into s[i][k]; KMAJOR: k runs along memory,
// otherwise i does.  i < ni and k < nk are read, the rest is zero.
template <bool KMAJOR>
__device__ __forceinline__ void fill(uint16_t (*s)[kKB + kPad], const uint16_t* m, int64_t stride, int ni, int nk) {
#pragma unroll
  for (int t = 0; t < kT * kKB / kThreads; ++t) {
    const int q = t * kThreads + threadIdx.x;
    const int i = KMAJOR ? q / kKB : q % kT, k = KMAJOR ? q % kKB : q / kT;
    s[i][k] = i < ni && k < nk ? m[KMAJOR ? i * stride + k : k * stride + i] : uint16_t(0);
  }
}

template <bool BF16, int PROD, bool GATED>
__global__ void __launch_bounds__(kThreads) linear_any_kernel(const LinearArgs a, int col_tiles) {
  constexpr int NB = GATED ? 2 : 1;
  __shared__ __align__(16) uint16_t sA[kT][kKB + kPad];
  __shared__ __align__(16) uint16_t sB[NB][kT][kKB + kPad];
  __shared__ int s_off[kMaxGroups + 1], s_pre[kMaxGroups + 1], s_tot[64];
  pdl_wait();
  pdl_launch_dependents();
  group_table(a.offsets, a.groups, a.rows, kT, s_off, s_pre, s_tot);

  const uint16_t* ga = static_cast<const uint16_t*>(a.a);
  const uint16_t* gb = static_cast<const uint16_t*>(a.b);
  uint16_t* out = static_cast<uint16_t*>(a.out);
  uint16_t* preact = static_cast<uint16_t*>(a.preact);
  const int half = a.n / NB;  // forward: columns of y; rows of W past the gate's
  const int cols = PROD == kProdForward ? half : a.k;
  if constexpr (PROD != kProdWeight) {
    zero_uncovered(s_off, a.groups, a.rows, out, a.out_stride, cols, blockIdx.x, gridDim.x);
    if (preact) zero_uncovered(s_off, a.groups, a.rows, preact, a.preact_stride, a.n, blockIdx.x, gridDim.x);
  }
  const int row_tiles = PROD == kProdWeight ? (a.n + kT - 1) / kT : 0;  // dW: of every group
  const int64_t tiles = static_cast<int64_t>(col_tiles) *
                        (PROD == kProdWeight ? static_cast<int64_t>(a.groups) * row_tiles : s_pre[a.groups]);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int wi = (warp >> 1) * 32, wj = (warp & 1) * 32;

  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int j0 = static_cast<int>(tile % col_tiles) * kT;
    const int rt = static_cast<int>(tile / col_tiles);
    int e, i0, ni, kn;
    const uint16_t *pa, *pb;
    if constexpr (PROD == kProdWeight) {
      e = rt / row_tiles;
      i0 = (rt - e * row_tiles) * kT;
      ni = min(kT, a.n - i0);
      kn = s_off[e + 1] - s_off[e];
      pa = ga + s_off[e] * a.a_stride + i0;
      pb = gb + s_off[e] * a.b_stride + j0;
    } else {
      e = group_of(s_pre, a.groups, rt);
      i0 = s_off[e] + (rt - s_pre[e]) * kT;
      ni = min(kT, s_off[e + 1] - i0);
      kn = PROD == kProdForward ? a.k : a.n;
      pa = ga + i0 * a.a_stride;
      pb = gb + e * a.b_group_stride + (PROD == kProdForward ? j0 * a.b_stride : int64_t(j0));
    }
    const int nj = min(kT, cols - j0);
    float acc[NB][2][4][4] = {};
    for (int k0 = 0; k0 < kn; k0 += kKB) {
      const int nk = min(kKB, kn - k0);
      if constexpr (PROD == kProdWeight) {
        fill<false>(sA, pa + k0 * a.a_stride, a.a_stride, ni, nk);
        fill<false>(sB[0], pb + k0 * a.b_stride, a.b_stride, nj, nk);
      } else {
        fill<true>(sA, pa + k0, a.a_stride, ni, nk);
        if constexpr (PROD == kProdForward) {
#pragma unroll
          for (int h = 0; h < NB; ++h) fill<true>(sB[h], pb + h * half * a.b_stride + k0, a.b_stride, nj, nk);
        } else {
          fill<false>(sB[0], pb + k0 * a.b_stride, a.b_stride, nj, nk);
        }
      }
      __syncthreads();
#pragma unroll
      for (int ks = 0; ks < kKB; ks += 16) {
        uint32_t fa[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int r = wi + m * 16 + g, c = ks + 2 * t4;
          fa[m][0] = *reinterpret_cast<const uint32_t*>(&sA[r][c]);
          fa[m][1] = *reinterpret_cast<const uint32_t*>(&sA[r + 8][c]);
          fa[m][2] = *reinterpret_cast<const uint32_t*>(&sA[r][c + 8]);
          fa[m][3] = *reinterpret_cast<const uint32_t*>(&sA[r + 8][c + 8]);
        }
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int r = wj + n * 8 + g, c = ks + 2 * t4;
            const uint32_t b0 = *reinterpret_cast<const uint32_t*>(&sB[h][r][c]);
            const uint32_t b1 = *reinterpret_cast<const uint32_t*>(&sB[h][r][c + 8]);
#pragma unroll
            for (int m = 0; m < 2; ++m) mma16816<BF16>(acc[h][m][n], fa[m], b0, b1);
          }
      }
      __syncthreads();
    }
    // epilogue
    const uint16_t* bias = static_cast<const uint16_t*>(a.bias);
    const uint16_t* res = static_cast<const uint16_t*>(a.residual);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = wi + m * 16 + g + (q >> 1) * 8, j = wj + n * 8 + 2 * t4 + (q & 1);
          if (i >= ni || j >= nj) continue;
          float z = acc[0][m][n][q];
          if (PROD != kProdForward && a.dz_max) z *= power_of_two(dz_exponent(a.dz_max[e]));
          if constexpr (PROD == kProdForward) {
            const int64_t row = i0 + i;
            const int64_t bcol = static_cast<int64_t>(e) * a.n + j0 + j;
            if (bias) z += to_f32<BF16>(bias[bcol]);
            if (preact) preact[row * a.preact_stride + j0 + j] = from_f32<BF16>(z);
            float y = act_value(a.act, z);
            if constexpr (GATED) {
              float u = acc[1][m][n][q];
              if (bias) u += to_f32<BF16>(bias[bcol + half]);
              if (preact) preact[row * a.preact_stride + half + j0 + j] = from_f32<BF16>(u);
              y *= u;
            }
            if (res) y += to_f32<BF16>(res[row * a.residual_stride + j0 + j]);
            out[row * a.out_stride + j0 + j] = from_f32<BF16>(y);
          } else if constexpr (PROD == kProdInput) {
            out[static_cast<int64_t>(i0 + i) * a.out_stride + j0 + j] = from_f32<BF16>(z);
          } else {
            out[e * a.out_group_stride + static_cast<int64_t>(i0 + i) * a.out_stride + j0 + j] = from_f32<BF16>(z);
          }
        }
  }
}

template <bool BF16, int PROD, bool GATED>
cudaError_t launch_t(const LinearArgs& a, cudaStream_t st) {
  const int cols = PROD == kProdForward ? a.n / (GATED ? 2 : 1) : a.k;
  const int col_tiles = (cols + kT - 1) / kT;
  const int64_t row_tiles = PROD == kProdWeight ? static_cast<int64_t>(a.groups) * ((a.n + kT - 1) / kT)
                                                : (a.rows + kT - 1) / kT + (a.offsets ? a.groups : 0);
  int64_t grid = row_tiles * col_tiles;
  if (grid > 148 * 8) grid = 148 * 8;  // a few blocks an SM; the rest by the stride
  if (grid < 1) grid = 1;
  return launch_pdl(linear_any_kernel<BF16, PROD, GATED>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, a,
                    col_tiles);
}

template <bool BF16> cudaError_t launch_dtype(const LinearArgs& a, LinearProduct p, cudaStream_t st) {
  if (p == kProdInput) return launch_t<BF16, kProdInput, false>(a, st);
  if (p == kProdWeight) return launch_t<BF16, kProdWeight, false>(a, st);
  return act_gated(a.act) ? launch_t<BF16, kProdForward, true>(a, st) : launch_t<BF16, kProdForward, false>(a, st);
}

}  // namespace

cudaError_t launch_linear_any(const LinearArgs& a, LinearProduct p, cudaStream_t st) {
  return a.bf16 ? launch_dtype<true>(a, p, st) : launch_dtype<false>(a, p, st);
}

}  // namespace senmoe
