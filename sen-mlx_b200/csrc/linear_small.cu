// linear_small.cu -- forward linear products of few rows (decode): the
// weights stream once from global memory into the registers of warp-level
// MMAs, with no shared memory, barrier or TMEM between.
//
// A block computes 16 rows of W (a gated pair: 8 features' gate rows over
// their 8 up rows, which leaves a feature's two sums in one thread) for one
// chunk of up to 8 * NT rows of one group; its eight warps take 32-column
// steps of K in turn.  In a step thread 4g + t of a warp loads the 8
// consecutive columns 8t .. 8t + 7 of W's rows g and g + 8 and of the
// chunk's rows g, g + 8, ...: 16 bytes each.  An m16n8k16 MMA wants k pairs
// (2t, 2t + 1) and (2t + 8, 2t + 9) in a thread; since a contraction does not
// depend on the order of k, elements 0-3 of the 8 serve as one MMA's and 4-7
// as the next one's, the same for both operands, so what is loaded is the
// fragment.  The warps' partial sums meet in shared memory and are added in
// warp order: the same bits every time.
//
// Bound by HBM, and for the smallest products by the launch and one trip to
// memory: the tcgen05 kernel's set-up (TMEM, barriers, tensor maps, a K split
// over a cluster) costs more than such a product itself.  Measured: one row x
// 2048 x 2048 3.3 us with W in L2, 4.3 from HBM (the tcgen05 kernel 10.5); one
// token's 8 experts, 2048 -> 2 x 768, 10.7 us = 4.7 TB/s (18): 768 blocks for the
// 444 places that 77 registers a thread leave, 1.73 waves.

#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kWarps = 8;
constexpr int kRows = 16;  // of W, a block

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes at p, or zeros; W is read once and passes L1 by.
__device__ __forceinline__ uint4 load_w(const uint16_t* p, bool live) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (live)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 load_x(const uint16_t* p, bool live) {
  return live ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

template <bool BF16, bool GATED, int NT>
__global__ void __launch_bounds__(kWarps * 32) linear_small_kernel(const __grid_constant__ LinearArgs a) {
  constexpr int kFeat = GATED ? kRows / 2 : kRows;  // features of a block
  constexpr int kSteps = NT > 2 ? 2 : 4;  // K steps whose loads, of W and of the rows, are in flight together
  __shared__ float s_part[kWarps / 2][kRows][NT * 8 + 1];
  __shared__ int s_sum[kWarps], s_tile[3];  // group, first row, rows
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  constexpr int kChunk = 8 * NT;
  const int features = GATED ? a.n / 2 : a.n, f0 = blockIdx.x * kFeat, want = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();

  // ---- this block's rows: chunk `want` of the groups' chunks
  int e = 0, row0 = want * kChunk, rows;
  if (a.offsets) {
    const int cap = static_cast<int>(a.rows), per = (a.groups + kWarps * 32 - 1) / (kWarps * 32);
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
    uint16_t *out = static_cast<uint16_t*>(a.out), *pre = static_cast<uint16_t*>(a.preact);
    const int n = head + (cap - tail), f = f0 + tid % kFeat;
    for (int i = want + gridDim.y * (tid / kFeat); i < n; i += gridDim.y * (kWarps * 32 / kFeat)) {
      const int64_t r = i < head ? i : tail + (i - head);
      if (f < features) {
        out[r * a.out_stride + f] = 0;
        if (pre) pre[r * a.preact_stride + f] = 0;
        if (GATED && pre) pre[r * a.preact_stride + features + f] = 0;
      }
    }
    if (rows == 0) return;
  } else {
    rows = static_cast<int>(min(static_cast<int64_t>(kChunk), a.rows - row0));
  }

  // ---- the products: warp w takes K steps w, w + 8, ...
  // W's rows g and g + 8 of the block: features f0 + g and f0 + g + 8, or one feature's gate and up
  const uint16_t* w0 = static_cast<const uint16_t*>(a.b) + e * a.b_group_stride + (f0 + g) * a.b_stride + 8 * t4;
  const uint16_t* w1 = w0 + (GATED ? features : 8) * a.b_stride;
  const uint16_t* x0 = static_cast<const uint16_t*>(a.a) + (row0 + g) * a.a_stride + 8 * t4;
  const bool live0 = f0 + g < features, live1 = GATED ? live0 : f0 + g + 8 < features;
  float acc[NT][4] = {};
  for (int s0 = warp * 32; s0 < a.k; s0 += kWarps * 32 * kSteps) {
    uint4 wa[kSteps][2], xb[kSteps][NT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = s0 + s * kWarps * 32;
      const bool in = c + 8 * t4 < a.k;
      wa[s][0] = load_w(w0 + c, live0 && in);
      wa[s][1] = load_w(w1 + c, live1 && in);
#pragma unroll
      for (int n = 0; n < NT; ++n) xb[s][n] = load_x(x0 + n * 8 * a.a_stride + c, n * 8 + g < rows && in);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = s0 + s * kWarps * 32;
      if (c >= a.k) break;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = xb[s][n];
        mma16816<BF16>(acc[n], wa[s][0].x, wa[s][1].x, wa[s][0].y, wa[s][1].y, b.x, b.y);
        mma16816<BF16>(acc[n], wa[s][0].z, wa[s][1].z, wa[s][0].w, wa[s][1].w, b.z, b.w);
      }
    }
  }

  // ---- partial sums: warps 4-7 hand over to 0-3, then the four are added
  auto each = [&](auto&& f) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) f(acc[n][q], s_part[warp & 3][g + (q >> 1) * 8][n * 8 + 2 * t4 + (q & 1)]);
  };
  if (warp >= kWarps / 2) each([](float& v, float& s) { s = v; });
  __syncthreads();
  if (warp < kWarps / 2) each([](float& v, float& s) { s += v; });
  __syncthreads();

  // ---- epilogue: the block's features of a row at a time
  const uint16_t *bias = static_cast<const uint16_t*>(a.bias), *res = static_cast<const uint16_t*>(a.residual);
  uint16_t *out = static_cast<uint16_t*>(a.out), *pre = static_cast<uint16_t*>(a.preact);
  const int fi = tid % kFeat, f = f0 + fi;
  if (f >= features) return;
  const float b0 = bias ? to_f32<BF16>(bias[static_cast<int64_t>(e) * a.n + f]) : 0.0f;
  const float b1 = GATED && bias ? to_f32<BF16>(bias[static_cast<int64_t>(e) * a.n + features + f]) : 0.0f;
  for (int r = tid / kFeat; r < rows; r += kWarps * 32 / kFeat) {
    const int64_t row = row0 + r;
    float z = b0;
#pragma unroll
    for (int w = 0; w < kWarps / 2; ++w) z += s_part[w][fi][r];
    if (pre) pre[row * a.preact_stride + f] = from_f32<BF16>(z);
    float y = act_value(a.act, z);
    if constexpr (GATED) {
      float u = b1;
#pragma unroll
      for (int w = 0; w < kWarps / 2; ++w) u += s_part[w][fi + 8][r];
      if (pre) pre[row * a.preact_stride + features + f] = from_f32<BF16>(u);
      y *= u;
    }
    if (res) y += to_f32<BF16>(res[row * a.residual_stride + f]);
    out[row * a.out_stride + f] = from_f32<BF16>(y);
  }
}

template <bool BF16, bool GATED> cudaError_t launch_t(const LinearArgs& a, int nt, dim3 grid, cudaStream_t st) {
  auto kern = nt == 1 ? linear_small_kernel<BF16, GATED, 1> : nt == 2 ? linear_small_kernel<BF16, GATED, 2>
            : nt == 4 ? linear_small_kernel<BF16, GATED, 4> : linear_small_kernel<BF16, GATED, 8>;
  return launch_pdl(kern, grid, dim3(kWarps * 32), 0, st, a);
}

}  // namespace

bool linear_small_supported(const LinearArgs& a) {
  const auto on16 = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0;
  };
  return a.k % 8 == 0 && on16(a.a, a.a_stride) && on16(a.b, a.b_stride) &&
         (a.groups == 1 || a.b_group_stride % 8 == 0) && (a.rows + 7) / 8 + a.groups <= 65535;
}

cudaError_t launch_linear_small(const LinearArgs& a, cudaStream_t st) {
  const bool gated = act_gated(a.act);
  // rows of a chunk: those of the mean group that has any
  const int64_t mean = a.rows / a.groups;
  const int nt = mean <= 8 ? 1 : mean <= 16 ? 2 : mean <= 32 ? 4 : 8;
  const int64_t most = (a.rows + 8 * nt - 1) / (8 * nt) + (a.offsets ? a.groups : 0);
  const int features = gated ? a.n / 2 : a.n;
  const int feat = gated ? kRows / 2 : kRows;
  const dim3 grid((features + feat - 1) / feat, static_cast<unsigned>(most < a.rows ? most : a.rows));
  return a.bf16 ? (gated ? launch_t<true, true>(a, nt, grid, st) : launch_t<true, false>(a, nt, grid, st))
                : (gated ? launch_t<false, true>(a, nt, grid, st) : launch_t<false, false>(a, nt, grid, st));
}

}  // namespace senmoe
