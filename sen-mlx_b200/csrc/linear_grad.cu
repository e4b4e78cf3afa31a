// linear_grad.cu -- the elementwise and column-sum parts of the linear
// products' backward pass.
//
// dz = dy * act'(z) (gated: dg = dy * u * act'(g), du = dy * act(g)),
// evaluated in fp32.  The bias gradient, the sum of each group's dz, is taken
// here from the fp32 values.  dz itself is rounded once to the operands' 16-bit
// type, because it is an operand of both gradient products on the 16-bit
// tensor cores.  That rounding (at most 2^-8 of the value in bf16, 2^-11 in
// fp16, whose range dz_exponent extends) is independent from element to
// element and so adds to dx and dW about as much as their own rounding does:
// 0.0023 of a gradient's norm in bf16 against 0.0017 for fp32 sums of an
// unrounded dz.  Over some 10,000 random sizes the ratio was 1.4, and up to 1.8
// where a few large elements decide (a handful of rows).  Carrying dz in two
// 16-bit parts would bring it to 1 for twice the products.

#include <type_traits>

#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLargest = 3.402823466e38f;  // finite fp32


// One row's V columns (gated: the gate's and the up's) as loaded, and dz of them.
template <bool BF16, int V, int ACT> struct Piece {
  static constexpr bool kGated = ACT >= kActSwiglu, kStore = ACT != kActNone;  // none: dz is dy
  using Raw = std::conditional_t<V == 8, uint4, uint16_t>;
  Raw y, z, u;
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[V]) {
    if constexpr (V == 8) unpack8<BF16>(v, f);
    else f[0] = to_f32<BF16>(v);
  }
  static __device__ __forceinline__ void store(uint16_t* p, const float (&f)[V]) {
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = pack8<BF16>(f);
    else *p = from_f32<BF16>(f[0]);
  }
  __device__ __forceinline__ void load(const uint16_t* dy, const uint16_t* pre, int cols) {
    y = *reinterpret_cast<const Raw*>(dy);
    if constexpr (kStore) z = *reinterpret_cast<const Raw*>(pre);
    if constexpr (kGated) u = *reinterpret_cast<const Raw*>(pre + cols);
  }
  // g: dz, or its gate half; up: its up half
  __device__ __forceinline__ void gradient(float (&g)[V], float (&up)[V]) const {
    unpack(y, g);
    if constexpr (kStore) {
      float zf[V];
      unpack(z, zf);
      if constexpr (kGated) unpack(u, up);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float value;
        const float d = g[i];
        g[i] = d * act_both(ACT, zf[i], value);
        if constexpr (kGated) {
          g[i] *= up[i];
          up[i] = d * value;
        }
      }
    }
  }
};

// dz alone.  A warp takes a piece of a row (kUnroll steps), V columns a lane
// and step: 8 (16-byte accesses) where every row starts on a 16-byte boundary,
// else 1.  The loads of kUnroll steps are in flight together.  Bound by HBM: dy and z read once, dz written once; 36 us
// for 32768 rows of 2 x 768 (252 MB, 7.0 TB/s with part of the writes still in
// L2; 82 us with a thread an element group and a division each).
template <bool BF16, int V, int ACT>
__global__ void __launch_bounds__(kThreads) dz_kernel(const LinearGradArgs a) {
  using P = Piece<BF16, V, ACT>;
  constexpr int kUnroll = V == 8 ? 3 : 1;
  pdl_wait();
  pdl_launch_dependents();
  const int cols = P::kGated ? a.n / 2 : a.n;
  const int lane = threadIdx.x & 31;
  const unsigned pieces = (cols + 32 * V * kUnroll - 1) / (32 * V * kUnroll);
  const int64_t items = a.rows * pieces, warps = gridDim.x * kWarps;
  for (int64_t it = blockIdx.x * kWarps + (threadIdx.x >> 5); it < items; it += warps) {
    const int64_t r = it < 0xffffffffll ? static_cast<unsigned>(it) / pieces : it / pieces;
    const uint16_t* dy = static_cast<const uint16_t*>(a.dy) + r * a.dy_stride;
    const uint16_t* pre = static_cast<const uint16_t*>(a.preact) + r * a.preact_stride;
    uint16_t* dz = static_cast<uint16_t*>(a.dz) + r * a.dz_stride;
    const int c0 = static_cast<int>(it - r * pieces) * 32 * V * kUnroll + lane * V;
    P piece[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (c0 + j * 32 * V < cols) piece[j].load(dy + c0 + j * 32 * V, pre + c0 + j * 32 * V, cols);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int c = c0 + j * 32 * V;
      if (c >= cols) break;
      float g[V], up[V];
      piece[j].gradient(g, up);
      P::store(dz + c, g);
      if constexpr (P::kGated) P::store(dz + cols + c, up);
    }
  }
}

// dz and its column sums; for ACT none the sums alone.  A block takes a run of
// kWarps * kRows rows and 32 * V columns, each warp kRows of the rows with all
// their loads in flight together, and the warps' fp32 sums meet in shared
// memory.  Each group's part of a run goes to slot (run + group) of `partial`:
// along the rows every new pair of run and group raises that number, so no two
// share a slot, and a group's slots follow from its offsets alone.  A dense
// product of one run goes straight to dbias (without an activation its runs
// are longer, read in turns, for a small workspace: dW mostly takes these
// sums).  The order of every sum is fixed.
//
// 57 us for 32768 rows of 2 x 768 in 128 groups, 18 for 4096 x 2112 (dz alone
// 38.5 and 11), a join kernel included; dW's launch joins the parts for
// nothing.  With a block's rows in a loop, or more than 85 registers (two
// blocks an SM), it took 72 and 20.
//
// fp16 (with or without a bias gradient): a first launch stores dz as it is and
// raises each group's dz_max to its largest finite |dz|; a second one (SCALED)
// stores the groups again that need a scale (dz_exponent).  Where none does,
// the maxima and that launch cost 3 us (333 x 2048 -> 2048 silu, 23.7 -> 26.4)
// to a tenth of the backward pass (512 rows in 128 groups, 150 -> 163).
template <bool BF16, int V, int ACT, bool SCALED>
__global__ void __launch_bounds__(kThreads, 3) dz_sums_kernel(const LinearGradArgs a) {
  using P = Piece<BF16, V, ACT>;
  constexpr int kRows = dz_run_rows(P::kGated), kRun = kRows * kWarps, kHalves = P::kGated ? 2 : 1;
  __shared__ int s_off[kMaxGroups + 1];
  __shared__ unsigned s_max[2][kWarps];
  __shared__ __align__(16) float s_sum[2][kWarps][kHalves][32 * V];
  pdl_wait();
  pdl_launch_dependents();
  const int rows = static_cast<int>(a.rows), groups = a.groups;
  const int cols = P::kGated ? a.n / 2 : a.n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col_blocks = (cols + 32 * V - 1) / (32 * V);
  const int length = P::kStore ? kRun : a.run;  // rows of a run
  const int64_t items = static_cast<int64_t>((rows + length - 1) / length) * col_blocks;
  if constexpr (SCALED) {
    int some = 0;
    for (int i = threadIdx.x; i < groups; i += kThreads) some |= dz_exponent(a.dz_max[i]);
    if (!__syncthreads_or(some)) return;
  }
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int run = static_cast<int>(it / col_blocks), cb = static_cast<int>(it - static_cast<int64_t>(run) * col_blocks);
    const int r0 = run * length, r1 = min(r0 + length, rows), mine = r0 + warp * kRows, c = (cb * 32 + lane) * V;
    const bool live = c < cols;
    P piece[kRows];
    const uint16_t* dy = static_cast<const uint16_t*>(a.dy) + mine * a.dy_stride + c;
    const uint16_t* pre = static_cast<const uint16_t*>(a.preact) + mine * a.preact_stride + c;
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (live && mine + j < r1) piece[j].load(dy + j * a.dy_stride, pre + j * a.preact_stride, cols);
    if (a.offsets && it == blockIdx.x)  // the groups, while the loads are on their way
      for (int i = threadIdx.x; i <= groups; i += kThreads) s_off[i] = min(max(a.offsets[i], 0), rows);
    // the run's parts, one a group; s_sum takes turns, so a part needs one barrier
    if (a.offsets) __syncthreads();
    int e = 0;
    if (a.offsets) {  // the last i with s_off[i] <= r0, or -1
      int lo = -1, hi = groups + 1;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_off[mid] <= r0) lo = mid;
        else hi = mid;
      }
      e = lo;
    }
    for (int from = r0, to, turn = 0; from < r1; from = to) {
      to = r1;
      if (a.offsets) {
        while (e < groups && s_off[e + 1] <= from) ++e;
        if (e < groups) to = min(r1, s_off[e + 1]);
        if (e < 0 || e >= groups) continue;  // rows of no group
      }
      float scale = 1.0f, most = 0.0f;
      if constexpr (SCALED) {
        const int x = dz_exponent(a.dz_max[e]);
        if (x == 0) continue;
        scale = power_of_two(-x);
      }
      float sum[kHalves][V] = {};
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (!live || mine + j < from || mine + j >= to) continue;
        float g[V], up[V];
        piece[j].gradient(g, up);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sum[0][i] += g[i];
          if constexpr (P::kGated) sum[1][i] += up[i];
          if constexpr (!BF16 && !SCALED) {  // (fmaxf passes NaN by)
            most = fmaxf(most, fabsf(g[i]) <= kLargest ? fabsf(g[i]) : 0.0f);
            if constexpr (P::kGated) most = fmaxf(most, fabsf(up[i]) <= kLargest ? fabsf(up[i]) : 0.0f);
          }
          if constexpr (SCALED) {
            g[i] *= scale;
            if constexpr (P::kGated) up[i] *= scale;
          }
        }
        if constexpr (P::kStore) {
          uint16_t* p = static_cast<uint16_t*>(a.dz) + (mine + j) * a.dz_stride + c;
          P::store(p, g);
          if constexpr (P::kGated) P::store(p + cols, up);
        }
      }
      if constexpr (!P::kStore) {
        for (int row = mine + kRun; row < r1 && live; row += kRun) {  // a dense run's further rows
          const int64_t at = row - mine;
          P more[kRows];
#pragma unroll
          for (int j = 0; j < kRows; ++j)
            if (row + j < r1) more[j].load(dy + (at + j) * a.dy_stride, nullptr, cols);
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            if (row + j >= r1) break;
            float g[V], up[V];
            more[j].gradient(g, up);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0][i] += g[i];
          }
        }
      }
      if constexpr (SCALED) continue;
      if constexpr (!BF16 && P::kStore) {
        const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if (lane == 0) s_max[turn][warp] = bits;
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        if (!a.dbias) break;
        if constexpr (V == 8) {
          float4* p = reinterpret_cast<float4*>(&s_sum[turn][warp][h][8 * lane]);
          p[0] = make_float4(sum[h][0], sum[h][1], sum[h][2], sum[h][3]);
          p[1] = make_float4(sum[h][4], sum[h][5], sum[h][6], sum[h][7]);
        } else {
          s_sum[turn][warp][h][lane] = sum[h][0];
        }
      }
      __syncthreads();
      if constexpr (!BF16 && P::kStore) {
        if (a.dz_max && threadIdx.x == 0) {
          unsigned bits = 0;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) bits = max(bits, s_max[turn][w]);
          atomicMax(a.dz_max + e, bits);
        }
      }
      for (int t = threadIdx.x; t < (a.dbias ? kHalves * 32 * V : 0); t += kThreads) {
        const int h = t / (32 * V), col = cb * 32 * V + t % (32 * V);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += s_sum[turn][w][h][t % (32 * V)];
        if (col >= cols) continue;
        if (a.partial) a.partial[static_cast<int64_t>(run + e) * a.n + h * cols + col] = v;
        else static_cast<uint16_t*>(a.dbias)[h * cols + col] = from_f32<BF16>(v);
      }
      turn ^= 1;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) clear_kernel(unsigned* p, int n) {
  pdl_wait();
  pdl_launch_dependents();
  for (int i = threadIdx.x; i < n; i += kThreads) p[i] = 0;
}

template <bool BF16> __global__ void __launch_bounds__(kThreads) join_kernel(const BiasJoin j) {
  pdl_wait();
  pdl_launch_dependents();
  join_bias<BF16>(j, blockIdx.x * kWarps + (threadIdx.x >> 5), gridDim.x * kWarps);
}

template <bool BF16, int V> struct Dz {
  static auto of(int act) {
    switch (act) {
      case kActRelu: return dz_kernel<BF16, V, kActRelu>;
      case kActSilu: return dz_kernel<BF16, V, kActSilu>;
      case kActGelu: return dz_kernel<BF16, V, kActGelu>;
      case kActGeluTanh: return dz_kernel<BF16, V, kActGeluTanh>;
      case kActSwiglu: return dz_kernel<BF16, V, kActSwiglu>;
      default: return dz_kernel<BF16, V, kActGeglu>;
    }
  }
};
template <bool BF16, int V> struct DzSums {
  static auto of(int act) {
    switch (act) {
      case kActRelu: return dz_sums_kernel<BF16, V, kActRelu, false>;
      case kActSilu: return dz_sums_kernel<BF16, V, kActSilu, false>;
      case kActGelu: return dz_sums_kernel<BF16, V, kActGelu, false>;
      case kActGeluTanh: return dz_sums_kernel<BF16, V, kActGeluTanh, false>;
      case kActSwiglu: return dz_sums_kernel<BF16, V, kActSwiglu, false>;
      case kActGeglu: return dz_sums_kernel<BF16, V, kActGeglu, false>;
      default: return dz_sums_kernel<BF16, V, kActNone, false>;
    }
  }
};
template <int V> auto dz_scaled(int act) {
  switch (act) {
    case kActRelu: return dz_sums_kernel<false, V, kActRelu, true>;
    case kActSilu: return dz_sums_kernel<false, V, kActSilu, true>;
    case kActGelu: return dz_sums_kernel<false, V, kActGelu, true>;
    case kActGeluTanh: return dz_sums_kernel<false, V, kActGeluTanh, true>;
    case kActSwiglu: return dz_sums_kernel<false, V, kActSwiglu, true>;
    default: return dz_sums_kernel<false, V, kActGeglu, true>;
  }
}

bool on16(const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; }

unsigned grid_for(int64_t items, int64_t cap) {
  const int64_t g = items < cap ? items : cap;
  return static_cast<unsigned>(g < 1 ? 1 : g);
}

}  // namespace

int dz_run(int64_t rows, bool grouped, int act) {
  if (act == kActNone && !grouped)  // read in turns: at most 64 runs, and one up to 512 rows
    return rows <= 512 ? 512 : rows <= 64 * 256 ? 256 : static_cast<int>((rows / 64 + 32) & ~int64_t(31));
  return kWarps * dz_run_rows(act_gated(act));
}

int64_t dz_slots(int64_t rows, int groups, bool grouped, int run) {
  if (rows == 0 || (!grouped && rows <= run)) return 0;
  return (rows + run - 1) / run + (grouped ? groups : 0);
}

template <template <bool, int> class F> static auto pick(bool bf16, bool wide, int act) {
  return bf16 ? (wide ? F<true, 8>::of(act) : F<true, 1>::of(act)) : (wide ? F<false, 8>::of(act) : F<false, 1>::of(act));
}

cudaError_t launch_dz(const LinearGradArgs& a, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  const int cols = act_gated(a.act) ? a.n / 2 : a.n;
  const bool act = a.act != kActNone;
  const bool wide = cols % 8 == 0 && on16(a.dy, a.dy_stride) &&
                    (!act || (on16(a.preact, a.preact_stride) && on16(a.dz, a.dz_stride)));
  const dim3 block(kThreads);
  if (!a.dbias && !a.dz_max) {
    const int64_t items = a.rows * ((cols + (wide ? 767 : 31)) / (wide ? 768 : 32));
    return launch_pdl(pick<Dz>(a.bf16, wide, a.act), dim3(grid_for((items + kWarps - 1) / kWarps, 148 * 16)), block, 0, st, a);
  }
  const int64_t items = (a.rows + a.run - 1) / a.run * ((cols + (wide ? 255 : 31)) / (wide ? 256 : 32));
  const dim3 grid(grid_for(items, 148 * 64));
  if (a.dz_max) {
    const cudaError_t e = launch_pdl(clear_kernel, dim3(1), block, 0, st, a.dz_max, a.groups);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = launch_pdl(pick<DzSums>(a.bf16, wide, a.act), grid, block, 0, st, a);
  if (e != cudaSuccess || !a.dz_max) return e;
  return launch_pdl(wide ? dz_scaled<8>(a.act) : dz_scaled<1>(a.act), dim3(grid_for(items, 148 * 3)), block, 0, st, a);
}

cudaError_t launch_bias_join(const BiasJoin& j, bool bf16, cudaStream_t st) {
  const int64_t warps = bias_join_items(j);
  return launch_pdl(bf16 ? join_kernel<true> : join_kernel<false>, dim3(grid_for((warps + kWarps - 1) / kWarps, 148 * 8)),
                    dim3(kThreads), 0, st, j);
}

}  // namespace senmoe
