// linear_tc.cu -- the linear products on the 5th-generation tensor cores
// (tcgen05, accumulators in TMEM, operands by TMA).
//
// One kernel for the three products.  A tile is D[128 features, w columns]:
// the M side (128 lanes) always runs along the output's contiguous dimension
// and the N side (w <= 256 columns, a multiple of 16 issued) along its rows,
// so w follows a group's own row count and a small or ragged group costs
// MMA time in proportion to its rows:
//
//   forward  M = rows of W (K-major), N = rows of x (K-major), K = in
//   dx       M = in (W, MN-major),    N = rows of dz (K-major), K = rows of W
//   dW       M = in (x, MN-major),    N = rows of W (dz, MN-major), K = rows of the group
//
// All operands arrive by TMA as 64-element, 128-byte-swizzled boxes straight
// from the caller's tensors; a K-major box holds 64 k of each row, an MN-major
// box 64 features of 64 k rows.  Past the tensors' edges TMA fills zeros.  In
// dW the k rows after a group's last are another group's: the rows up to the
// next multiple of 16 are zeroed in shared memory (in both operands, as the
// strangers may hold infinities) and the MMAs stop there.
//
// Warp roles of a persistent CTA: warp 0 TMA producer, warp 1 MMA issuer (and
// TMEM owner; it also zeroes dW's last rows), warps 4-11 epilogue (warps 2
// and 3 only place these on the TMEM lane quarters).
// Two accumulator sets in TMEM (2 x 256 columns) let the epilogue of a tile
// run under the next tile's MMAs.  A gated pair keeps gate and up of the same
// features as two accumulators of 128 columns, so its activation needs no
// exchange between threads.
//
// Every wait is bounded (wait_or_abort): a role that gives up raises the
// CTA's abort flag and records kDevWaitTimeout, the others follow, copies in
// flight are awaited, and TMEM is freed.

#include <cuda.h>

#include "kernels.h"
#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kBK = 64;                  // k of a stage: one 128-byte line
constexpr int kBM = 128;
constexpr int kEpiWarps = 8;
constexpr int kEpiWarp0 = 4;
constexpr int kTcThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kMaxStages = 10;
constexpr uint32_t kMBytes = kBM * kBK * 2;  // one 128-feature operand tile
constexpr int kTurnStride = 36;          // 32-bit words between column pairs of a warp's turning buffer
constexpr uint32_t kRingBudget = 196608;

__device__ int g_linear_error;           // first device error of the linear kernels on this device

enum Epilogue : int { kEpiPlain = 0, kEpiAct = 1, kEpiGated = 2 };

struct TcArgs {
  LinearArgs l;
  int bn;           // columns of a tile (N side), a multiple of 16
  int box_rows;     // rows of an N-side K-major box
  int m_tiles;
  int n_tiles;      // dW: tiles along W's rows
  int stages;
  uint32_t stage_bytes, n_offset;  // a stage, and where its N operand starts
};

// ------------------------------------------------------------ PTX wrappers
// Shared-memory matrix descriptor, SWIZZLE_128B.  K-major: 8-row groups SBO =
// 1024 bytes apart (LBO unused).  MN-major: 8-k groups SBO = 1024 bytes
// apart, the next 64 features LBO = one box (64 x 128 bytes) on.
template <bool MN> __device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  constexpr uint64_t lbo = MN ? (64 * 128) >> 4 : 1, sbo = 1024 >> 4;
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (lbo << 16) | (sbo << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: D fp32, A and B fp16 (0) or bf16 (1), majors, N and M.
template <bool MN_A, bool MN_B> __device__ __forceinline__ uint32_t instr_desc(int bf16, int n, int m) {
  return (1u << 4) | (static_cast<uint32_t>(bf16) << 7) | (static_cast<uint32_t>(bf16) << 10) |
         (MN_A ? 1u << 15 : 0u) | (MN_B ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_at(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}

// ------------------------------------------------------------------ tiles
struct Tile {
  int e;        // group
  int m0;       // first feature (M side)
  int c0;       // first column: a row of x / dz, or a row of W (dW)
  int w;        // columns, 1 .. bn
  int k;        // extent of the contraction (dW: the group's rows, may be 0)
  int krow;     // dW: first row
};

template <int PROD>
__device__ __forceinline__ Tile tile_at(const TcArgs& a, const int* s_off, const int* s_pre, int idx) {
  Tile t;
  const int mt = idx % a.m_tiles, rest = idx / a.m_tiles;
  t.m0 = mt * kBM;
  if constexpr (PROD == kProdWeight) {
    t.e = rest / a.n_tiles;
    t.c0 = (rest - t.e * a.n_tiles) * a.bn;
    t.w = min(a.bn, a.l.n - t.c0);
    t.krow = s_off[t.e];
    t.k = s_off[t.e + 1] - t.krow;
  } else {
    // a group's rows in equal chunks of at most bn, so that the last one is
    // not a sliver (chunks are cheap in proportion to their width)
    t.e = group_of(s_pre, a.l.groups, rest);
    const int off = s_off[t.e], cnt = s_off[t.e + 1] - off, nch = s_pre[t.e + 1] - s_pre[t.e], j = rest - s_pre[t.e];
    const int each = ((cnt + nch - 1) / nch + 15) & ~15;
    t.c0 = off + j * each;
    t.w = min(each, cnt - j * each);
    t.k = PROD == kProdForward ? a.l.k : a.l.n;
    t.krow = 0;
  }
  return t;
}

template <int ACT> __device__ __forceinline__ void act_chunk(float (&z)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = act_value(ACT, z[i]);
}
__device__ __forceinline__ void act_chunk(int act, float (&z)[16]) {
  switch (act) {  // one uniform branch a chunk
    case kActRelu: act_chunk<kActRelu>(z); break;
    case kActSilu: case kActSwiglu: act_chunk<kActSilu>(z); break;
    case kActGelu: act_chunk<kActGelu>(z); break;
    case kActGeluTanh: case kActGeglu: act_chunk<kActGeluTanh>(z); break;
    default: break;
  }
}

// 16 columns x 32 features held one feature a lane -> rows of out.  The
// values are rounded, turned in shared memory (two columns a word), and
// leave as 16 bytes of one row a lane: lane 4p + o writes features 8o .. 8o +
// 7 of columns 2p and 2p + 1.  Rows that cannot take 16-byte stores, and a
// tile's last features, go one element at a time.
template <bool BF16>
__device__ __forceinline__ void store_chunk(const float (&v)[16], uint32_t* turn, uint16_t* out, int64_t stride, int w,
                                            int feats, bool vec, int lane) {
  // out: first row and feature of the warp's block; w columns, feats features are valid
  if (vec) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      turn[p * kTurnStride + lane] =
          uint32_t(from_f32<BF16>(v[2 * p])) | (uint32_t(from_f32<BF16>(v[2 * p + 1])) << 16);
    __syncwarp();
    const int p = lane >> 2, o = lane & 3;
    const uint4 a = *reinterpret_cast<const uint4*>(turn + p * kTurnStride + o * 8);
    const uint4 b = *reinterpret_cast<const uint4*>(turn + p * kTurnStride + o * 8 + 4);
    __syncwarp();
    uint16_t* row = out + 2 * p * stride + o * 8;
    if (8 * o + 8 <= feats) {
      if (2 * p < w)
        *reinterpret_cast<uint4*>(row) =
            make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410), __byte_perm(b.x, b.y, 0x5410),
                       __byte_perm(b.z, b.w, 0x5410));
      if (2 * p + 1 < w)
        *reinterpret_cast<uint4*>(row + stride) =
            make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632), __byte_perm(b.x, b.y, 0x7632),
                       __byte_perm(b.z, b.w, 0x7632));
    } else if (8 * o < feats) {
      const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (8 * o + i < feats && 2 * p < w) row[i] = static_cast<uint16_t>(words[i]);
        if (8 * o + i < feats && 2 * p + 1 < w) row[stride + i] = static_cast<uint16_t>(words[i] >> 16);
      }
    }
  } else if (lane < feats) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < w) out[i * stride + lane] = from_f32<BF16>(v[i]);
  }
}

template <int PROD, bool GATED, bool BF16>
__global__ void __launch_bounds__(kTcThreads, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap tm_m, const __grid_constant__ CUtensorMap tm_n,
                     const TcArgs a) {
  constexpr bool MN_M = PROD != kProdForward, MN_N = PROD == kProdWeight;
  constexpr int NACC = GATED ? 2 : 1;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kMaxStages], bar_empty[kMaxStages], bar_accfull[2], bar_accempty[2],
      bar_drain;
  __shared__ __align__(16) uint32_t s_turn[kEpiWarps][8 * kTurnStride];
  __shared__ int s_off[kMaxGroups + 1], s_pre[kMaxGroups + 1], s_tot[64];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = &g_linear_error;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* ring_ptr = smem_raw + (ring - raw);
  const int stages = a.stages;

  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_accfull[i], 1);
      mbar_init(&bar_accempty[i], kEpiWarps);
    }
    mbar_init(&bar_drain, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  // chunks of bn rows; dW has no chunks, only the groups' row ranges
  group_table(a.l.offsets, a.l.groups, a.l.rows, PROD == kProdWeight ? 1 : a.bn, s_off, s_pre, s_tot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int tiles = a.m_tiles * (PROD == kProdWeight ? a.l.groups * a.n_tiles : s_pre[a.l.groups]);
  const int grid = gridDim.x;

  if (warp == 0) {
    // ============================================================ producer
    if (lane == 0) {
      uint32_t issued = 0, parity = 0;  // by stage: loaded at least once, parity of the last load
      int st = 0, ph = 0;
      bool ok = true;
      for (int idx = blockIdx.x; idx < tiles && ok; idx += grid) {
        const Tile t = tile_at<PROD>(a, s_off, s_pre, idx);
        const int kb = (t.k + kBK - 1) / kBK;
        const int nbox = MN_N ? (t.w + 63) / 64 : (t.w + a.box_rows - 1) / a.box_rows;
        const uint32_t box_bytes = MN_N ? 64 * 128 : a.box_rows * 128;
        const uint32_t bytes = NACC * kMBytes + nbox * box_bytes;
        for (int b = 0; b < kb; ++b) {
          if (!(ok = wait_or_abort(&bar_empty[st], ph ^ 1, &s_abort, err))) break;
          const uint32_t sm = ring + st * a.stage_bytes, sn = sm + a.n_offset;
          uint64_t* full = &bar_full[st];
          mbar_arrive_expect_tx(full, bytes);
          const int k0 = t.krow + b * kBK;
          if constexpr (PROD == kProdForward) {
#pragma unroll
            for (int h = 0; h < NACC; ++h)
              tma_load_3d(sm + h * kMBytes, &tm_m, k0, t.m0 + h * (a.l.n / NACC), t.e, full);
          } else if constexpr (PROD == kProdInput) {
            tma_load_3d(sm, &tm_m, t.m0, k0, t.e, full);
            tma_load_3d(sm + 64 * 128, &tm_m, t.m0 + 64, k0, t.e, full);
          } else {
            tma_load_2d_at(sm, &tm_m, t.m0, k0, full);
            tma_load_2d_at(sm + 64 * 128, &tm_m, t.m0 + 64, k0, full);
          }
          for (int i = 0; i < nbox; ++i) {
            if constexpr (MN_N) tma_load_2d_at(sn + i * box_bytes, &tm_n, t.c0 + 64 * i, k0, full);
            else tma_load_2d_at(sn + i * box_bytes, &tm_n, k0, t.c0 + a.box_rows * i, full);
          }
          issued |= 1u << st;
          parity = (parity & ~(1u << st)) | (static_cast<uint32_t>(ph) << st);
          if (++st == stages) { st = 0; ph ^= 1; }
        }
      }
      if (!ok) {  // copies already issued: a bounded chance to land before the CTA leaves
        volatile int never = 0;
        for (int i = 0; i < stages; ++i)
          if (issued >> i & 1) wait_or_abort(&bar_full[i], parity >> i & 1, &never, nullptr);
      }
    }
  } else if (warp == 1) {
    // ========================================================== MMA issuer
    const bool leader = elect_one();
    bool ok = true;
    int st = 0, ph = 0, it = 0;
    for (int idx = blockIdx.x; idx < tiles && ok; idx += grid, ++it) {
      const Tile t = tile_at<PROD>(a, s_off, s_pre, idx);
      const int ab = it & 1, aph = (it >> 1) & 1;
      if (!(ok = __all_sync(0xffffffffu, wait_or_abort(&bar_accempty[ab], aph ^ 1, &s_abort, err)))) break;
      tc_fence_after();
      const uint32_t d = tmem + ab * 256;
      const uint32_t idesc = instr_desc<MN_M, MN_N>(a.l.bf16, (t.w + 15) & ~15, kBM);
      const int kb = (t.k + kBK - 1) / kBK;
      for (int b = 0; b < kb; ++b) {
        ok = __all_sync(0xffffffffu, wait_or_abort(&bar_full[st], ph, &s_abort, err));
        if (!ok) break;
        const int left = t.k - b * kBK;
        if (PROD == kProdWeight && left < kBK && (left & 15)) {
          // the k rows after the group's last, up to the MMAs' next multiple
          // of 16; the MMAs issued before run meanwhile
          const int line = (16 - (left & 15)) * 8, boxes = 2 + (t.w + 63) / 64;  // 16-byte pieces of a box
          unsigned char* p = ring_ptr + st * a.stage_bytes + left * 128;
          for (int q = lane; q < boxes * line; q += 32) {
            const int box = q / line, in = q - box * line;
            *reinterpret_cast<uint4*>(p + (box < 2 ? box * 8192u : a.n_offset + (box - 2) * 8192u) + in * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        tc_fence_after();
        if (leader) {
          const uint32_t sm = ring + st * a.stage_bytes, sn = sm + a.n_offset;
          const uint64_t dm = smem_desc<MN_M>(sm), dn = smem_desc<MN_N>(sn);
          const int ks = min(kBK, left + 15) >> 4;
          // 16 k: 32 bytes along a K-major line, 16 lines of an MN-major box
          for (int s = 0; s < ks; ++s) {
            const uint64_t am = dm + s * (MN_M ? 2048 >> 4 : 32 >> 4), an = dn + s * (MN_N ? 2048 >> 4 : 32 >> 4);
#pragma unroll
            for (int h = 0; h < NACC; ++h)
              umma_ss(d + h * 128, am + h * (kMBytes >> 4), an, idesc, (b | s) != 0);
          }
          umma_commit(&bar_empty[st]);
        }
        __syncwarp();
        if (++st == stages) { st = 0; ph ^= 1; }
      }
      if (ok && leader) umma_commit(&bar_accfull[ab]);
      __syncwarp();
    }
    if (leader) umma_commit(&bar_drain);  // every MMA issued has completed once this fires
    __syncwarp();
    volatile int never = 0;
    wait_or_abort(&bar_drain, 0, &never, nullptr);
  } else if (warp >= kEpiWarp0) {
    // ============================================================ epilogue
    const int ew = warp - kEpiWarp0, q = warp & 3, half = ew >> 2;
    uint32_t* turn = s_turn[ew];
    const LinearArgs& l = a.l;
    const int cols = PROD == kProdForward ? l.n / NACC : l.k;  // features of the output
    uint16_t* out = static_cast<uint16_t*>(l.out);
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (l.out_stride & 7) == 0 &&
                     (PROD != kProdWeight || (l.out_group_stride & 7) == 0);
    uint16_t* pre = static_cast<uint16_t*>(l.preact);
    const bool pvec = (reinterpret_cast<uintptr_t>(pre) & 15) == 0 && (l.preact_stride & 7) == 0 &&
                      (NACC == 1 || (cols & 7) == 0);
    int it = 0;
    for (int idx = blockIdx.x; idx < tiles; idx += grid, ++it) {
      const Tile t = tile_at<PROD>(a, s_off, s_pre, idx);
      const int ab = it & 1, aph = (it >> 1) & 1;
      if (!__all_sync(0xffffffffu, wait_or_abort(&bar_accfull[ab], aph, &s_abort, err))) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + ab * 256;
      const int f0 = t.m0 + q * 32, feats = min(32, cols - f0);  // this warp's features
      float b0 = 0.0f, b1 = 0.0f;
      if constexpr (PROD == kProdForward) {
        if (l.bias && lane < feats) {
          const uint16_t* bias = static_cast<const uint16_t*>(l.bias) + static_cast<int64_t>(t.e) * l.n + f0 + lane;
          b0 = to_f32<BF16>(*bias);
          if constexpr (GATED) b1 = to_f32<BF16>(bias[cols]);
        }
      }
      if (feats > 0) {
        for (int c = half * 16; c < t.w; c += 32) {
          const int w = min(16, t.w - c);
          uint32_t r0[16], r1[16];
          float z[16];
          if (PROD == kProdWeight && t.k == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = 0.0f;
          } else {
            tmem_ld16(acc + c, r0);
            if constexpr (GATED) tmem_ld16(acc + 128 + c, r1);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = __uint_as_float(r0[i]) + b0;
          }
          const int64_t row = t.c0 + c;
          if constexpr (PROD == kProdForward) {
            if (pre) store_chunk<BF16>(z, turn, pre + row * l.preact_stride + f0, l.preact_stride, w, feats, pvec, lane);
            act_chunk(l.act, z);
            if constexpr (GATED) {
              float u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) u[i] = __uint_as_float(r1[i]) + b1;
              if (pre)
                store_chunk<BF16>(u, turn, pre + row * l.preact_stride + cols + f0, l.preact_stride, w, feats, pvec,
                                  lane);
#pragma unroll
              for (int i = 0; i < 16; ++i) z[i] *= u[i];
            }
            if (l.residual && lane < feats) {
              const uint16_t* res = static_cast<const uint16_t*>(l.residual) + row * l.residual_stride + f0 + lane;
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (i < w) z[i] += to_f32<BF16>(res[i * l.residual_stride]);
            }
          }
          uint16_t* dst = out + row * l.out_stride + f0;
          if constexpr (PROD == kProdWeight) dst += t.e * l.out_group_stride;
          store_chunk<BF16>(z, turn, dst, l.out_stride, w, feats, vec, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_accempty[ab]);
    }
    if constexpr (PROD != kProdWeight) {
      if (l.offsets) {  // rows of no group: zero
        const int64_t head = s_off[0], tail = s_off[l.groups], n = head + (l.rows - tail);
        for (int64_t i = blockIdx.x; i < n; i += grid) {
          const int64_t r = i < head ? i : tail + (i - head);
          for (int f = tid - kEpiWarp0 * 32; f < cols; f += kEpiWarps * 32) out[r * l.out_stride + f] = 0;
          if (pre)
            for (int f = tid - kEpiWarp0 * 32; f < l.n; f += kEpiWarps * 32) pre[r * l.preact_stride + f] = 0;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------- host side
int tc_sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    n = 148;
  return n;
}

bool tma_ok(const void* p, int64_t stride, int64_t group_stride, int groups) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0 && stride < (int64_t(1) << 36) &&
         (groups <= 1 || (group_stride % 8 == 0 && group_stride < (int64_t(1) << 38)));
}

template <int PROD, bool GATED, bool BF16>
cudaError_t launch_t(const CUtensorMap& m, const CUtensorMap& n, const TcArgs& a, int grid, size_t smem,
                     cudaStream_t st) {
  auto kern = linear_tc_kernel<PROD, GATED, BF16>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(grid), dim3(kTcThreads), smem, st, m, n, a);
}

}  // namespace

bool linear_tc_supported(const LinearArgs& a, LinearProduct p) {
  const bool w_ok = p == kProdWeight ? tma_ok(a.b, a.b_stride, 0, 1) : tma_ok(a.b, a.b_stride, a.b_group_stride, a.groups);
  return a.rows > 0 && w_ok && tma_ok(a.a, a.a_stride, 0, 1);
}

cudaError_t launch_linear_tc(const LinearArgs& l, LinearProduct p, cudaStream_t st) {
  const bool gated = p == kProdForward && act_gated(l.act);
  TcArgs a{};
  a.l = l;
  const int features = p == kProdForward ? (gated ? l.n / 2 : l.n) : l.k;
  a.m_tiles = (features + kBM - 1) / kBM;
  const int bn_max = gated ? 128 : 256;
  int64_t tiles;
  if (p == kProdWeight) {
    a.bn = l.n >= 256 ? 256 : (l.n + 63) / 64 * 64;
    a.n_tiles = (l.n + a.bn - 1) / a.bn;
    tiles = static_cast<int64_t>(l.groups) * a.n_tiles * a.m_tiles;
  } else {
    // columns for the mean group with a quarter to spare
    const int64_t mean = l.rows / l.groups, want = mean + mean / 4 + 1;
    a.bn = want >= bn_max ? bn_max : want > 64 ? static_cast<int>((want + 63) / 64 * 64) : static_cast<int>((want + 15) / 16 * 16);
    a.box_rows = a.bn < 64 ? a.bn : 64;
    tiles = ((l.rows + a.bn - 1) / a.bn + (l.offsets ? l.groups : 0)) * a.m_tiles;
  }
  a.n_offset = (gated ? 2 : 1) * kMBytes;
  a.stage_bytes = a.n_offset + a.bn * 128;
  a.stages = static_cast<int>(kRingBudget / a.stage_bytes);
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  const size_t smem = 1024 + static_cast<size_t>(a.stages) * a.stage_bytes;

  // tensor maps: 16-bit patterns, 64-element boxes
  CUtensorMap tm{}, tn{};
  const auto dt = CU_TENSOR_MAP_DATA_TYPE_UINT16;
  cudaError_t e;
  if (p == kProdWeight) {
    e = make_tmap_2d(&tm, l.b, dt, l.k, l.rows, l.b_stride * 2, 64, 64, true);
    if (e == cudaSuccess) e = make_tmap_2d(&tn, l.a, dt, l.n, l.rows, l.a_stride * 2, 64, 64, true);
  } else {
    const int64_t gs = l.groups > 1 ? l.b_group_stride : l.b_stride * l.n;
    e = make_tmap_3d(&tm, l.b, dt, l.k, l.n, l.groups, l.b_stride * 2, gs * 2, 64, p == kProdForward ? kBM : 64);
    if (e == cudaSuccess)
      e = make_tmap_2d(&tn, l.a, dt, p == kProdForward ? l.k : l.n, l.rows, l.a_stride * 2, 64, a.box_rows, true);
  }
  if (e != cudaSuccess) return e;
  const int sms = tc_sm_count();
  const int grid = static_cast<int>(tiles < 1 ? 1 : tiles < sms ? tiles : sms);
#define SENMOE_LINEAR_TC(P, G)                                               \
  (l.bf16 ? launch_t<P, G, true>(tm, tn, a, grid, smem, st) : launch_t<P, G, false>(tm, tn, a, grid, smem, st))
  if (p == kProdInput) return SENMOE_LINEAR_TC(kProdInput, false);
  if (p == kProdWeight) return SENMOE_LINEAR_TC(kProdWeight, false);
  return gated ? SENMOE_LINEAR_TC(kProdForward, true) : SENMOE_LINEAR_TC(kProdForward, false);
#undef SENMOE_LINEAR_TC
}

cudaError_t linear_device_error(cudaStream_t st, int* error) {
  *error = 0;
  cudaError_t e = cudaStreamSynchronize(st);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(error, g_linear_error, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && *error) e = cudaMemcpyToSymbol(g_linear_error, &zero, sizeof(int));
  return e;
}

}  // namespace senmoe
