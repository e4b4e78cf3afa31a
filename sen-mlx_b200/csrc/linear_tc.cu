// linear_tc.cu -- the linear products on the 5th-generation tensor cores
// (tcgen05, accumulators in TMEM, operands by TMA).
//
// One kernel for the three products.  A tile is D[features, w columns]: the M
// side (TMEM lanes) always runs along the output's contiguous dimension and
// the N side (w <= 256 columns) along its rows, so w follows a group's own
// row count and a small or ragged group costs MMA time in proportion to its
// rows:
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
// Three forms of a tile:
//   * one CTA: 128 features;
//   * a pair (cta_group::2): 256 features on two SMs, each holding half of
//     the M operand and half of the N operand, so a tile's operands cross L2
//     once for both;
//   * a K split: the CTAs of a cluster take shares of one tile's K and add
//     their fp32 accumulators over distributed shared memory in rank order
//     (no atomics: the same bits every time), for products with fewer tiles
//     than SMs.
// A gated pair lays 64 gate rows over the same features' 64 up rows in the
// 128 lanes; the epilogue warps of the two halves swap accumulators through
// shared memory, each finishing half of the columns.
//
// Warp roles of a persistent CTA: warp 0 TMA producer, warp 1 MMA issuer (and
// TMEM owner), warps 2-3 the bias gradient (dW), warps 4-11 epilogue.  Two
// accumulator sets in TMEM (2 x 256 columns) let the epilogue of a tile run
// under the next tile's MMAs.
//
// What bounds it, and what it measured (one B200, launches alone): large
// products stand between the tensor pipe, the operands' way from L2 (a pair's
// 256 x 256 tile asks for 64 bytes a cycle and SM of MMA time) and shared
// memory, whose bandwidth operands, TMA and the epilogue's turning share:
// 8192 x 2048 -> 8192 gelu with z kept 206 us = 1334 TFLOP/s, 78 % tensor pipe
// (153 with neither loads nor epilogue, 171 without the epilogue).  Experts'
// weights come from HBM once: 64 tokens down over 128 experts 69 us = 5.8 TB/s;
// 4096 tokens swiglu 210 us for 1.09 GB and 206 GFLOP.  dW is bound by its
// writes: 247 us for 805 MB, which a memset writes in 204.
//
// Waits.  Every wait on an mbarrier is bounded (wait_or_abort): a role that
// gives up raises the CTA's abort flag and records kDevWaitTimeout, the others
// follow, copies in flight are awaited, and TMEM is freed.  Three kinds of wait
// have no limit, and need none as long as these hold:
//   * barrier.cluster and the block's barriers: every thread arrives at each,
//     whatever its role's waits returned (a cluster's CTAs run together);
//   * the named barriers of a gated pair: its two warps first agree on whether
//     they go on (both_warps) and then take the same steps;
//   * tcgen05.alloc: only one of this package's CTAs that use TMEM fits an SM
//     at a time (one_cta_an_sm), on whichever stream, and none leaves before its TMEM is
//     free, a pair's CTAs together; and a pair asks only when both CTAs run.
// So launches on several streams wait for one another's SMs and nothing else.

#include <cuda.h>

#include <mutex>

#include "kernels.h"
#include "linear.cuh"

namespace senmoe {
namespace {

constexpr int kBK = 64;                  // k of a stage: one 128-byte line
constexpr int kEpiWarps = 8;
constexpr int kEpiWarp0 = 4;
constexpr int kTcThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kMaxStages = 10;
constexpr uint32_t kMBytes = 128 * kBK * 2;  // a CTA's M operand of a stage
constexpr uint32_t kBoxBytes = 64 * 128;     // an MN-major box: 64 features of 64 k
constexpr int kTurnStride = 36;          // 32-bit words between column pairs of a warp's turning buffer
// Dynamic shared memory: the ring, then each epilogue warp's turning buffer,
// then (gated) its half of the swap; beside them the static row-group tables
// and barriers and the ring's alignment.
constexpr uint32_t kTurnBytes = 8 * kTurnStride * 4, kSwapBytes = 16 * 32 * 4;
constexpr uint32_t kStaticBytes = 9 * 1024 + 1024;
constexpr uint32_t epilogue_bytes(bool gated) { return kEpiWarps * (kTurnBytes + (gated ? kSwapBytes : 0)); }
constexpr uint32_t ring_budget(bool gated) { return 227 * 1024 - kStaticBytes - epilogue_bytes(gated); }
constexpr int kColStep = kEpiWarps / 4 * 32;  // columns the epilogue warps take between them
// Largest K split, and how many clusters of that size are resident at once
// (of 148 SMs; cudaOccupancyMaxActiveClusters): one more would wait for a
// whole round.  Clusters of 8 (15 at once) were slower
// than 4 wherever both fit (16 rows of 2048 x 2048: 16.2 us against 8.8).
constexpr int kMaxSplit = 4, kMaxQuads = 33;
constexpr int kSumPieces = 4;  // bias gradient inside dW: most 8-column pieces of a warp

__device__ int g_linear_error;           // first device error of the linear kernels on this device
__device__ int g_linear_taken;           // what the last check found there

struct TcArgs {
  LinearArgs l;
  int bn;           // columns of a tile (N side)
  int part;         // columns of a CTA's N operand: bn, or half of it in a pair
  int m_pieces, n_pieces;  // MN-major: rows are whole 64-feature pieces (load_mn)
  int m_tiles;
  int n_tiles;      // dW: tiles along W's rows
  int stages;
  int split;        // K split (one-CTA form): the cluster's size
  uint32_t stage_bytes;  // a stage: the M operand, then the N operand
  long long tile_limit;  // of the wait for a tile's accumulators, cycles
  uint16_t* dbias;  // dW: column sums of dz, [groups, n], or null
  BiasJoin join;    // dW: the bias gradient from its parts
};

// ------------------------------------------------------------ PTX wrappers
// Shared-memory matrix descriptor, SWIZZLE_128B.  K-major: 8-row groups SBO =
// 1024 bytes apart (LBO unused).  MN-major: 8-k groups SBO = 1024 bytes
// apart, the next 64 features LBO = one box on.
template <bool MN> __device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  constexpr uint64_t lbo = MN ? kBoxBytes >> 4 : 1, sbo = 1024 >> 4;
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (lbo << 16) | (sbo << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: D fp32, A and B fp16 (0) or bf16 (1), majors, N and M.
template <bool MN_A, bool MN_B> __device__ __forceinline__ uint32_t instr_desc(int bf16, int n, int m) {
  return (1u << 4) | (static_cast<uint32_t>(bf16) << 7) | (static_cast<uint32_t>(bf16) << 10) |
         (MN_A ? 1u << 15 : 0u) | (MN_B ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on `bar` (a pair: on both CTAs' barrier at that offset) once every
// MMA this thread issued has completed.
template <bool PAIR> __device__ __forceinline__ void umma_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// All 512 columns: the ring leaves no room for a second CTA on the SM.
template <bool PAIR> __device__ __forceinline__ void tmem_alloc(uint32_t* dst) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR> __device__ __forceinline__ void tmem_free(uint32_t addr) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// TMA load of a box; PAIR: `bar` may be the other CTA's (a shared::cluster address).
template <bool PAIR>
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                       uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// An MN-major operand: `boxes` columns of 64 features from f0 on, 64 k rows
// from k0.  Where the tensor's rows are whole 64-feature pieces the map has
// these as a dimension and one load brings all (a load costs the TMA unit
// some 100 cycles beside its bytes); otherwise one load a box.
template <bool PAIR>
__device__ __forceinline__ void load_mn(uint32_t dst, const CUtensorMap* map, bool pieces, int boxes, int f0, int k0,
                                        int e, uint32_t bar) {
  if (pieces) {
    tma_4d<PAIR>(dst, map, 0, k0, f0 >> 6, e, bar);
  } else {
    for (int i = 0; i < boxes; ++i) tma_4d<PAIR>(dst + i * kBoxBytes, map, f0 + 64 * i, k0, 0, e, bar);
  }
}

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                          long long limit = kWaitLimitCycles) {
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag, err, limit));
}

// Named barrier of two warps (64 threads) that also joins a condition.
__device__ __forceinline__ bool both_warps(int id, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.aligned.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(mine ? 1u : 0u)
      : "memory");
  return r != 0;
}

// ------------------------------------------------------------------ tiles
struct Tile {
  int e;        // group
  int m0;       // this CTA's first feature
  int c0;       // first column: a row of x / dz, or a row of W (dW)
  int w;        // columns, 1 .. bn
  int n;        // columns of the MMA: w rounded up
  int kb0, kb1; // this CTA's k blocks
  int k;        // extent of the contraction (dW: the group's rows, may be 0)
  int krow;     // dW: first row
};

template <int PROD, bool GATED, bool PAIR>
__device__ __forceinline__ Tile tile_at(const TcArgs& a, const int* s_off, const int* s_pre, int idx, int rank) {
  constexpr int kFeat = GATED ? 64 : 128;
  Tile t;
  const int mt = idx % a.m_tiles, rest = idx / a.m_tiles;
  t.m0 = PAIR ? (2 * mt + rank) * kFeat : mt * kFeat;
  if constexpr (PROD == kProdWeight) {
    t.e = rest / a.n_tiles;
    t.c0 = (rest - t.e * a.n_tiles) * a.bn;
    t.w = min(a.bn, a.l.n - t.c0);
    t.n = PAIR ? (t.w + 127) & ~127 : (t.w + 15) & ~15;  // a pair: whole 64-feature boxes on each side
    t.krow = s_off[t.e];
    t.k = s_off[t.e + 1] - t.krow;
  } else {
    // a group's rows in equal chunks of at most bn, so that the last one is
    // not a sliver (a chunk costs time in proportion to its width)
    constexpr int kStep = PAIR ? 32 : 16;
    t.e = group_of(s_pre, a.l.groups, rest);
    const int off = s_off[t.e], cnt = s_off[t.e + 1] - off, nch = s_pre[t.e + 1] - s_pre[t.e], j = rest - s_pre[t.e];
    const int each = ((cnt + nch - 1) / nch + kStep - 1) & ~(kStep - 1);
    t.c0 = off + j * each;
    t.w = min(each, cnt - j * each);
    t.n = (t.w + kStep - 1) & ~(kStep - 1);
    t.k = PROD == kProdForward ? a.l.k : a.l.n;
    t.krow = 0;
  }
  const int kb = (t.k + kBK - 1) / kBK;
  t.kb0 = 0;
  t.kb1 = kb;
  if constexpr (!PAIR) {
    if (a.split > 1) {
      t.kb0 = static_cast<int>(static_cast<int64_t>(kb) * rank / a.split);
      t.kb1 = static_cast<int>(static_cast<int64_t>(kb) * (rank + 1) / a.split);
    }
  }
  return t;
}

// The lines `left` up to the next multiple of 16 of a stage's MN-major boxes
// (two of the M operand, n_boxes of the N operand behind it), one warp.
__device__ __forceinline__ void zero_rows(unsigned char* stage, int left, int n_boxes, int lane) {
  const int line = (16 - (left & 15)) * 8;  // 16-byte pieces of a box
  for (int q = lane; q < (2 + n_boxes) * line; q += 32) {
    const int box = q / line, in = q - box * line;
    *reinterpret_cast<uint4*>(stage + box * kBoxBytes + left * 128 + in * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
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
// tile's last features, go one element at a time.  w columns and feats
// features are valid (either may be 0 or less).
template <bool BF16>
__device__ __forceinline__ void store_chunk(const float (&v)[16], uint32_t* turn, uint16_t* out, int64_t stride, int w,
                                            int feats, bool vec, int lane) {
  if (vec) {
#pragma unroll
    for (int p = 0; p < 8; ++p) turn[p * kTurnStride + lane] = pack2<BF16>(v[2 * p], v[2 * p + 1]);
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

// What a warp needs to finish a tile's accumulators.
template <int PROD, bool GATED, bool BF16, bool SCALED> struct Finish {
  const LinearArgs& l;
  uint16_t *out, *pre;
  int cols;           // features of the output
  bool vec, pvec;
  uint32_t* turn;
  int lane;
  __device__ __forceinline__ Finish(const LinearArgs& args, uint32_t* t, int ln) : l(args), turn(t), lane(ln) {
    cols = PROD == kProdForward ? l.n / (GATED ? 2 : 1) : l.k;
    out = static_cast<uint16_t*>(l.out);
    pre = PROD == kProdForward ? static_cast<uint16_t*>(l.preact) : nullptr;
    vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (l.out_stride & 7) == 0 &&
          (PROD != kProdWeight || (l.out_group_stride & 7) == 0);
    pvec = (reinterpret_cast<uintptr_t>(pre) & 15) == 0 && (l.preact_stride & 7) == 0 && (!GATED || (cols & 7) == 0);
  }
  __device__ __forceinline__ float bias(int e, int f, int lanes, int up) const {
    if constexpr (PROD == kProdForward) {
      if (l.bias && lane < lanes)
        return to_f32<BF16>(static_cast<const uint16_t*>(l.bias)[static_cast<int64_t>(e) * l.n + up + f + lane]);
    }
    return 0.0f;
  }
  // dz's scale, undone in its products
  __device__ __forceinline__ float scale(int e) const {
    return SCALED ? power_of_two(dz_exponent(l.dz_max[e])) : 1.0f;
  }
  // z (bias added) of 16 columns -> preact, at column `at` of its rows
  __device__ __forceinline__ void keep(const float (&z)[16], int64_t row, int at, int w, int feats) const {
    if (PROD == kProdForward && pre)
      store_chunk<BF16>(z, turn, pre + row * l.preact_stride + at, l.preact_stride, w, feats, pvec, lane);
  }
  // the activated values, + residual (gradients: times dz's scale) -> out
  __device__ __forceinline__ void write(float (&y)[16], float scale, int e, int64_t row, int f, int w, int feats) const {
    if constexpr (PROD == kProdForward) {
      if (l.residual && lane < feats) {
        const uint16_t* res = static_cast<const uint16_t*>(l.residual) + row * l.residual_stride + f + lane;
        uint16_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = i < w ? res[i * l.residual_stride] : uint16_t(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] += to_f32<BF16>(r[i]);
      }
    }
    if constexpr (SCALED) {  // (a branch: mostly 1, and a dW of few rows is bound by its epilogue)
      if (scale != 1.0f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] *= scale;
      }
    }
    uint16_t* dst = out + row * l.out_stride + f;
    if constexpr (PROD == kProdWeight) dst += e * l.out_group_stride;
    store_chunk<BF16>(y, turn, dst, l.out_stride, w, feats, vec, lane);
  }
};

// SCALED: dx or dW of an fp16 dz stored by a power of two a group (dz_exponent).
// JOIN: dW that also joins the parts of the bias gradient.  (Instances of their
// own: in every dW's code either costs the shortest launches 2 to 4 %.)
template <int PROD, bool GATED, bool BF16, bool PAIR, bool SCALED, bool JOIN>
__global__ void __launch_bounds__(kTcThreads, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap tm_m, const __grid_constant__ CUtensorMap tm_n,
                     const __grid_constant__ CUtensorMap tm_half, const __grid_constant__ TcArgs a) {
  constexpr bool MN_M = PROD != kProdForward, MN_N = PROD == kProdWeight;
  constexpr int kCtas = PAIR ? 2 : 1;
  // dW in a pair: the second CTA's loads land on its own barrier (its warps 1
  // to 3 work on them) and its warp 1 passes each on to the leader; elsewhere
  // both CTAs' loads count on the leader's barrier
  constexpr bool kRelay = PAIR && PROD == kProdWeight;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kMaxStages], bar_empty[kMaxStages], bar_accfull[2], bar_accempty[2],
      bar_drain;
  __shared__ int s_off[kMaxGroups + 1], s_pre[kMaxGroups + 1], s_tot[64];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = &g_linear_error;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* ring_ptr = smem_raw + (ring - raw);
  const int stages = a.stages;
  unsigned char* epi_ptr = ring_ptr + stages * a.stage_bytes;
  const auto turn_of = [&](int ew) { return reinterpret_cast<uint32_t*>(epi_ptr + ew * kTurnBytes); };
  const auto swap_of = [&](int ew) { return reinterpret_cast<float*>(epi_ptr + kEpiWarps * kTurnBytes + ew * kSwapBytes); };
  const int csize = PAIR ? 2 : a.split;  // CTAs of the cluster
  const int rank = csize > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int unit = blockIdx.x / csize, units = gridDim.x / csize;
  const bool sums = PROD == kProdWeight && a.dbias != nullptr;

  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bar_full[i], kRelay && rank == 0 ? 2 : 1);
      mbar_init(&bar_empty[i], sums ? 3 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_accfull[i], 1);
      mbar_init(&bar_accempty[i], kCtas * kEpiWarps);
    }
    mbar_init(&bar_drain, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_map(&tm_m);
    prefetch_map(&tm_n);
  }
  // chunks of bn rows; dW has no chunks, only the groups' row ranges
  group_table(a.l.offsets, a.l.groups, a.l.rows, PROD == kProdWeight ? 1 : a.bn, s_off, s_pre, s_tot);
  __syncthreads();
  // the other CTAs run and their barriers exist before anything arrives on
  // them, and before a pair asks for its TMEM on both SMs
  if (csize > 1) cluster_sync();
  if (warp == 1) tmem_alloc<PAIR>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int tiles = a.m_tiles * (PROD == kProdWeight ? a.l.groups * a.n_tiles : s_pre[a.l.groups]);
  // shared by all roles: the tile's k blocks walk the ring in order
  auto next = [stages](int& st, int& ph) {
    if (++st == stages) { st = 0; ph ^= 1; }
  };

  if (warp == 0) {
    // ============================================================ producer
    if (lane == 0) {
      uint32_t issued = 0, parity = 0;  // by stage: loaded at least once, parity of the last load
      int st = 0, ph = 0;
      bool ok = true;
      for (int idx = unit; idx < tiles && ok; idx += units) {
        const Tile t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, idx, rank);
        const int part = t.n / kCtas, col = t.c0 + (PAIR ? rank * part : 0);  // this CTA's share of the columns
        // K-major columns: one load of a full part, or of half of one where that holds them
        const bool small = !MN_N && 2 * part <= a.part && a.part >= 32;
        const uint32_t bytes = kMBytes + (small ? a.part / 2 : a.part) * 128;
        for (int b = t.kb0; b < t.kb1; ++b) {
          if (!(ok = wait_or_abort(&bar_empty[st], ph ^ 1, &s_abort, err))) break;
          const uint32_t sm = ring + st * a.stage_bytes, sn = sm + kMBytes;
          uint32_t full = smem_u32(&bar_full[st]);
          if constexpr (PAIR && !kRelay) {
            if (rank == 0) mbar_arrive_expect_tx(&bar_full[st], 2 * bytes);
            full = map_rank(full, 0);
          } else {
            mbar_arrive_expect_tx(&bar_full[st], bytes);
          }
          const int k0 = t.krow + b * kBK;
          if constexpr (PROD == kProdForward) tma_4d<PAIR>(sm, &tm_m, k0, t.m0, 0, t.e, full);
          else load_mn<PAIR>(sm, &tm_m, a.m_pieces, 2, t.m0, k0, PROD == kProdInput ? t.e : 0, full);
          if constexpr (MN_N) load_mn<PAIR>(sn, &tm_n, a.n_pieces, a.part / 64, col, k0, 0, full);
          else tma_4d<PAIR>(sn, small ? &tm_half : &tm_n, k0, col, 0, 0, full);
          issued |= 1u << st;
          parity = (parity & ~(1u << st)) | (static_cast<uint32_t>(ph) << st);
          next(st, ph);
        }
      }
      // the last loads of every stage have been consumed (a pair: so no
      // arrival is still on its way when the CTA leaves)
      volatile int never = 0;
      for (int i = 0; i < stages; ++i) {
        if (!(issued >> i & 1)) continue;
        if (ok) ok = wait_or_abort(&bar_empty[i], parity >> i & 1, &s_abort, err);
        // gave up: copies already issued get a bounded chance to land
        if (!ok && (!PAIR || kRelay || rank == 0)) wait_or_abort(&bar_full[i], parity >> i & 1, &never, nullptr);
      }
    }
  } else if (warp == 1 && (!PAIR || rank == 0)) {
    // ========================================================== MMA issuer
    const bool leader = elect_one();
    bool ok = true;
    int st = 0, ph = 0, it = 0;
    for (int idx = unit; idx < tiles && ok; idx += units, ++it) {
      const Tile t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, idx, rank);
      const int ab = it & 1, aph = (it >> 1) & 1;
      if (!(ok = warp_wait(&bar_accempty[ab], aph ^ 1, &s_abort, err))) break;
      tc_fence_after();
      const uint32_t d = tmem + ab * 256;
      const uint32_t idesc = instr_desc<MN_M, MN_N>(a.l.bf16, t.n, 128 * kCtas);
      for (int b = t.kb0; b < t.kb1; ++b) {
        if (!(ok = warp_wait(&bar_full[st], ph, &s_abort, err))) break;
        const int left = t.k - b * kBK;
        if (PROD == kProdWeight && left < kBK && (left & 15))
          zero_rows(ring_ptr + st * a.stage_bytes, left, (t.n / kCtas + 63) / 64, lane);
        tc_fence_after();
        if (leader) {
          const uint32_t sm = ring + st * a.stage_bytes;
          const uint64_t dm = smem_desc<MN_M>(sm), dn = smem_desc<MN_N>(sm + kMBytes);
          const int ks = min(kBK, left + 15) >> 4;
          // 16 k: 32 bytes along a K-major line, 16 lines of an MN-major box
          for (int s = 0; s < ks; ++s)
            umma_ss<PAIR>(d, dm + s * (MN_M ? 2048 >> 4 : 32 >> 4), dn + s * (MN_N ? 2048 >> 4 : 32 >> 4), idesc,
                          (b > t.kb0 || s > 0) ? 1u : 0u);
          umma_commit<PAIR>(&bar_empty[st]);
        }
        __syncwarp();
        next(st, ph);
      }
      if (ok && leader) umma_commit<PAIR>(&bar_accfull[ab]);
      __syncwarp();
    }
    // every MMA issued has completed once this fires
    if (leader)
      umma_commit<PAIR>(&bar_drain);
    __syncwarp();
    volatile int never = 0;
    wait_or_abort(&bar_drain, 0, &never, nullptr);
  } else if (warp == 1) {
    // ====================== the pair's second CTA, dW: loads passed on
    if constexpr (kRelay) {
      bool ok = true;
      int st = 0, ph = 0;
      for (int idx = unit; idx < tiles && ok; idx += units) {
        const Tile t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, idx, rank);
        for (int b = t.kb0; b < t.kb1; ++b) {
          if (!(ok = warp_wait(&bar_full[st], ph, &s_abort, err))) break;
          const int left = t.k - b * kBK;
          if (left < kBK && (left & 15)) zero_rows(ring_ptr + st * a.stage_bytes, left, t.n / 128, lane);
          if (lane == 0) arrive_at(map_rank(smem_u32(&bar_full[st]), 0));
          next(st, ph);
        }
      }
    }
  } else if (warp < kEpiWarp0) {
    // ============================== dW: column sums of dz, the bias gradient
    // Every feature tile of a column tile loads the same dz, so the column
    // tile's 8-column pieces are dealt to its feature tiles (piece c to tile c
    // mod m_tiles) and there to these two warps: a CTA adds few columns a
    // block and keeps pace with the MMAs (one tile adding all of them took
    // three times as long as its MMAs), and no sums cross CTAs.  Lane l adds
    // rows l, l + 32, ... in fp32, then the lanes are added, all in a fixed
    // order.  (As ones times dz on the warp-level MMA the sums held up the
    // tcgen05 MMAs: 871 cycles a block of 64 rows instead of 535.)
    // With an activation the sums come from the fp32 dz, in parts, which these
    // warps join while the tiles run.
    if constexpr (PROD == kProdWeight) {
      if constexpr (JOIN) join_bias<BF16>(a.join, blockIdx.x * 2 + warp - 2, gridDim.x * 2);
      if (sums) {
        bool ok = true;
        int st = 0, ph = 0;
        for (int idx = unit; idx < tiles && ok; idx += units) {
          const Tile t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, idx, rank);
          const int part = t.n / kCtas, col = t.c0 + (PAIR ? rank * part : 0);
          const int c0 = idx % a.m_tiles + a.m_tiles * (warp - 2);  // first piece of this CTA's columns
          float acc[kSumPieces][8] = {};
          for (int b = t.kb0; b < t.kb1; ++b) {
            if (!(ok = warp_wait(&bar_full[st], ph, &s_abort, err))) break;
            const int rows = min(kBK, t.k - b * kBK);
            const unsigned char* base = ring_ptr + st * a.stage_bytes + kMBytes;
#pragma unroll
            for (int j = 0; j < kSumPieces; ++j) {
              const int c = c0 + 2 * j * a.m_tiles;
              if (8 * c >= part) break;
#pragma unroll
              for (int h = 0; h < kBK / 32; ++h) {
                const int r = 32 * h + lane;
                if (r < rows) {
                  const uint4 v = *reinterpret_cast<const uint4*>(base + (c >> 3) * kBoxBytes + r * 128 +
                                                                  (((c & 7) ^ (r & 7)) << 4));
                  const uint32_t wd[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    acc[j][2 * i] += to_f32<BF16>(static_cast<uint16_t>(wd[i]));
                    acc[j][2 * i + 1] += to_f32<BF16>(static_cast<uint16_t>(wd[i] >> 16));
                  }
                }
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_empty[st]);
            next(st, ph);
          }
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < kSumPieces; ++j) {
            const int c = c0 + 2 * j * a.m_tiles;
            if (8 * c >= part) break;
            // halves of the warp swap halves of the columns, until lane 4i has column i
            float v4[4], v2[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool up = lane & 16;
              v4[i] = (up ? acc[j][i + 4] : acc[j][i]) +
                      __shfl_xor_sync(0xffffffffu, up ? acc[j][i] : acc[j][i + 4], 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool up = lane & 8;
              v2[i] = (up ? v4[i + 2] : v4[i]) + __shfl_xor_sync(0xffffffffu, up ? v4[i] : v4[i + 2], 8);
            }
            float v = (lane & 4 ? v2[1] : v2[0]) + __shfl_xor_sync(0xffffffffu, lane & 4 ? v2[0] : v2[1], 4);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            const int n = col + 8 * c + (lane >> 2);
            if ((lane & 3) == 0 && n < a.l.n) a.dbias[static_cast<int64_t>(t.e) * a.l.n + n] = from_f32<BF16>(v);
          }
        }
      }
    }
  } else if (PAIR || a.split <= 1) {
    // ============================================================ epilogue
    // 32 columns at a time, the warps of a lane quarter in turn
    const int ew = warp - kEpiWarp0, q = warp & 3, turn2 = ew >> 2;
    const Finish<PROD, GATED, BF16, SCALED> fin(a.l, turn_of(ew), lane);
    int it = 0;
    for (int idx = unit; idx < tiles; idx += units, ++it) {
      const Tile t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, idx, rank);
      const int ab = it & 1, aph = (it >> 1) & 1;
      // a gated pair: quarters 0, 1 hold the gate of features 32 (q & 1) on, 2, 3 the up
      const int f0 = t.m0 + (GATED ? q & 1 : q) * 32, feats = min(32, fin.cols - f0);
      const int up = GATED && q >= 2 ? fin.cols : 0;
      const float bias = fin.bias(t.e, f0, feats, up), scale = fin.scale(t.e);
      bool go = warp_wait(&bar_accfull[ab], aph, &s_abort, err, a.tile_limit);
      // the two warps that swap leave together, or one would wait for the other
      if constexpr (GATED) go = both_warps(1 + (turn2 * 2 + (q & 1)), go);
      if (!go) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + ab * 256;
      const uint32_t release = PAIR ? map_rank(smem_u32(&bar_accempty[ab]), 0) : smem_u32(&bar_accempty[ab]);
      bool released = false;
      for (int c = turn2 * 32; c < t.w; c += kColStep) {
        uint32_t r[32];
        if (PROD == kProdWeight && t.k == 0) {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        } else {
          tmem_ld16(acc + c, r);
          tmem_ld16(acc + c + 16, r + 16);
          tmem_ld_wait();
        }
        if (c + kColStep >= t.w) {  // this warp's last read of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(release);
          released = true;
        }
        const int64_t row = t.c0 + c;
        float z[2][16];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i >> 4][i & 15] = __uint_as_float(r[i]) + bias;
        if constexpr (GATED) {
#pragma unroll
          for (int h = 0; h < 2; ++h) fin.keep(z[h], row + 16 * h, up + f0, t.w - c - 16 * h, feats);
          // gate warps finish columns c .. c + 15 and hand the others over, up warps the reverse
          const bool gate = q < 2;
          float* mine = swap_of(ew);
          const float* theirs = swap_of(ew ^ 2);
          const int bar = 1 + (turn2 * 2 + (q & 1));
          float y[16], u[16];
          if (gate) {
#pragma unroll
            for (int i = 0; i < 16; ++i) mine[i * 32 + lane] = z[1][i];
            asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              y[i] = z[0][i];
              u[i] = theirs[i * 32 + lane];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) mine[i * 32 + lane] = z[0][i];
            asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              y[i] = theirs[i * 32 + lane];
              u[i] = z[1][i];
            }
          }
          asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
          act_chunk(a.l.act, y);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] *= u[i];
          const int h = gate ? 0 : 16;
          fin.write(y, scale, t.e, row + h, f0, t.w - c - h, feats);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int w = t.w - c - 16 * h;
            if (w <= 0) break;
            if constexpr (PROD == kProdForward) {
              fin.keep(z[h], row + 16 * h, f0, w, feats);
              act_chunk(a.l.act, z[h]);
            }
            fin.write(z[h], scale, t.e, row + 16 * h, f0, w, feats);
          }
        }
      }
      if (!released) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(release);
      }
    }
  } else {
    // =========================== K split: this CTA's accumulator is ready
    if (unit < tiles) warp_wait(&bar_accfull[0], 0, &s_abort, err, a.tile_limit);
    tc_fence_after();
  }

  __syncwarp();
  if constexpr (!PAIR) {
    if (csize > 1) {
      // Chunks of 16 columns are dealt to the cluster's CTAs.  Every CTA sends
      // its share of a chunk to the chunk's owner, whose ring is free by then
      // (stores, so nothing waits for a trip between SMs; a warp's 32 lanes
      // are one line), and the owner adds the shares in rank order:
      // [its chunk][rank][column][lane].
      cluster_sync();
      const bool epi = warp >= kEpiWarp0 && unit < tiles;
      const int ew = warp - kEpiWarp0;
      Tile t{};
      if (epi) t = tile_at<PROD, GATED, PAIR>(a, s_off, s_pre, unit, rank);
      const int chunks = (t.w + 15) / 16;
      if (epi) {
        const int q = warp & 3;
        const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
        for (int c = ew >> 2; c < chunks; c += kEpiWarps / 4) {
          uint32_t r[16];
          if (t.kb1 > t.kb0) {
            tmem_ld16(acc + 16 * c, r);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = 0;
          }
          const uint32_t dst =
              map_rank(ring + (((c / csize) * csize + rank) * 16 * 128 + q * 32 + lane) * 4, c % csize);
#pragma unroll
          for (int i = 0; i < 16; ++i) st_cluster(dst + i * 512, r[i]);
        }
        tc_fence_before();
      }
      __syncwarp();
      cluster_sync();  // every share is where it is added
      if (epi) {
        const Finish<PROD, GATED, BF16, SCALED> fin(a.l, turn_of(ew), lane);
        const float scale = fin.scale(t.e);
        constexpr int kQuarters = GATED ? 2 : 4;
        const int mine = chunks > rank ? (chunks - rank + csize - 1) / csize : 0;  // chunks rank, rank + csize, ...
        for (int i = ew; i < mine * kQuarters; i += kEpiWarps) {
          const int q = i % kQuarters, slot = i / kQuarters, c = (slot * csize + rank) * 16, w = t.w - c;
          const int f0 = t.m0 + q * 32, feats = min(32, fin.cols - f0);
          const float b0 = fin.bias(t.e, f0, feats, 0), b1 = GATED ? fin.bias(t.e, f0, feats, fin.cols) : 0.0f;
          const float* src = reinterpret_cast<const float*>(ring_ptr) + slot * csize * 16 * 128 + q * 32 + lane;
          float z[16], u[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float v = 0.0f, v2 = 0.0f;
#pragma unroll
            for (int r = 0; r < kMaxSplit; ++r) {
              if (r < csize) {
                v += src[(r * 16 + k) * 128];
                if constexpr (GATED) v2 += src[(r * 16 + k) * 128 + 64];
              }
            }
            z[k] = v + b0;
            u[k] = v2 + b1;
          }
          if constexpr (PROD == kProdForward) {
            const int64_t row = t.c0 + c;
            fin.keep(z, row, f0, w, feats);
            if constexpr (GATED) fin.keep(u, row, fin.cols + f0, w, feats);
            act_chunk(a.l.act, z);
            if constexpr (GATED) {
#pragma unroll
              for (int k = 0; k < 16; ++k) z[k] *= u[k];
            }
          }
          fin.write(z, scale, t.e, t.c0 + c, f0, w, feats);
        }
      }
      __syncwarp();
    }
  }
  if constexpr (PROD != kProdWeight) {
    if (a.l.offsets && warp >= kEpiWarp0) {  // rows of no group: zero
      const LinearArgs& l = a.l;
      uint16_t *out = static_cast<uint16_t*>(l.out), *pre = static_cast<uint16_t*>(l.preact);
      const int cols = PROD == kProdForward ? l.n / (GATED ? 2 : 1) : l.k;
      const int64_t head = s_off[0], tail = s_off[l.groups], n = head + (l.rows - tail);
      for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t r = i < head ? i : tail + (i - head);
        for (int f = tid - kEpiWarp0 * 32; f < cols; f += kEpiWarps * 32) out[r * l.out_stride + f] = 0;
        if (PROD == kProdForward && pre)
          for (int f = tid - kEpiWarp0 * 32; f < l.n; f += kEpiWarps * 32) pre[r * l.preact_stride + f] = 0;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR && rank == 1 && warp == 1) {
    // The leader's drain commit arrives here too.  Waited for only now, with
    // this CTA's tiles finished, so that the limit does not run from the
    // kernel's start and a long kernel's CTA cannot leave before the arrival.
    volatile int never = 0;
    wait_or_abort(&bar_drain, 0, &never, nullptr);
    __syncwarp();
  }
  if (csize > 1) cluster_sync();  // nobody reads this CTA's shared memory or TMEM any more
  if (warp == 1) {
    tc_fence_after();
    tmem_free<PAIR>(tmem);
  }
  // A pair frees its TMEM together: neither CTA leaves before both have, or
  // the SM of the first could take another kernel's CTA, and its allocation,
  // with the pair's still half undone.
  __syncwarp();
  if constexpr (PAIR) cluster_sync();
}

// Reads and clears in one step: an error that a kernel on another stream
// records meanwhile is this check's or the next one's.
__global__ void take_error_kernel() { g_linear_taken = atomicExch(&g_linear_error, 0); }

// A wait that nothing ends, through its limit.
__global__ void selftest_wait_kernel() {
  __shared__ __align__(8) uint64_t bar;
  __shared__ volatile int abort_flag;
  mbar_init(&bar, 1);
  fence_mbar_init();
  abort_flag = 0;
  wait_or_abort(&bar, 0, &abort_flag, &g_linear_error);
}

// ------------------------------------------------------------- host side
int tc_sm_count() {
  static int counts[64] = {};  // by device; the same value whoever writes it
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && counts[dev] > 0) return counts[dev];
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  if (dev < 64) counts[dev] = n;
  return n;
}

bool tma_ok(const void* p, int64_t stride, int64_t group_stride, int groups) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0 && stride < (int64_t(1) << 36) &&
         (groups <= 1 || (group_stride % 8 == 0 && group_stride < (int64_t(1) << 38)));
}

// Stages of the ring, as many as fit.
constexpr uint32_t stage_bytes_for(int part) { return kMBytes + part * 128; }
constexpr int stages_for(bool gated, int part) {
  const int fit = static_cast<int>(ring_budget(gated) / stage_bytes_for(part));
  return fit < kMaxStages ? fit : kMaxStages;
}
constexpr size_t tc_smem(bool gated, int part) {
  return 1024 + static_cast<size_t>(stages_for(gated, part)) * stage_bytes_for(part) + epilogue_bytes(gated);
}
// More than half an SM, and more than the quantized experts' tcgen05 kernels
// (169 KB at least) leave: no two CTAs that use TMEM share one.
constexpr bool one_cta_an_sm() {
  for (int part = 16; part <= 256; part += 16)
    if (tc_smem(false, part) < 120 * 1024 || tc_smem(true, part) < 120 * 1024) return false;
  return true;
}
static_assert(one_cta_an_sm(), "tcgen05.alloc would wait for the CTA beside");

template <int PROD, bool GATED, bool BF16, bool PAIR, bool SCALED, bool JOIN>
cudaError_t launch_t(const CUtensorMap& m, const CUtensorMap& n, const CUtensorMap& half, const TcArgs& a, int grid, size_t smem,
                     cudaStream_t st) {
  auto kern = linear_tc_kernel<PROD, GATED, BF16, PAIR, SCALED, JOIN>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  // Launched in plain stream order, unlike the other kernels here: this one
  // takes the whole SM, TMEM included, so a dependent started early would gain
  // nothing but a place to wait in.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR || a.split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, m, n, half, a);
}

template <bool PAIR, typename... A>
cudaError_t launch_prod(LinearProduct p, bool gated, const LinearArgs& l, bool join, const A&... args) {
#define SENMOE_LINEAR_TC(P, G, S, J) \
  (l.bf16 ? launch_t<P, G, true, PAIR, false, J>(args...) : launch_t<P, G, false, PAIR, S, J>(args...))
  if (p == kProdInput) return l.dz_max ? SENMOE_LINEAR_TC(kProdInput, false, true, false) : SENMOE_LINEAR_TC(kProdInput, false, false, false);
  if (p == kProdWeight && join) return SENMOE_LINEAR_TC(kProdWeight, false, true, true);  // (an fp16 dz with parts has scales)
  if (p == kProdWeight) return l.dz_max ? SENMOE_LINEAR_TC(kProdWeight, false, true, false) : SENMOE_LINEAR_TC(kProdWeight, false, false, false);
  return gated ? SENMOE_LINEAR_TC(kProdForward, true, false, false) : SENMOE_LINEAR_TC(kProdForward, false, false, false);
#undef SENMOE_LINEAR_TC
}

// The form of a product's tiles and its estimated time in SM cycles.
struct Plan {
  bool pair = false;
  int bn = 16, split = 1;
  int64_t tiles = 0;
  double cycles = 0;
};

// Estimate of one form.  A k block of 64 costs the larger of its MMAs (8
// cycles a 16-column step and K step of 16) and its operands' way from L2
// (kL2Bytes a cycle and SM); tiles run in waves over the SMs.  A K split adds
// a cluster's barriers and its shares' way between SMs.
constexpr double kL2Bytes = 57, kTileCycles = 900, kSplitCycles = 2000, kSplitColumn = 20;

Plan make_plan(const LinearArgs& l, LinearProduct p, bool gated, int sms, bool pair, int bn, int split) {
  Plan q;
  q.pair = pair;
  q.bn = bn;
  q.split = split;
  const int features = p == kProdForward ? (gated ? l.n / 2 : l.n) : l.k;
  const int feat = (gated ? 64 : 128) * (pair ? 2 : 1);
  const int64_t m_tiles = (features + feat - 1) / feat;
  const double mean = static_cast<double>(l.rows) / l.groups;
  double k, chunks, width;
  if (p == kProdWeight) {
    k = mean;
    chunks = static_cast<double>(l.groups) * ((l.n + bn - 1) / bn);
    width = l.n < bn ? l.n : bn;
    q.tiles = static_cast<int64_t>(chunks) * m_tiles;
  } else {
    k = p == kProdForward ? l.k : l.n;
    // no group has more chunks than rows
    const int64_t upper = (l.rows + bn - 1) / bn + (l.offsets ? l.groups : 0);
    q.tiles = (upper < l.rows ? upper : l.rows) * m_tiles;
    if (l.offsets) {  // counts spread about the mean: a group near a multiple of bn takes one chunk more half the time
      const double used = mean < 1 ? l.rows : l.groups;  // groups with rows, about
      chunks = used * (mean < 1 ? 1.0 : static_cast<int64_t>(mean / bn + 0.5) < 1 ? 1.0 : mean / bn + 0.5);
      width = mean < 1 ? 1 : l.rows / chunks;
    } else {
      chunks = static_cast<double>((l.rows + bn - 1) / bn);
      width = l.rows / chunks;
    }
  }
  const int step = pair ? (p == kProdWeight ? 128 : 32) : 16;
  const double n = (static_cast<int64_t>(width + step - 1) / step) * step;
  const double blocks = (k + kBK - 1) / kBK;
  const double mma = 2.0 * n > 128 ? 2.0 * n : 128, load = 128.0 * (128 + (pair ? n / 2 : n)) / kL2Bytes;
  const double per = mma > load ? mma : load;
  const double slots = static_cast<double>(sms / ((pair ? 2 : 1) * split));
  double waves = chunks * m_tiles / slots;
  waves = waves < 8 ? static_cast<double>(static_cast<int64_t>(waves + 0.999)) : waves;
  q.cycles = waves * (blocks / split * per + kTileCycles) + (split > 1 ? kSplitCycles + kSplitColumn * n : 0);
  return q;
}

// form: kFormAuto, or the only form to consider.
Plan choose_plan(const LinearArgs& l, LinearProduct p, bool gated, int sms, int form) {
  static const int kWidths[] = {16, 32, 64, 96, 128, 160, 192, 224, 256};  // dW: whole 64-feature boxes
  Plan best;
  const int64_t rows = p == kProdWeight ? l.n : l.rows;
  for (int w : kWidths) {
    if (p == kProdWeight && w % 64 != 0) continue;
    for (int pair = 0; pair < 2; ++pair) {
      // a pair's CTAs hold at least 32 columns each, in dW two 64-feature boxes
      if (pair && (w < 64 || (p == kProdWeight && w < 256))) continue;
      if (form == (pair ? kFormOne : kFormPair)) continue;
      const Plan q = make_plan(l, p, gated, sms, pair, w, 1);
      if (form != kFormSplit && (best.cycles == 0 || q.cycles < best.cycles)) best = q;
      if (pair || form == kFormOne) continue;
      for (int s = 2; s <= kMaxSplit; s *= 2) {
        if (q.tiles > (s == 2 ? sms / 2 : kMaxQuads * sms / 148)) break;
        const Plan t = make_plan(l, p, gated, sms, false, w, s);
        if (best.cycles == 0 || t.cycles < best.cycles) best = t;
      }
    }
    if (w >= rows && best.cycles > 0) break;
  }
  return best;
}

}  // namespace

bool linear_tc_supported(const LinearArgs& a, LinearProduct p) {
  const bool w_ok = p == kProdWeight ? tma_ok(a.b, a.b_stride, 0, 1) : tma_ok(a.b, a.b_stride, a.b_group_stride, a.groups);
  return a.rows > 0 && w_ok && tma_ok(a.a, a.a_stride, 0, 1);
}

cudaError_t launch_linear_tc(const LinearArgs& l, LinearProduct p, int form, const BiasJoin* bias, bool* summed,
                             cudaStream_t st) {
  const bool gated = p == kProdForward && act_gated(l.act);
  const int sms = tc_sm_count();
  const Plan plan = choose_plan(l, p, gated, sms, form);
  if (plan.cycles == 0) return cudaErrorNotSupported;  // too many tiles for the K split asked for
  TcArgs a{};
  a.l = l;
  a.bn = plan.bn;
  a.split = plan.split;
  const int features = p == kProdForward ? (gated ? l.n / 2 : l.n) : l.k;
  const int feat = (gated ? 64 : 128) * (plan.pair ? 2 : 1);
  a.m_tiles = (features + feat - 1) / feat;
  if (bias && bias->partial) {
    a.join = *bias;
    *summed = true;
  } else if (bias && plan.split == 1 && a.m_tiles * 2 * kSumPieces * 8 >= (plan.pair ? a.bn / 2 : a.bn)) {
    // (a K split leaves each CTA part of a column's rows: no sums there)
    a.dbias = static_cast<uint16_t*>(bias->dbias);
    *summed = true;
  }
  a.n_tiles = p == kProdWeight ? (l.n + a.bn - 1) / a.bn : 0;
  a.part = plan.pair ? a.bn / 2 : a.bn;
  a.stage_bytes = stage_bytes_for(a.part);
  // a k block takes some 600 cycles; dW: a group may hold every row
  const int64_t k = p == kProdForward ? l.k : p == kProdInput ? l.n : l.rows;
  a.tile_limit = kWaitLimitCycles + 2048ll * ((k + kBK - 1) / kBK);
  a.stages = stages_for(gated, a.part);
  const int csize = plan.pair ? 2 : plan.split, most = sms / csize;
  const int grid = static_cast<int>(plan.tiles < 1 ? 1 : plan.tiles < most ? plan.tiles : most) * csize;
  const size_t smem = tc_smem(gated, a.part);

  CUtensorMap tm{}, tn{}, half{};
  cudaError_t e;
  // the M operand: W (forward, dx) or x (dW); the N operand: x, dz
  const uint64_t b_row = l.b_stride * 2, a_row = l.a_stride * 2;
  if (p == kProdForward) {
    const uint64_t n = gated ? l.n / 2 : l.n, gs = l.groups > 1 ? l.b_group_stride * 2 : b_row * l.n;
    e = make_tmap_4d(&tm, l.b, {uint64_t(l.k), n, gated ? 2u : 1u, uint64_t(l.groups)}, {b_row, n * b_row, gs},
                     {64, gated ? 64u : 128u, gated ? 2u : 1u, 1});
  } else {
    const uint64_t rows = p == kProdInput ? l.n : l.rows, groups = p == kProdInput ? l.groups : 1;
    const uint64_t gs = groups > 1 ? l.b_group_stride * 2 : b_row * rows;
    a.m_pieces = l.k % 64 == 0;
    e = a.m_pieces ? make_tmap_4d(&tm, l.b, {64, rows, uint64_t(l.k / 64), groups}, {b_row, 128, gs}, {64, 64, 2, 1})
                   : make_tmap_4d(&tm, l.b, {uint64_t(l.k), rows, 1, groups}, {b_row, b_row, gs}, {64, 64, 1, 1});
  }
  if (e != cudaSuccess) return e;
  const uint64_t rows = l.rows;
  if (p == kProdWeight) {
    a.n_pieces = l.n % 64 == 0;
    e = a.n_pieces ? make_tmap_4d(&tn, l.a, {64, rows, uint64_t(l.n / 64), 1}, {a_row, 128, a_row},
                                  {64, 64, uint32_t(a.part / 64), 1})
                   : make_tmap_4d(&tn, l.a, {uint64_t(l.n), rows, 1, 1}, {a_row, a_row, a_row}, {64, 64, 1, 1});
    half = tn;
  } else {
    const uint64_t cols = p == kProdForward ? l.k : l.n;
    e = make_tmap_4d(&tn, l.a, {cols, rows, 1, 1}, {a_row, a_row, a_row}, {64, uint32_t(a.part), 1, 1});
    half = tn;
    if (e == cudaSuccess && a.part >= 32)
      e = make_tmap_4d(&half, l.a, {cols, rows, 1, 1}, {a_row, a_row, a_row}, {64, uint32_t(a.part / 2), 1, 1});
  }
  if (e != cudaSuccess) return e;
  return plan.pair ? launch_prod<true>(p, gated, l, a.join.partial, tm, tn, half, a, grid, smem, st)
                   : launch_prod<false>(p, gated, l, a.join.partial, tm, tn, half, a, grid, smem, st);
}

cudaError_t selftest_linear_wait(cudaStream_t st) {
  return cudaLaunchKernel(reinterpret_cast<const void*>(selftest_wait_kernel), dim3(1), dim3(1), nullptr, 0, st);
}

cudaError_t linear_device_error(cudaStream_t st, int* error) {
  static std::mutex once;  // g_linear_taken is one word a device
  const std::lock_guard<std::mutex> hold(once);
  *error = 0;
  cudaError_t e = cudaLaunchKernel(reinterpret_cast<const void*>(take_error_kernel), dim3(1), dim3(1), nullptr, 0, st);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(error, g_linear_taken, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  const cudaError_t done = cudaStreamSynchronize(st);
  return e != cudaSuccess ? e : done;
}

}  // namespace senmoe
