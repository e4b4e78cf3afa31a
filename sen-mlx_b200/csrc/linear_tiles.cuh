// linear_tiles.cuh -- what the tcgen05 kernels of the linear products share,
// over 16-bit and over 8-bit operands: the sizes of a CTA, PTX wrappers, and
// the way of 16 accumulator columns into rows of the output.
#pragma once

#include <cuda.h>

#include "kernels.h"
#include "linear.cuh"

namespace senmoe {

constexpr int kEpiWarps = 8;
constexpr int kEpiWarp0 = 4;
constexpr int kTcThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kMaxStages = 10;
constexpr uint32_t kBoxBytes = 64 * 128;     // an MN-major box: 64 features of 64 k
constexpr int kTurnStride = 36;          // 32-bit words between column pairs of a warp's turning buffer
constexpr uint32_t kTurnBytes = 8 * kTurnStride * 4, kSwapBytes = 16 * 32 * 4;
constexpr int kColStep = kEpiWarps / 4 * 32;  // columns the epilogue warps take between them
// Largest K split, and how many clusters of that size are resident at once
// (of 148 SMs; cudaOccupancyMaxActiveClusters): one more would wait for a
// whole round.  Clusters of 8 (15 at once) were slower
// than 4 wherever both fit (16 rows of 2048 x 2048: 16.2 us against 8.8).
constexpr int kMaxSplit = 4, kMaxQuads = 33;

// ------------------------------------------------------------ PTX wrappers
// Shared-memory matrix descriptor, SWIZZLE_128B.  K-major: 8-row groups SBO =
// 1024 bytes apart (LBO unused).  MN-major: 8-k groups SBO = 1024 bytes
// apart, the next 64 features LBO = one box on.
template <bool MN> __device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  constexpr uint64_t lbo = MN ? kBoxBytes >> 4 : 1, sbo = 1024 >> 4;
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (lbo << 16) | (sbo << 32) | (1ull << 46) | (2ull << 61);
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

// ---------------------------------------------------------------- epilogue
template <int ACT, bool FINE> __device__ __forceinline__ void act_chunk(float (&z)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = act_value<FINE>(ACT, z[i]);
}
template <bool FINE = false> __device__ __forceinline__ void act_chunk(int act, float (&z)[16]) {
  switch (act) {  // one uniform branch a chunk
    case kActRelu: act_chunk<kActRelu, FINE>(z); break;
    case kActSilu: case kActSwiglu: act_chunk<kActSilu, FINE>(z); break;
    case kActGelu: act_chunk<kActGelu, FINE>(z); break;
    case kActGeluTanh: case kActGeglu: act_chunk<kActGeluTanh, FINE>(z); break;
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

}  // namespace senmoe
