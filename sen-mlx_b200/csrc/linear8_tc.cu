// linear8_tc.cu -- the products over 8-bit rows on the 5th-generation tensor
// cores: tcgen05.mma kind::mxf8f6f4 with block scales, accumulators in TMEM.
//
// A tile is D[features, w columns] as in linear_tc.cu: M (TMEM lanes) runs
// along W's rows, N (w <= 224 columns) along the rows of x, so that a ragged
// group costs MMA time in proportion to its rows.  A stage holds 256 k: the
// operands as 128-byte-swizzled boxes by TMA, one byte an element, and their
// scales, 8 bytes a row.  The tensor core multiplies by the scales itself:
//
//   D += sum over blocks b of 32 k:  2^(sw[m, b] + sx[n, b])  sum_k W[m, k] x[n, k]
//
// with fp32 sums.  It reads the scales from TMEM, where row r of an operand is
// lane r mod 32 (the same in each quarter of the lanes) and column r / 32, the
// four bytes of a word being four consecutive blocks.  Six warps bring them
// there: the words of rows l, l + 32, l + 64, l + 96 of 128 rows, laid side by
// side, are the 16 bytes that tcgen05.cp 32x128b wants for lane l, and the MMA
// warp issues the copies ahead of the MMAs.  Copies and MMAs of one thread run
// in order; two sets of scale columns alternate all the same, so that a copy
// need not wait for the MMAs before it.
//
// Forms of a tile: one CTA (128 features), a pair (cta_group::2, 256 features
// on two SMs, each holding half of the columns' codes and all of their
// scales), or a K split over a cluster; gated pairs lay 64 gate rows over the
// same features' 64 up rows.  Waits are bounded, and those without a limit
// need none, as in linear_tc.cu.
//
// 8-bit output: a warp's 32 lanes are 32 consecutive features, one block of a
// row of y, which is finished where it stands (store_chunk8).
//
// What bounds it, and what it measured (one B200, a graph of launches on cold
// inputs): power first, as SM clocks fall to 1.2 to 1.6 GHz under it, and shared
// memory, which takes an 8-bit tile's bytes in half of a 16-bit tile's MMA time.
// 8192 x 2048 -> 8192 gelu 144 us = 1900 TFLOP/s (110 without the epilogue, 131
// without the scales, 89 without either), 50 % tensor pipe.  4096 tokens of 128
// experts, 2048 -> 2 x 768 swiglu to 8 bits with z kept, 140 to 160 us for 0.61 GB
// and 206 GFLOP; in pairs of 160 columns the groups, 256 rows on average, are two
// chunks or three, each with its trip of W from L2.
//
// The sums round towards zero: z is off by 1.5e-7 of its root mean square at K
// 2816 and smaller by 1.1e-7 on average, where fp32 products are off by 0.7e-7.

#include <cuda.h>

#include <cmath>

#include "kernels.h"
#include "linear8.cuh"
#include "linear_tiles.cuh"

namespace senmoe {
namespace {

// k of a stage: two pieces of one 128-byte line.  (With one piece a stage took
// 480 cycles in its barriers alone, whatever its bytes and MMAs.)
constexpr int kPiece = 128, kPieces = 2, kBK8 = kPiece * kPieces;
constexpr uint32_t kMPiece = 128 * kPiece;     // a piece of a CTA's M operand
constexpr int kMaxWidth = 224;                 // columns of a tile: two accumulators and two sets of scales in 512
constexpr uint32_t kAccColumn = 256;           // from one accumulator to the other
constexpr uint32_t kScaleColumn = 240;         // of the scales, behind each accumulator
constexpr uint32_t kAtomBytes = 512;           // 128 rows' scales of a piece
constexpr uint32_t kPieceScales = 3 * kAtomBytes;  // W's rows, then up to 256 columns
constexpr uint32_t kScaleBytes = kPieces * kPieceScales;
// Scales on their way: units of two stages, 16 bytes a row, 128 rows three times.
constexpr int kUnits = 2;
constexpr uint32_t kUnitAtom = 128 * 16, kUnitBytes = kUnits * 3 * kUnitAtom;  // [unit][W, columns 0-127, 128 on][row]
// Warps: 0 the loads, 1 the MMAs, 2 to 7 the scales, the others the epilogue.
// With 8 epilogue warps, two a scheduler, it waited for its own latencies
// (8192 rows of 2048 -> 8192 gelu 200 us); with 2 warps for the scales, whose
// gathered loads take 200 cycles an instruction, the MMAs waited for them.  20
// warps leave 96 registers a thread, one more would leave 80.
constexpr int kScaleWarp0 = 2, kScaleWarps = 6, kEpi0 = kScaleWarp0 + kScaleWarps;
constexpr int kEpi8 = 12, kThreads8 = (kEpi0 + kEpi8) * 32;
static_assert(kEpi0 % 4 == 0);  // an epilogue warp's number gives its quarter of the lanes
// An epilogue warp's shared memory: 16 columns of 32 features in fp32 where a
// gated pair swaps them or 8 bits are made of them, else a turning buffer.
constexpr uint32_t epi_stride(bool words) { return words ? kSwapBytes : kTurnBytes; }
static_assert(kSwapBytes == 16 * 32 * 4 && kSwapBytes >= kTurnBytes);
constexpr int kTileCache = 64;  // of a CTA's tiles in shared memory
constexpr uint32_t kStaticBytes8 = kTileCache * 32 + 1024 + 1024;  // tiles and barriers; the ring's alignment
constexpr uint32_t table_bytes(int groups) { return (2 * (groups + 1) * 4 + 15) & ~15; }  // row groups' offsets and chunks
constexpr uint32_t epilogue_bytes8(bool words) { return kEpi8 * epi_stride(words); }
constexpr uint32_t ring_budget8(bool words, int groups) {
  return 227 * 1024 - kStaticBytes8 - table_bytes(groups) - epilogue_bytes8(words) - kUnitBytes;
}

__device__ int g_linear8_error;  // first device error of these kernels on this device

constexpr int kScaleMap = 0;     // see Tc8Args

struct Tc8Args {
  Linear8Args l;
  int bn, part;          // columns of a tile, and of a CTA's N operand (half of it in a pair)
  int m_tiles, stages, split;
  uint32_t stage_bytes;  // a stage's operands: W's pieces, then the columns'
  int pieces;            // rows are whole pieces, which the maps have as a dimension
  int w_load, x_load;    // bytes of a scale row in one copy: 8, 4, or 1 (rows on no grid); kScaleMap: by TMA
  long long tile_limit;  // of the wait for a tile's accumulators, cycles
};

// Instruction descriptor, block-scaled 8-bit kinds: e4m3 x e4m3 (0, 0), both
// K-major, N / 8 from bit 17, scales in e8m0 (bit 23), M / 128 from bit 27.
// The byte of a scale word that an MMA of 32 k takes is in bits 4 (B) and 29 (A).
__device__ __forceinline__ uint32_t instr_desc8(int n, int m) {
  return (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27);
}
template <bool PAIR>
__device__ __forceinline__ void umma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                            uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 bytes at saddr -> 4 TMEM columns, the same in every quarter of
// the lanes.  Unswizzled descriptor: 8-row groups 128 bytes apart.
template <bool PAIR> __device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// TMA load of a box of a 5-d map; PAIR: `bar` may be the other CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4,
                                       uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
        : "memory");
}
// Both pieces of stage b of an operand, its rows from `row` on.  Rows of whole
// pieces: one load (a piece past the last is zeros).  Otherwise two, as the map
// must know where a row ends.
template <bool PAIR>
__device__ __forceinline__ void load_stage(uint32_t dst, uint32_t piece_bytes, const CUtensorMap* map, bool pieces,
                                           int b, int row, int e, uint32_t bar) {
  if (pieces) {
    tma_5d<PAIR>(dst, map, 0, row, 0, b * kPieces, e, bar);
  } else {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)  // (the maps count pairs of elements)
      tma_5d<PAIR>(dst + i * piece_bytes, map, (b * kPieces + i) * (kPiece / 2), row, 0, 0, e, bar);
  }
}

// TMA load of scale rows into this CTA's shared memory.
__device__ __forceinline__ void tma_scales(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// ------------------------------------------------------------------ tiles
struct __align__(16) Tile8 {
  int e;         // group
  int m0;        // this CTA's first feature
  int c0, w, n;  // first column (a row of x), columns, columns of the MMA
  int kb0, kb1;  // this CTA's k blocks
  int unused;
};

template <bool GATED, bool PAIR>
__device__ __forceinline__ Tile8 find_tile8(const Tc8Args& a, const int* s_off, const int* s_pre, int idx, int rank) {
  constexpr int kFeat = GATED ? 64 : 128, kStep = PAIR ? 32 : 16;
  Tile8 t;
  const int mt = idx % a.m_tiles, rest = idx / a.m_tiles;
  t.m0 = PAIR ? (2 * mt + rank) * kFeat : mt * kFeat;
  // a group's rows in equal chunks of at most bn
  t.e = group_of(s_pre, a.l.groups, rest);
  const int off = s_off[t.e], cnt = s_off[t.e + 1] - off, nch = s_pre[t.e + 1] - s_pre[t.e], j = rest - s_pre[t.e];
  const int each = ((cnt + nch - 1) / nch + kStep - 1) & ~(kStep - 1);
  t.c0 = off + j * each;
  t.w = min(each, cnt - j * each);
  t.n = (t.w + kStep - 1) & ~(kStep - 1);
  const int kb = (a.l.k + kBK8 - 1) / kBK8;
  t.kb0 = 0;
  t.kb1 = kb;
  if constexpr (!PAIR) {
    if (a.split > 1) {
      const KRange r = k_share(kb, rank, a.split);
      t.kb0 = r.begin;
      t.kb1 = r.end;
    }
  }
  return t;
}

// The 16 scales from p on, of which `have` are in the row, into shared memory
// with `load` bytes a copy; those of rows on no grid (1) are there at once.  What
// lies past the row is of no meaning: no MMA takes it.
__device__ __forceinline__ void fetch_scales(unsigned char* dst, const uint8_t* p, int have, int load,
                                             const uint8_t* begin, const uint8_t* end) {
  if (load == 8) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      if (i < have) cp_async_8(smem_u32(dst + i), p + i);
  } else if (load == 4) {
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      if (i < have) cp_async_4(smem_u32(dst + i), p + i);
  } else {
    uint32_t w[4];
    scale_words<4>(p, have, begin, end, w);
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---------------------------------------------------------------- epilogue
// 16 columns x 32 features, a feature a lane -> 8 bits: each column's 32
// values are one block of a row of y.  They are turned in shared memory (16-byte
// pieces of a column in an order of its own, against bank conflicts), after
// which a lane has 16 features of a column.  (With a warp reduction a column the
// block's largest cost three times the instructions.)
__device__ __forceinline__ void store_chunk8(const float (&v)[16], uint32_t* turn, uint8_t* codes, int64_t stride,
                                             uint8_t* scales, int64_t scales_stride, int w, int lane) {
  float* t = reinterpret_cast<float*>(turn);
#pragma unroll
  for (int i = 0; i < 16; ++i) t[i * 32 + ((lane >> 2) ^ (i & 7)) * 4 + (lane & 3)] = v[i];
  __syncwarp();
  const int c = lane >> 1, half = lane & 1;
  float f[16];
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float4 q = *reinterpret_cast<const float4*>(t + c * 32 + ((half * 4 + k) ^ (c & 7)) * 4);
    f[4 * k] = q.x; f[4 * k + 1] = q.y; f[4 * k + 2] = q.z; f[4 * k + 3] = q.w;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, magnitude(f[i]));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const uint32_t byte = scale_byte(m);
  const float inv = scale_inverse(byte);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = to_e4m3x2(f[2 * i] * inv, f[2 * i + 1] * inv);
  if (c < w) {
    *reinterpret_cast<uint4*>(codes + c * stride + half * 16) =
        make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    if (half == 0) scales[c * scales_stride] = static_cast<uint8_t>(byte);
  }
}

// What a warp needs to finish a tile's accumulators.
template <bool GATED, bool BF16, bool EIGHT> struct Finish8 {
  const Linear8Args& l;
  uint16_t *out, *pre;
  int cols;  // features of the output
  bool vec, pvec;
  uint32_t* turn;
  int lane;
  __device__ __forceinline__ Finish8(const Linear8Args& args, uint32_t* t, int ln) : l(args), turn(t), lane(ln) {
    cols = l.n / (GATED ? 2 : 1);
    out = static_cast<uint16_t*>(l.y);
    pre = static_cast<uint16_t*>(l.preact);
    vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (l.y_stride & 7) == 0;
    pvec = (reinterpret_cast<uintptr_t>(pre) & 15) == 0 && (l.preact_stride & 7) == 0 && (!GATED || (cols & 7) == 0);
  }
  __device__ __forceinline__ float bias(int e, int f, int lanes, int up) const {
    if (l.bias && lane < lanes)
      return to_f32<BF16>(static_cast<const uint16_t*>(l.bias)[static_cast<int64_t>(e) * l.n + up + f + lane]);
    return 0.0f;
  }
  // z (bias added) of 16 columns -> preact, at column `at` of its rows
  __device__ __forceinline__ void keep(const float (&z)[16], int64_t row, int at, int w, int feats) const {
    if (pre) store_chunk<BF16>(z, turn, pre + row * l.preact_stride + at, l.preact_stride, w, feats, pvec, lane);
  }
  // the activated values, + residual -> y
  __device__ __forceinline__ void write(float (&y)[16], int64_t row, int f, int w, int feats) const {
    if (l.residual && lane < feats) {
      const uint16_t* res = static_cast<const uint16_t*>(l.residual) + row * l.residual_stride + f + lane;
      uint16_t r[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = i < w ? res[i * l.residual_stride] : uint16_t(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] += to_f32<BF16>(r[i]);
    }
    if constexpr (EIGHT) {
      if (feats > 0)  // whole blocks: 32 features or none
        store_chunk8(y, turn, l.codes + row * l.codes_stride + f, l.codes_stride,
                     l.scales + row * l.scales_stride + f / kBlock8, l.scales_stride, w, lane);
    } else {
      store_chunk<BF16>(y, turn, out + row * l.y_stride + f, l.y_stride, w, feats, vec, lane);
    }
  }
};

template <bool GATED, bool BF16, bool PAIR, bool EIGHT>
__global__ void __launch_bounds__(kThreads8, 1)
    linear8_tc_kernel(const __grid_constant__ CUtensorMap tm_m, const __grid_constant__ CUtensorMap tm_n,
                      const __grid_constant__ CUtensorMap tm_half, const __grid_constant__ CUtensorMap tm_sw,
                      const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ Tc8Args a) {
  constexpr int kCtas = PAIR ? 2 : 1;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kMaxStages], bar_empty[kMaxStages], bar_accfull[2], bar_accempty[2],
      bar_ufull[2][kUnits], bar_uempty[2][kUnits], bar_drain;
  __shared__ int s_tot[64];
  __shared__ Tile8 s_tile[kTileCache];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = &g_linear8_error;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* ring_ptr = smem_raw + (ring - raw);
  const int stages = a.stages;
  const uint32_t scale_base = ring + stages * a.stage_bytes;  // [stage][W's rows, columns 0-127, columns 128 on]
  unsigned char* scale_ptr = ring_ptr + stages * a.stage_bytes;
  unsigned char* unit_ptr = scale_ptr + stages * kScaleBytes;
  unsigned char* epi_ptr = unit_ptr + kUnitBytes;
  int* const s_off = reinterpret_cast<int*>(epi_ptr + epilogue_bytes8(GATED || EIGHT));
  int* const s_pre = s_off + a.l.groups + 1;
  // (a warp turns its chunk after the swap, when its partner has read)
  const auto turn_of = [&](int ew) { return reinterpret_cast<uint32_t*>(epi_ptr + ew * epi_stride(GATED || EIGHT)); };
  const auto swap_of = [&](int ew) { return reinterpret_cast<float*>(turn_of(ew)); };
  const int csize = PAIR ? 2 : a.split;  // CTAs of the cluster
  const int rank = csize > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int unit = blockIdx.x / csize, units = gridDim.x / csize;

  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bar_full[i], 1 + kScaleWarps * kCtas);  // the loads, and the scale warps of both CTAs
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_accfull[i], 1);
      mbar_init(&bar_accempty[i], kCtas * kEpi8);
    }
    for (int i = 0; i < kUnits; ++i) {  // W's scales, the columns'
      mbar_init(&bar_ufull[0][i], 1);
      mbar_init(&bar_ufull[1][i], 1);
      mbar_init(&bar_uempty[0][i], 2);
      mbar_init(&bar_uempty[1][i], 4);
    }
    mbar_init(&bar_drain, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_map(&tm_m);
    prefetch_map(&tm_n);
  }
  group_table(a.l.offsets, a.l.groups, a.l.rows, a.bn, s_off, s_pre, s_tot);
  __syncthreads();
  // the other CTAs run and their barriers exist before anything arrives on
  // them, and before a pair asks for its TMEM on both SMs
  if (csize > 1) cluster_sync();
  if (warp == 1) tmem_alloc<PAIR>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int tiles = a.m_tiles * s_pre[a.l.groups];
  // The CTA's first tiles, found by a thread each: a search and three divisions
  // that every role would otherwise make for itself, between a tile and the next.
  if (tid < kTileCache && unit + tid * units < tiles)
    s_tile[tid] = find_tile8<GATED, PAIR>(a, s_off, s_pre, unit + tid * units, rank);
  __syncthreads();
  const int mine = unit < tiles ? (tiles - unit + units - 1) / units : 0;
  const auto tile = [&](int it) {
    return it < kTileCache ? s_tile[it] : find_tile8<GATED, PAIR>(a, s_off, s_pre, unit + it * units, rank);
  };
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
      for (int it = 0; it < mine && ok; ++it) {
        const Tile8 t = tile(it);
        const int part = t.n / kCtas, col = t.c0 + (PAIR ? rank * part : 0);  // this CTA's share of the columns
        // one load of a full part, or of half of one where that holds the columns
        const bool small = 2 * part <= a.part && a.part >= 32;
        const uint32_t n_piece = (small ? a.part / 2 : a.part) * kPiece, bytes = kPieces * (kMPiece + n_piece);
        for (int b = t.kb0; b < t.kb1; ++b) {
          if (!(ok = wait_or_abort(&bar_empty[st], ph ^ 1, &s_abort, err))) break;
          const uint32_t sm = ring + st * a.stage_bytes, sn = sm + kPieces * kMPiece;
          uint32_t full = smem_u32(&bar_full[st]);
          if constexpr (PAIR) {
            if (rank == 0) mbar_arrive_expect_tx(&bar_full[st], 2 * bytes);
            full = map_rank(full, 0);
          } else {
            mbar_arrive_expect_tx(&bar_full[st], bytes);
          }
          load_stage<PAIR>(sm, kMPiece, &tm_m, a.pieces, b, t.m0, t.e, full);
          load_stage<PAIR>(sn, n_piece, small ? &tm_half : &tm_n, a.pieces, b, col, 0, full);
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
        if (!ok && (!PAIR || rank == 0)) wait_or_abort(&bar_full[i], parity >> i & 1, &never, nullptr);
      }
    }
  } else if (warp == 1 && (!PAIR || rank == 0)) {
    // ========================================================== MMA issuer
    const bool leader = elect_one();
    bool ok = true;
    int st = 0, ph = 0;
    for (int it = 0; it < mine && ok; ++it) {
      const Tile8 t = tile(it);
      const int ab = it & 1, aph = (it >> 1) & 1;
      if (!(ok = warp_wait(&bar_accempty[ab], aph ^ 1, &s_abort, err))) break;
      tc_fence_after();
      const uint32_t d = tmem + ab * kAccColumn;
      const uint32_t idesc = instr_desc8(t.n, 128 * kCtas);
      const int part = t.n / kCtas;
      const uint32_t n_piece = (2 * part <= a.part && a.part >= 32 ? a.part / 2 : a.part) * kPiece;  // as loaded
      for (int b = t.kb0; b < t.kb1; ++b) {
        if (!(ok = warp_wait(&bar_full[st], ph, &s_abort, err))) break;
        tc_fence_after();
        if (leader) {
          const uint32_t sm = ring + st * a.stage_bytes, sn = sm + kPieces * kMPiece, sc = scale_base + st * kScaleBytes;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int ks = min(kPiece, a.l.k - (b * kPieces + i) * kPiece) / kBlock8;
            if (ks <= 0) break;
            const uint32_t sa = tmem + kScaleColumn + i * kAccColumn, sb = sa + 4;
            copy_scales<PAIR>(sa, sc + i * kPieceScales);
            copy_scales<PAIR>(sb, sc + i * kPieceScales + kAtomBytes);
            if (t.n > 128) copy_scales<PAIR>(sb + 4, sc + i * kPieceScales + 2 * kAtomBytes);
            const uint64_t dm = smem_desc<false>(sm + i * kMPiece), dn = smem_desc<false>(sn + i * n_piece);
#pragma unroll
            for (int s = 0; s < kPiece / kBlock8; ++s) {  // 32 k: 32 bytes along a line
              if (s < ks)
                umma_scaled<PAIR>(d, dm + s * (32 >> 4), dn + s * (32 >> 4), idesc | (s << 4) | (s << 29), sa, sb,
                                  (b > t.kb0 || i > 0 || s > 0) ? 1u : 0u);
            }
          }
          umma_commit<PAIR>(&bar_empty[st]);
        }
        __syncwarp();
        next(st, ph);
      }
      if (ok && leader) umma_commit<PAIR>(&bar_accfull[ab]);
      __syncwarp();
    }
    // every MMA issued has completed once this fires
    if (leader) umma_commit<PAIR>(&bar_drain);
    __syncwarp();
    volatile int never = 0;
    wait_or_abort(&bar_drain, 0, &never, nullptr);
  } else if (warp >= kScaleWarp0 && warp < kEpi0) {
    // ============================================================== scales
    // Half of an atom a warp (atom: W's 128 rows, the first 128 columns, the
    // others).  Rows come as 16 bytes, two stages' worth, one such unit ahead
    // (also of the next tile): by TMA where their strides allow a map,
    // else each lane its two rows with cp.async.  With each stage a lane lays
    // its rows' words side by side to where tcgen05.cp takes them.
    const Linear8Args& l = a.l;
    const int blocks = l.k / kBlock8, cap = static_cast<int>(l.rows) - 1;
    const int atom = (warp - kScaleWarp0) >> 1, half = (warp - kScaleWarp0) & 1, side = atom > 0;
    const bool maps = side ? a.x_load == kScaleMap : a.w_load == kScaleMap;
    const bool lead = lane == 0 && (warp == kScaleWarp0 || warp == kScaleWarp0 + 2);  // issues a side's loads
    const auto place = [&](int slot, int i) {
      return unit_ptr + (slot * 3 + atom) * kUnitAtom + ((half * 2 + i) * 32 + lane) * 16;
    };
    const auto some = [&](const Tile8& t) { return atom < 2 || t.n > 128; };
    // all scales of a side, for rows on no grid
    const uint8_t* const begin = side ? l.x_scales : l.w_scales;
    const uint8_t* const end = side ? begin + cap * l.x_scales_stride + blocks
                                    : begin + (l.groups - 1) * l.w_scales_group_stride + (l.n - 1) * l.w_scales_stride + blocks;
    bool ok = true;
    Tile8 f{};               // the tile being fetched
    const uint8_t* p[2];     // cp.async: this lane's rows of it
    int f_it = -1, f_unit = 0, f_end = 0, f_count = 0;
    const auto fetch = [&]() {  // the next unit, if there is one
      while (f_unit >= f_end && f_it < mine) {
        if (++f_it == mine) break;
        f = tile(f_it);
        const KRange u = scale_units(f.kb0, f.kb1);
        f_unit = u.begin;
        f_end = u.end;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // past the last row, that one: no result is of it
          const int r = (half * 2 + i) * 32 + lane;
          if (atom == 0) {
            const int up = GATED ? l.n / 2 : l.n, row = min(GATED ? f.m0 + (r & 63) : f.m0 + r, up - 1) + (GATED && r >= 64 ? up : 0);
            p[i] = l.w_scales + f.e * l.w_scales_group_stride + row * l.w_scales_stride;
          } else {
            p[i] = l.x_scales + static_cast<int64_t>(min(f.c0 + (atom - 1) * 128 + r, cap)) * l.x_scales_stride;
          }
        }
      }
      if (f_it < mine) {
        const int slot = f_count % kUnits, at = f_unit * 16;
        if (!maps) {
          if (some(f)) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              fetch_scales(place(slot, i), p[i] + at, blocks - at, side ? a.x_load : a.w_load, begin, end);
          }
        } else if (lead && ok) {
          uint64_t* full = &bar_ufull[side][slot];
          ok = wait_or_abort(&bar_uempty[side][slot], (f_count / kUnits & 1) ^ 1, &s_abort, err);
          if (ok) {
            unsigned char* dst = unit_ptr + (slot * 3 + side) * kUnitAtom;
            mbar_arrive_expect_tx(full, side ? a.bn * 16 : kUnitAtom);
            if (side) tma_scales(dst, &tm_sx, at, f.c0, 0, 0, full);
            else tma_scales(dst, &tm_sw, at, f.m0, 0, f.e, full);
          }
        }
        ++f_unit;
        ++f_count;
      }
      if (!maps) asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kUnits - 1; ++i) fetch();
    int st = 0, ph = 0, count = -1;
    for (int it = 0; it < mine && ok; ++it) {
      const Tile8 t = tile(it);
      const bool used = some(t);
      for (int b = t.kb0; b < t.kb1; ++b) {
        const bool first = b == t.kb0 || b % 2 == 0, last = b + 1 == t.kb1 || b % 2 == 1;  // of a unit
        if (first) {
          ++count;
          fetch();
          if (!maps) asm volatile("cp.async.wait_group %0;" ::"n"(kUnits - 1) : "memory");
          else ok = warp_wait(&bar_ufull[side][count % kUnits], count / kUnits & 1, &s_abort, err) && __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        // a stage's scales of the two rows
        const uint2 v0 = *reinterpret_cast<const uint2*>(place(count % kUnits, 0) + b % 2 * 8);
        const uint2 v1 = *reinterpret_cast<const uint2*>(place(count % kUnits, 1) + b % 2 * 8);
        if (last && maps) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_uempty[side][count % kUnits]);
        }
        if (!(ok = warp_wait(&bar_empty[st], ph ^ 1, &s_abort, err))) break;
        if (used) {
          unsigned char* dst = scale_ptr + st * kScaleBytes + atom * kAtomBytes + lane * 16 + half * 8;
          *reinterpret_cast<uint2*>(dst) = make_uint2(v0.x, v1.x);
          *reinterpret_cast<uint2*>(dst + kPieceScales) = make_uint2(v0.y, v1.y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        // (to the other CTA too with the plain arrive: what it guards is this
        // SM's shared memory, which the proxy fence has ordered; with
        // .release.cluster a stage took 1600 cycles)
        if (lane == 0) arrive_at(PAIR ? map_rank(smem_u32(&bar_full[st]), 0) : smem_u32(&bar_full[st]));
        next(st, ph);
      }
    }
    if (!maps) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (lead && maps) {  // every load issued has landed (after giving up: gets a bounded chance to)
      volatile int never = 0;
      for (int i = max(count, 0); i < f_count; ++i) wait_or_abort(&bar_ufull[side][i % kUnits], i / kUnits & 1, &never, nullptr);
    }
  } else if (warp >= kEpi0 && (PAIR || a.split <= 1)) {
    // ============================================================ epilogue
    // 16 columns at a time (gated: 32), the warps of a lane quarter in turn
    constexpr int kChunk = GATED ? 32 : 16, kStep = kEpi8 / 4 * kChunk;
    const int ew = warp - kEpi0, q = warp & 3, turn2 = ew >> 2;
    const Finish8<GATED, BF16, EIGHT> fin(a.l, turn_of(ew), lane);
    for (int it = 0; it < mine; ++it) {
      const Tile8 t = tile(it);
      const int ab = it & 1, aph = (it >> 1) & 1;
      // a gated pair: quarters 0, 1 hold the gate of features 32 (q & 1) on, 2, 3 the up
      const int f0 = t.m0 + (GATED ? q & 1 : q) * 32, feats = min(32, fin.cols - f0);
      const int up = GATED && q >= 2 ? fin.cols : 0;
      const float bias = fin.bias(t.e, f0, feats, up);
      bool go = warp_wait(&bar_accfull[ab], aph, &s_abort, err, a.tile_limit);
      // the two warps that swap leave together, or one would wait for the other
      if constexpr (GATED) go = both_warps(1 + (turn2 * 2 + (q & 1)), go);
      if (!go) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + ab * kAccColumn;
      const uint32_t release = PAIR ? map_rank(smem_u32(&bar_accempty[ab]), 0) : smem_u32(&bar_accempty[ab]);
      bool released = false;
      for (int c = turn2 * kChunk; c < t.w; c += kStep) {
        uint32_t r[kChunk];
        tmem_ld16(acc + c, r);
        if constexpr (GATED) tmem_ld16(acc + c + 16, r + 16);
        tmem_ld_wait();
        if (c + kStep >= t.w) {  // this warp's last read of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(release);
          released = true;
        }
        const int64_t row = t.c0 + c;
        float z[kChunk / 16][16];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) z[i >> 4][i & 15] = __uint_as_float(r[i]) + bias;
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
          act_chunk<EIGHT>(a.l.act, y);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] *= u[i];
          const int h = gate ? 0 : 16;
          fin.write(y, row + h, f0, t.w - c - h, feats);
        } else {
          fin.keep(z[0], row, f0, t.w - c, feats);
          act_chunk<EIGHT>(a.l.act, z[0]);
          fin.write(z[0], row, f0, t.w - c, feats);
        }
      }
      if (!released) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(release);
      }
    }
  } else if (warp >= kEpi0) {
    // =========================== K split: this CTA's accumulator is ready
    if (mine > 0) warp_wait(&bar_accfull[0], 0, &s_abort, err, a.tile_limit);
    tc_fence_after();
  }

  __syncwarp();
  if constexpr (!PAIR) {
    if (csize > 1) {
      // Chunks of 16 columns are dealt to the cluster's CTAs; every CTA sends
      // its share of a chunk to the chunk's owner, whose ring is free by then,
      // and the owner adds the shares in rank order: [its chunk][rank][column][lane].
      cluster_sync();
      const bool epi = warp >= kEpi0 && mine > 0;
      const int ew = warp - kEpi0;
      Tile8 t{};
      if (epi) t = tile(0);
      const int chunks = (t.w + 15) / 16;
      if (epi) {
        const int q = warp & 3;
        const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
        for (int c = ew >> 2; c < chunks; c += kEpi8 / 4) {
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
        const Finish8<GATED, BF16, EIGHT> fin(a.l, turn_of(ew), lane);
        constexpr int kQuarters = GATED ? 2 : 4;
        const int mine = chunks > rank ? (chunks - rank + csize - 1) / csize : 0;  // chunks rank, rank + csize, ...
        for (int i = ew; i < mine * kQuarters; i += kEpi8) {
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
          const int64_t row = t.c0 + c;
          fin.keep(z, row, f0, w, feats);
          if constexpr (GATED) fin.keep(u, row, fin.cols + f0, w, feats);
          act_chunk<EIGHT>(a.l.act, z);
          if constexpr (GATED) {
#pragma unroll
            for (int k = 0; k < 16; ++k) z[k] *= u[k];
          }
          fin.write(z, row, f0, w, feats);
        }
      }
      __syncwarp();
    }
  }
  if (a.l.offsets && warp >= kEpi0) {  // rows of no group: zero
    const Linear8Args& l = a.l;
    uint16_t *out = static_cast<uint16_t*>(l.y), *pre = static_cast<uint16_t*>(l.preact);
    const int cols = l.n / (GATED ? 2 : 1), first = tid - kEpi0 * 32;
    const int64_t head = s_off[0], tail = s_off[l.groups], n = head + (l.rows - tail);
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
      const int64_t r = i < head ? i : tail + (i - head);
      if constexpr (EIGHT) {
        for (int f = first; f < cols; f += kEpi8 * 32) l.codes[r * l.codes_stride + f] = 0;
        for (int f = first; f < cols / kBlock8; f += kEpi8 * 32) l.scales[r * l.scales_stride + f] = 0;
      } else {
        for (int f = first; f < cols; f += kEpi8 * 32) out[r * l.y_stride + f] = 0;
      }
      if (pre)
        for (int f = first; f < l.n; f += kEpi8 * 32) pre[r * l.preact_stride + f] = 0;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR && rank == 1 && warp == 1) {
    // The leader's drain commit arrives here too: waited for with this CTA's
    // tiles finished, so that the limit does not run from the kernel's start.
    volatile int never = 0;
    wait_or_abort(&bar_drain, 0, &never, nullptr);
    __syncwarp();
  }
  if (csize > 1) cluster_sync();  // nobody reads this CTA's shared memory or TMEM any more
  if (warp == 1) {
    tc_fence_after();
    tmem_free<PAIR>(tmem);
  }
  // A pair frees its TMEM together, see linear_tc.cu.
  __syncwarp();
  if constexpr (PAIR) cluster_sync();
}

// ------------------------------------------------------------- host side
constexpr uint32_t stage_bytes8(int part) { return kPieces * (kMPiece + part * kPiece); }
constexpr int stages8(bool words, int part, int groups) {
  const int fit = static_cast<int>(ring_budget8(words, groups) / (stage_bytes8(part) + kScaleBytes));
  return fit < kMaxStages ? fit : kMaxStages;
}
constexpr size_t smem8(bool words, int part, int groups) {
  return 1024 + static_cast<size_t>(stages8(words, part, groups)) * (stage_bytes8(part) + kScaleBytes) + kUnitBytes +
         epilogue_bytes8(words) + table_bytes(groups);
}
// As in linear_tc.cu: no two CTAs that use TMEM share an SM.  (Forms with less than two stages are not taken.)
constexpr bool one_cta_an_sm8() {
  for (int part = 16; part <= kMaxWidth; part += 16)
    for (int groups : {1, kMaxGroups})
      for (bool words : {false, true})
        if (stages8(words, part, groups) >= 2 && smem8(words, part, groups) < 120 * 1024) return false;
  return true;
}
static_assert(one_cta_an_sm8(), "tcgen05.alloc would wait for the CTA beside");

// Bytes of scale rows that one load may take: the rows' alignment allows it,
// and rows are whole loads, so that none passes the last row's end.
int scale_load(const void* p, int64_t stride, int64_t group_stride, int k) {
  for (int n = 16; n > 2; n /= 2)
    if (reinterpret_cast<uintptr_t>(p) % n == 0 && stride % n == 0 && group_stride % n == 0 &&
        k / kBlock8 % n == 0)
      return n;
  return 1;
}

struct Maps8 {
  CUtensorMap w, x, half, sw, sx;
};

template <bool GATED, bool BF16, bool PAIR, bool EIGHT>
cudaError_t launch_t(const Maps8& m, const Tc8Args& a, int grid, size_t smem, cudaStream_t st) {
  auto kern = linear8_tc_kernel<GATED, BF16, PAIR, EIGHT>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  // in plain stream order: the kernel takes the whole SM, TMEM included
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads8);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR || a.split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, m.w, m.x, m.half, m.sw, m.sx, a);
}

// The form of a product's tiles and its estimated time in SM cycles.
struct Plan8 {
  bool pair = false;
  int bn = 16, split = 1;
  int64_t tiles = 0;
  double cycles = 0;
};

// As in linear_tc.cu, with a k block of 256: the bytes and MMA cycles of 128 16-bit k.
// A K split pays from K about 4096 on: 16 rows of 8192 -> 2048 20.0 us without,
// 12.5 over four CTAs; 64 rows of 2048 -> 2048 9.4 without, 10.1 over four.
constexpr double kL2Bytes8 = 57, kTileCycles8 = 900, kSplitCycles8 = 6500, kSplitColumn8 = 20;

Plan8 make_plan8(const Linear8Args& l, bool gated, int sms, bool pair, int bn, int split) {
  Plan8 q;
  q.pair = pair;
  q.bn = bn;
  q.split = split;
  const int features = gated ? l.n / 2 : l.n, feat = (gated ? 64 : 128) * (pair ? 2 : 1);
  const int64_t m_tiles = (features + feat - 1) / feat;
  const double mean = static_cast<double>(l.rows) / l.groups;
  // no group has more chunks than rows
  const int64_t upper = (l.rows + bn - 1) / bn + (l.offsets ? l.groups : 0);
  q.tiles = (upper < l.rows ? upper : l.rows) * m_tiles;
  double chunks = static_cast<double>((l.rows + bn - 1) / bn), width = l.rows / chunks;
  if (l.offsets) {
    if (mean < 1) {  // groups with rows, about
      chunks = static_cast<double>(l.rows);
    } else {
      // Counts spread about the mean as random routing's do: a chunk more for each
      // multiple of bn below a count.  Multiples 8 sd below the mean are below every
      // count; where the spread is wider than bn, the mean of that many is as below to
      // 2^-28 (both keep the host's time the same for any rows).
      const double sd = std::sqrt(mean);
      double each = mean / bn + 0.5;
      if (sd < bn) {
        const double sure = mean > 8 * sd + bn ? std::floor((mean - 8 * sd) / bn) : 0.0;
        each = 1.0 + sure;
        for (double at = (sure + 1) * bn; at < mean + 4 * sd; at += bn) each += 0.5 * std::erfc((at - mean) / (1.4142136 * sd));
      }
      chunks = each * l.groups;
    }
    width = l.rows / chunks;
  }
  const int step = pair ? 32 : 16;
  const double n = (static_cast<int64_t>(width + step - 1) / step) * step;
  const double blocks = static_cast<double>((l.k + kPiece - 1) / kPiece) / kPieces;
  const double mma = kPieces * (2.0 * n > 128 ? 2.0 * n : 128);
  const double loaded = 2 * n <= bn && bn >= 32 ? bn / 2 : bn;  // columns: a whole box, or half of one
  const double load = kBK8 * (128 + (pair ? loaded / 2 : loaded)) / kL2Bytes8;
  const double per = mma > load ? mma : load;
  const double slots = static_cast<double>(sms / ((pair ? 2 : 1) * split));
  double waves = chunks * m_tiles / slots;
  waves = waves < 8 ? static_cast<double>(static_cast<int64_t>(waves + 0.999)) : waves;
  q.cycles = waves * (blocks / split * per + kTileCycles8) + (split > 1 ? kSplitCycles8 + kSplitColumn8 * n : 0);
  return q;
}

// form: kFormAuto, or the only form to consider.
Plan8 choose_plan8(const Linear8Args& l, bool gated, int sms, int form) {
  static const int kWidths[] = {16, 32, 64, 96, 128, 160, 192, 224};
  Plan8 best;
  for (int w : kWidths) {
    for (int pair = 0; pair < 2; ++pair) {
      if (pair && w < 64) continue;  // a pair's CTAs hold at least 32 columns each
      if (stages8(gated || l.codes, pair ? w / 2 : w, l.groups) < 2) continue;
      if (form == (pair ? kFormOne : kFormPair)) continue;
      const Plan8 q = make_plan8(l, gated, sms, pair, w, 1);
      if (form != kFormSplit && (best.cycles == 0 || q.cycles < best.cycles)) best = q;
      if (pair || form == kFormOne) continue;
      for (int s = 2; s <= kMaxSplit; s *= 2) {
        if (q.tiles > (s == 2 ? sms / 2 : kMaxQuads * sms / 148)) break;
        const Plan8 t = make_plan8(l, gated, sms, false, w, s);
        if (best.cycles == 0 || t.cycles < best.cycles) best = t;
      }
    }
    if (w >= l.rows && best.cycles > 0) break;
  }
  return best;
}

template <bool PAIR, bool EIGHT, typename... A>
cudaError_t launch_form(bool gated, bool bf16, const A&... args) {
  if (gated) return bf16 ? launch_t<true, true, PAIR, EIGHT>(args...) : launch_t<true, false, PAIR, EIGHT>(args...);
  return bf16 ? launch_t<false, true, PAIR, EIGHT>(args...) : launch_t<false, false, PAIR, EIGHT>(args...);
}

}  // namespace

cudaError_t launch_linear8_tc(const Linear8Args& l, int form, cudaStream_t st) {
  const bool gated = act_gated(l.act);
  const int sms = sm_count();
  const Plan8 plan = choose_plan8(l, gated, sms, form);
  if (plan.cycles == 0) return cudaErrorNotSupported;  // too many tiles for the K split asked for
  Tc8Args a{};
  a.l = l;
  a.bn = plan.bn;
  a.split = plan.split;
  const int features = gated ? l.n / 2 : l.n, feat = (gated ? 64 : 128) * (plan.pair ? 2 : 1);
  a.m_tiles = (features + feat - 1) / feat;
  a.part = plan.pair ? a.bn / 2 : a.bn;
  a.stage_bytes = stage_bytes8(a.part);
  const int64_t sgs = l.groups > 1 ? l.w_scales_group_stride : 0;
  a.w_load = scale_load(l.w_scales, l.w_scales_stride, sgs, l.k);
  a.x_load = scale_load(l.x_scales, l.x_scales_stride, 0, l.k);
  a.tile_limit = kWaitLimitCycles + 2048ll * ((l.k + kBK8 - 1) / kBK8);
  a.stages = stages8(gated || l.codes, a.part, l.groups);
  const int csize = plan.pair ? 2 : plan.split, most = sms / csize;
  const int grid = static_cast<int>(plan.tiles < 1 ? 1 : plan.tiles < most ? plan.tiles : most) * csize;
  const size_t smem = smem8(gated || l.codes, a.part, l.groups);

  // two elements a 16-bit unit of the maps: [unit, row, gate or up, piece, group]
  Maps8 m{};
  a.pieces = l.k % kPiece == 0;
  const uint64_t w_row = l.w_stride, x_row = l.x_stride, n = features, rows = l.rows;
  const uint64_t units = a.pieces ? kPiece / 2 : l.k / 2, pieces = a.pieces ? l.k / kPiece : 1;
  const uint32_t box = a.pieces ? kPieces : 1;
  const uint64_t gs = l.groups > 1 ? l.w_group_stride : w_row * l.n;
  cudaError_t e = make_tmap_5d(&m.w, l.w, {units, n, gated ? 2u : 1u, pieces, uint64_t(l.groups)},
                               {w_row, n * w_row, kPiece, gs}, {kPiece / 2, gated ? 64u : 128u, gated ? 2u : 1u, box, 1});
  const auto columns = [&](CUtensorMap* map, int part) {
    return make_tmap_5d(map, l.x, {units, rows, 1, pieces, 1}, {x_row, x_row, kPiece, x_row},
                        {kPiece / 2, uint32_t(part), 1, box, 1});
  };
  if (e == cudaSuccess) e = columns(&m.x, a.part);
  m.half = m.x;
  if (e == cudaSuccess && a.part >= 32) e = columns(&m.half, a.part / 2);
  // scales: 16 bytes of each row
  const uint64_t s_row = l.w_scales_stride, blocks = l.k / kBlock8;
  if (e == cudaSuccess && a.w_load == 16) {
    e = make_tmap_bytes_4d(&m.sw, l.w_scales, {blocks, n, gated ? 2u : 1u, uint64_t(l.groups)},
                           {s_row, n * s_row, l.groups > 1 ? uint64_t(sgs) : s_row * l.n},
                           {16, gated ? 64u : 128u, gated ? 2u : 1u, 1});
    a.w_load = kScaleMap;
  }
  if (e == cudaSuccess && a.x_load == 16) {
    const uint64_t xs = l.x_scales_stride;
    e = make_tmap_bytes_4d(&m.sx, l.x_scales, {blocks, rows, 1, 1}, {xs, xs, xs}, {16, uint32_t(a.bn), 1, 1});
    a.x_load = kScaleMap;
  }
  if (e != cudaSuccess) return e;
  if (plan.pair)
    return l.codes ? launch_form<true, true>(gated, l.bf16, m, a, grid, smem, st)
                   : launch_form<true, false>(gated, l.bf16, m, a, grid, smem, st);
  return l.codes ? launch_form<false, true>(gated, l.bf16, m, a, grid, smem, st)
                 : launch_form<false, false>(gated, l.bf16, m, a, grid, smem, st);
}

cudaError_t linear8_error_word(int** word) {
  void* p = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&p, g_linear8_error);
  *word = static_cast<int*>(p);
  return e;
}

}  // namespace senmoe
