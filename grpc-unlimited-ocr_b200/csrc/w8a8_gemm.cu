// W8A8 products on the tensor cores (include/uocr_int8.h): tcgen05.mma of
// signed 8-bit operands with int32 accumulators in TMEM, dense or grouped.
//
// The weights are the M operand and the tokens the N operand: a pair of SMs
// (cta_group::2) multiplies 256 weight rows (128 in each SM) by up to 256
// tokens, N being the tile's own token count rounded up to 32. A ragged group
// so wastes at most 31 tokens' work, where a token tile of 256 rows would
// waste half of it, and a handful of tokens costs a narrow MMA. The 256 rows
// are output channels, or in the gated form the gate and up rows of 128
// channels, 64 and 64 in each SM.
//
// One persistent pair of blocks per two SMs (K in parts: a cluster of pairs a
// tile), warp-specialised:
//   warps 0, 2  producers, one lane each, per 128-byte slice of K: warp 0 the
//              CTA's 128 weight rows, warp 2 its half of the token rows (boxes
//              of 128, 64 or 16 rows);
//   warp 1     allocates TMEM; in the leader one lane issues the MMAs;
//   warps 4-11 epilogue, 32 tokens x 32 weight rows at a time: the scales,
//              then bf16 tiles are transposed into shared memory (stmatrix) and
//              leave as bulk tensor stores, fp32 ones as lines of 32 channels
//              (gated: sectors of 8), a residual arriving by TMA two units ahead.
//              When gated, the gate's warp and the up's warp of the same
//              channels exchange half of their tokens first.
// A dense product of few tiles and a long K has K in two or four parts, a pair
// for each in one cluster: a slice of K takes 0.19 us whether one pair is at work
// or all, since a pair waits for its own copies. The int32 sums, exact in any
// order, meet in shared memory (64 x 2048 x 8192: 9.7 us, by one pair a tile 16.7).
// Rows named by an index are first copied together (gather_rows_kernel): TMA
// gathers four rows of 128 bytes at a time, 44 clocks each, against 512 clocks
// of MMAs for 32 of them (1108 us at eight pages' gate/up, 649 us without the
// index), and loads by threads have to be announced across the pair by a
// release at cluster scope, which takes longer still (1277 us).
// The operands' copies into shared memory and the MMAs' reads of it take
// nearly all of its bandwidth (64 + 64 bytes a clock at the full MMA rate), and
// every store and shared-memory access of the epilogue takes a clock of the
// same pipe: the layout is chosen for few and full ones. Measured at 8192 x
// 8192 x 4096: 171 us, 3200 TOP/s, the tensor pipe active for 87 % of the time.
// Two forms of the epilogue go by single bf16 values, a warp's access being four
// tokens x 8 channels, 16 bytes together: outputs whose rows do not start at 16
// bytes (8192 x 2047 x 64 23.5 us, with 2048 12.5; 24576 rows of 64 groups by 1001 x
// 1024 41.8, by 1008 30.9, gated 67.5 and 57.4), and bf16 residuals, read when the
// sums are there (4096 x 2048 x 2048 23.7 us, without 17.3; fp32 22.6 and 20.1).
// With few slices of K the copies bound the product, at 55 bytes a clock into each SM:
// at 8192 x 8192 x 1024 the MMAs alone take 57 kcycles, the copies alone 67, all
// but the stores 81, the whole 91.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tc.cuh"
#include "tc_gemm.h"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kMaxGroups = 512;
constexpr int kBM = 128;               // weight rows per CTA
constexpr int kBK = 128;               // bytes of K per stage (one swizzle atom)
constexpr int kMaxN = 256;             // tokens per tile
constexpr int kABytes = kBM * kBK;
constexpr int kStageBytes = kABytes + kMaxN / 2 * kBK;
constexpr int kStages = 5;
constexpr int kEpilogueWarps = 8;
constexpr int kWays = kEpilogueWarps / 4;  // epilogue warps of a TMEM lane quarter
constexpr int kThreads = 128 + kEpilogueWarps * 32;
constexpr int kUnit = 32;              // tokens an epilogue warp takes at a time
constexpr int kOutBytes = kUnit * 32 * 2;        // a unit of 32 channels in bf16
constexpr int kXchBytes = kUnit / 2 * 32 * 4;    // gated: half a unit's values for the partner warp
constexpr int kRows32 = 16;            // tokens of an fp32 unit
constexpr int kSlotBytes = kRows32 * 32 * 4;     // an fp32 unit's residual
constexpr int kSlots = 3;              // two 3 % slower at a page of 2048, 6 % at 8192 x 8192 x 1024
// Per epilogue warp: two buffers of each in bf16 (a gated warp's output is half
// a unit), or the fp32 units' residuals.
template <bool kGated, bool kBf16>
constexpr int kWarpBytes = kGated ? kOutBytes + 2 * kXchBytes : kBf16 ? 2 * kOutBytes : kSlots * kSlotBytes;
template <bool kGated, bool kBf16>
constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * kWarpBytes<kGated, kBf16> + 1024;
constexpr int kTmemCols = 512;
constexpr int kBoxRows = 16;
constexpr int kBand = 8;               // token tiles of a band (decode_tile)

static_assert(kEpilogueWarps * 32 == kMaxN, "an epilogue thread for each token of a tile (Shared::x_scale)");

struct Args {
  CUtensorMap y;                         // boxes of a unit's tokens (gated: half) x 32 channels; unset unless tma_store
  CUtensorMap residual;                  // boxes of an fp32 unit's tokens x 32 channels; unset unless tma_residual
  CUtensorMap x, x_wide, x_half, w, up;  // token boxes of 16, 64 and 128 rows; weight boxes of 128 (gated: 64)
  W8a8 p;
  int tokens_per_tile;  // at most kMaxN, a multiple of 32
  int channels;         // output channels per tile of a pair
  int c_tiles, k_blocks;
  bool tma_store;       // y is bf16 and its rows start at 16-byte boundaries
  bool tma_residual;    // y is fp32 and the residual's rows start at 16-byte boundaries
};

struct Tile {
  int g, row0, rows, c0;
};

struct Shared {
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drain;
  uint64_t residual[kEpilogueWarps][kSlots];
  uint32_t tmem;
  Tile tiles[3][32];  // of the three warps that work through one lane: what is next
  int failed[2];  // an epilogue warp's wait for this accumulator ran out
  alignas(16) float x_scale[2][kMaxN];
  int tile_start[kMaxGroups + 1];
  int first[kMaxGroups], count[kMaxGroups];
};

// After a wait that ran out: the copies in flight land before this CTA's shared memory is given up.
__device__ __noinline__ void wait_for_copies() {
  const uint64_t until = global_timer_ns() + 5000000ull;
  for (int i = 0; i < (1 << 20) && global_timer_ns() < until; ++i) __nanosleep(1000);
}

__device__ __forceinline__ int round32(int v) { return (v + 31) & ~31; }

__device__ __forceinline__ Tile decode_tile(int t, const Shared& sh, int groups, const Args& a) {
  int lo = 0, hi = groups - 1;  // last g with tile_start[g] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sh.tile_start[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  // (Unsigned divisions: with signed ones 300 x 2048 x 1024 took 7.8 us for 7.4.)
  const unsigned local = t - sh.tile_start[lo], count = sh.count[lo];
  const unsigned r_tiles = (count + a.tokens_per_tile - 1) / static_cast<unsigned>(a.tokens_per_tile);
  const unsigned per = (((count + r_tiles - 1) / r_tiles) + 31) & ~31u;  // the group's tokens dealt evenly
  // Bands of kBand token tiles, token tile fastest: the pairs at work at a time share both operands in L2.
  const unsigned band = local / (kBand * static_cast<unsigned>(a.c_tiles)), in_band = local - band * kBand * a.c_tiles;
  const unsigned high = min(static_cast<unsigned>(kBand), r_tiles - band * kBand);
  const unsigned c = in_band / high;
  const unsigned r = (band * kBand + in_band - c * high) * per;
  return Tile{lo, static_cast<int>(sh.first[lo] + r), static_cast<int>(min(per, count - r)),
              static_cast<int>(c) * a.channels};
}

template <bool kBf16>
using Out = typename std::conditional<kBf16, __nv_bfloat16, float>::type;

// (float(a0) * s0 * w, float(a1) * s1 * w): two tokens' sums scaled, with packed products.
__device__ __forceinline__ void scale_pair(int a0, int a1, uint64_t s2, uint64_t w2, float& v0, float& v1) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(static_cast<float>(a0)), "f"(static_cast<float>(a1)));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(s2));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(w2));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v0), "=f"(v1) : "l"(v));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight tokens x 32 channels of a warp: v[2 q + e] is channel t / 4 + 8 q of
// token 2 (t % 4) + e in thread t.
using Block = float[8];

// Block b of a unit in bf16 to the unit's rows of 64 bytes in shared memory, as the 64-byte swizzle has them.
__device__ __forceinline__ void stage_block(const Block& v, unsigned char* stg, int b, int lane) {
  const int token = b * 8 + (lane & 7);
  stmatrix_x4_trans(stg + token * 64 + (((lane >> 3) ^ ((token >> 1) & 3)) << 4), pack_bf16(v[0], v[1]),
                    pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// A block to (or a residual's block from) rows at `base`, the address of this
// thread's first token and channel: tokens below nr, channels below nc, or
// all of them, without a test that would keep the accesses from overlapping.
template <typename T>
__device__ __forceinline__ void store_block(const Block& v, T* base, int64_t ld) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int q = 0; q < 4; ++q) put(base + e * ld + 8 * q, v[2 * q + e]);
}
template <typename T>
__device__ __forceinline__ void store_block(const Block& v, T* base, int64_t ld, int nr, int nc) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (e >= nr) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (8 * q < nc) put(base + e * ld + 8 * q, v[2 * q + e]);
  }
}
template <typename T>
__device__ __forceinline__ void load_block(Block& v, const T* base, int64_t ld) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[2 * q + e] = to_f32(base[e * ld + 8 * q]);
}
template <typename T>
__device__ __forceinline__ void load_block(Block& v, const T* base, int64_t ld, int nr, int nc) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[2 * q + e] = e < nr && 8 * q < nc ? to_f32(base[e * ld + 8 * q]) : 0.0f;
}

// kS: pairs of a cluster, which share a tile's K; above 1 a cluster has one tile.
template <bool kGated, bool kBf16, int kS>
__global__ void __cluster_dims__(2 * kS, 1, 1) __launch_bounds__(kThreads, 1)
    w8a8_gemm_kernel(const __grid_constant__ Args args) {
  extern __shared__ unsigned char dyn_raw[];
  __shared__ Shared sh;
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const W8a8& p = args.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank() & 1u), part = static_cast<int>(cluster_rank() >> 1);
  const uint32_t leader = kS > 1 ? cluster_rank() & ~1u : 0u;
  const int pair0 = static_cast<int>(blockIdx.x) / (2 * kS);
  const int groups = static_cast<int>(p.groups);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], 2 * kEpilogueWarps);
    }
    mbar_init(&sh.drain, 1);
    for (int w = 0; w < kEpilogueWarps; ++w)
      for (int i = 0; i < kSlots; ++i) mbar_init(&sh.residual[w][i], 1);
    sh.failed[0] = sh.failed[1] = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(&sh.tmem, kTmemCols);
  pdl_wait();  // what precedes it touches nothing that the grid before may be using
  pdl_launch_dependents();
  if (warp == 0) {
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
      const int g = g0 + lane;
      int tiles = 0;
      if (g < groups) {
        int first = 0;
        int64_t count = p.rows;
        if (p.starts != nullptr) {
          first = p.starts[g];
          count = p.counts != nullptr ? p.counts[g] : static_cast<int64_t>(p.starts[g + 1]) - first;
          if (first < 0 || count < 0 || first + count > p.rows) {
            raise_error(p.err, kDevBadIndex, kSiteGroupRows, g, first);
            count = 0;
          }
        }
        sh.first[g] = first;
        sh.count[g] = static_cast<int>(count);
        tiles = static_cast<int>((count + args.tokens_per_tile - 1) / args.tokens_per_tile) * args.c_tiles;
      }
      int incl = tiles;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (g < groups) sh.tile_start[g] = carry + incl - tiles;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) sh.tile_start[groups] = carry;
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers exist before either is signalled from the other
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem;
  const int total = sh.tile_start[groups];
  const int step = static_cast<int>(gridDim.x) / (2 * kS);
  const int kb0 = kS > 1 ? part * args.k_blocks / kS : 0;
  const int kb1 = kS > 1 ? (part + 1) * args.k_blocks / kS : args.k_blocks;

  // One lane's pass over this pair's tiles, body(tile, n) for the n-th; the
  // warp works 32 of them out at a time, a lane each (one takes hundreds of
  // clocks, which between two tiles would leave the MMAs waiting).
  auto each_tile = [&](Tile* table, auto&& body) {
    bool ok = true;
    for (int n0 = 0; ok && pair0 + n0 * step < total; n0 += 32) {
      const int mine = pair0 + (n0 + lane) * step;
      if (mine < total) table[lane] = decode_tile(mine, sh, groups, args);
      __syncwarp();
      if (elect_one())
        for (int i = 0; i < 32 && ok && pair0 + (n0 + i) * step < total; ++i) ok = body(table[i], n0 + i);
      ok = __all_sync(0xffffffffu, ok);
    }
    return ok;
  };

  if (warp == 0) {
    // ---- weight producer: one lane; the leader also announces both CTAs' bytes of a stage ----
    const uint32_t full0 = cluster_addr(&sh.full[0], leader);
    int stage = 0;
    uint32_t phase = 0;
    const bool ok = each_tile(sh.tiles[0], [&](const Tile& tl, int) {
      const uint32_t bytes = 2 * kABytes + round32(tl.rows) * kBK;
      const int w_row = tl.g * static_cast<int>(p.n) + tl.c0 + rank * (args.channels / 2);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&sh.empty[stage], phase ^ 1)) {
          raise_error(p.err, kDevWaitTimeout, 82, tl.row0, kb);
          return false;
        }
        unsigned char* sa = smem + stage * kStageBytes;
        if (rank == 0) mbar_arrive_expect_tx(&sh.full[stage], bytes);
        tma_load_2d_pair(sa, &args.w, kb * kBK, w_row, full0 + stage * 8);
        if (kGated) tma_load_2d_pair(sa + kABytes / 2, &args.up, kb * kBK, w_row, full0 + stage * 8);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      return true;
    });
    if (!ok) wait_for_copies();
  } else if (warp == 2) {
    // ---- token producer: one lane ----
    const uint32_t full0 = cluster_addr(&sh.full[0], leader);
    int stage = 0;
    uint32_t phase = 0;
    const bool ok = each_tile(sh.tiles[1], [&](const Tile& tl, int) {
      const int half = round32(tl.rows) / 2;
      const int row = tl.row0 + rank * half;  // this CTA's first token row
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&sh.empty[stage], phase ^ 1)) {
          raise_error(p.err, kDevWaitTimeout, 87, tl.row0, kb);
          return false;
        }
        unsigned char* sb = smem + stage * kStageBytes + kABytes;
        const uint32_t bar = full0 + stage * 8;
        if (half == kMaxN / 2) {
          tma_load_2d_pair(sb, &args.x_half, kb * kBK, row, bar);
        } else {
          int i = 0;
          if (half >= 64) {
            tma_load_2d_pair(sb, &args.x_wide, kb * kBK, row, bar);
            i = 64;
          }
          for (; i < half; i += kBoxRows) tma_load_2d_pair(sb + i * kBK, &args.x, kb * kBK, row + i, bar);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      return true;
    });
    if (!ok) wait_for_copies();
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- MMA issuer (for both CTAs): one lane ----
      int stage = 0;
      uint32_t phase = 0;
      each_tile(sh.tiles[2], [&](const Tile& tl, int local) {
        const uint32_t idesc = i8_idesc(2 * kBM, round32(tl.rows));
        const int acc = local & 1;
        if (!mbar_wait(&sh.acc_empty[acc], ((local >> 1) & 1) ^ 1)) {
          raise_error(p.err, kDevWaitTimeout, 83, tl.row0, 0);
          return false;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kMaxN);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&sh.full[stage], phase)) {
            raise_error(p.err, kDevWaitTimeout, 84, tl.row0, kb);
            return false;
          }
          tc_fence_after();
          const uint32_t sa = smem_addr(smem + stage * kStageBytes);
          const uint64_t ad = sw128_kmajor_desc(sa);
          const uint64_t bd = sw128_kmajor_desc(sa + kABytes);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)  // 32 bytes of K per instruction: +2 in the address field
            umma_i8_pair(d, ad + 2 * k, bd + 2 * k, idesc, ((kb - kb0) | k) != 0 ? 1u : 0u);
          umma_commit_pair(&sh.empty[stage], leader);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        umma_commit_pair(&sh.acc_full[acc], leader);
        return true;
      });
      if (elect_one()) {  // the lane that issued: every MMA is complete before shared memory and TMEM are given up
        umma_commit_pair(&sh.drain, leader);
        if (!mbar_wait(&sh.drain, 0)) raise_error(p.err, kDevWaitTimeout, 85, 0, 0);
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue: TMEM lane quarter = warp % 4; the warps of a quarter take units in turn ----
    using T = Out<kBf16>;
    const int e = warp - 4, quarter = warp & 3, way = e >> 2;
    const int et = threadIdx.x - 128;
    const int tr = lane >> 2, tc = 2 * (lane & 3);  // this thread's first channel and token in a block
    // fp32 outputs: lane = channel, so that a token's 32 channels are a line of 128 bytes.
    constexpr bool kLaneIsChannel = !kGated && !kBf16;
    const int first_c = kLaneIsChannel ? lane : tr;
    unsigned char* area = smem + kStages * kStageBytes;
    unsigned char* stg = area + e * kWarpBytes<kGated, kBf16>;
    float4* xch = reinterpret_cast<float4*>(stg + kOutBytes);
    const float4* xch_other = reinterpret_cast<const float4*>(area + (e ^ 2) * kWarpBytes<kGated, kBf16> + kOutBytes);
    const bool gate = quarter < 2;  // gated: lanes 0-63 hold gate rows, 64-127 up rows
    const int local_c = kGated ? rank * 64 + (quarter & 1) * 32 : rank * kBM + quarter * 32;
    const float* w_scales = kGated && !gate ? p.w_up_scales : p.w_scales;
    T* y = static_cast<T*>(p.y);
    const bool has_bias = !kGated && p.bias != nullptr, has_residual = !kGated && p.residual != nullptr;
    const bool tma_residual = kLaneIsChannel && args.tma_residual;
    // K in parts: which pair finishes a unit, and where in its shared memory
    // another's (the src-th of the others') sums of it go, this lane's part of
    // this warp's: 16 bytes at a pitch of 512.
    constexpr int kPart = kLaneIsChannel ? kRows32 : kUnit;
    auto owner = [&](int unit) { return kS == 2 ? (unit >> 1) & 1 : unit % kS; };
    auto part_sums = [&](int unit, int src) {
      const int place = kS == 2 ? (unit >> 2) * 2 + (unit & 1) : unit / kS;
      return smem + ((place * (kS - 1) + src) * 4 + quarter) * (kPart * 128) + lane * 16;
    };
    // What the epilogue needs of a tile beside its sums; the next tile's is
    // fetched while this one's units are stored.
    struct Scales {
      Tile tl;
      float w[kLaneIsChannel ? 1 : 4], bias[kLaneIsChannel ? 1 : 4];  // of channels first_c + 8 q
      float x;                                                        // of token et
    };
    // Every 32 tiles each lane works one of them out (hundreds of clocks in a
    // row, which a tile's epilogue has not got).
    Tile lane_tile{};
    auto fetch = [&](int nth) {
      if ((nth & 31) == 0 && pair0 + (nth + lane) * step < total)
        lane_tile = decode_tile(pair0 + (nth + lane) * step, sh, groups, args);
      Scales f{};
      f.tl = Tile{__shfl_sync(0xffffffffu, lane_tile.g, nth & 31), __shfl_sync(0xffffffffu, lane_tile.row0, nth & 31),
                  __shfl_sync(0xffffffffu, lane_tile.rows, nth & 31), __shfl_sync(0xffffffffu, lane_tile.c0, nth & 31)};
      const int64_t c = f.tl.c0 + local_c + first_c;
#pragma unroll
      for (int q = 0; q < (kLaneIsChannel ? 1 : 4); ++q) {
        const bool in = c + 8 * q < p.n;
        f.w[q] = in ? w_scales[f.tl.g * p.n + c + 8 * q] : 0.0f;
        f.bias[q] = has_bias && in ? p.bias[c + 8 * q] : 0.0f;
      }
      if (et < f.tl.rows) {  // tokens past the tile, and rows x does not have: zero
        int64_t r = f.tl.row0 + et;
        if (p.row_index != nullptr) {
          const int v = p.row_index[r];
          if (v < 0 || v >= p.x_rows) {
            raise_error(p.err, kDevBadIndex, kSiteRowIndex, static_cast<int>(r), v);
            r = -1;
          } else {
            r = v;
          }
        }
        if (r >= 0) f.x = p.x_scales[r];
      }
      return f;
    };
    Scales next{};
    if (pair0 < total) next = fetch(0);
    int local = 0, xbuf = 0, obuf = 0, slot = 0;  // xbuf turns over with each unit, obuf with each bulk store
    uint32_t slot_phase = 0;
    bool ok = true;
    for (int t = pair0; t < total; t += step, ++local) {
      const Scales cur = next;
      const Tile& tl = cur.tl;
      const int acc = local & 1;
      const int64_t c0 = tl.c0 + local_c, c = c0 + first_c;
      const int nc = static_cast<int>(p.n - c < 32 ? p.n - c : 32);  // channels c, c + 8, .. below c + nc exist
      sh.x_scale[acc][et] = cur.x;
      uint64_t ws[kLaneIsChannel ? 1 : 4];
#pragma unroll
      for (int q = 0; q < (kLaneIsChannel ? 1 : 4); ++q) asm("mov.b64 %0, {%1, %1};" : "=l"(ws[q]) : "f"(cur.w[q]));
      // The residual of an fp32 unit whose 16 tokens all exist, into a slot of this warp.
      auto whole_unit = [&](int j0) { return tl.rows - j0 >= kRows32 && c0 < p.n; };
      auto fetch_residual = [&](int j0, int s) {
        if (!tma_residual || !whole_unit(j0) || !elect_one()) return;
        mbar_arrive_expect_tx(&sh.residual[e][s], kSlotBytes);
        tma_load_2d(stg + s * kSlotBytes, &args.residual, static_cast<int>(c0), tl.row0 + j0, &sh.residual[e][s]);
      };
      auto ahead = [&](int i) { return slot + i < kSlots ? slot + i : slot + i - kSlots; };
      if (kLaneIsChannel && ok)
        for (int i = 0; i < kSlots - 1; ++i) fetch_residual((way + i * kWays) * kRows32, ahead(i));
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], (local >> 1) & 1));
        if (!ok) raise_error(p.err, kDevWaitTimeout, 86, t, 0);
      }
      if (!ok && lane == 0) sh.failed[acc] = 1;
      named_bar_sync(1, kEpilogueWarps * 32);  // the scales are there; and all warps go on with this tile or none
      ok = sh.failed[acc] == 0;
      const uint32_t taddr =
          tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kMaxN);
      if constexpr (kS > 1) {
        // The pairs' sums over their parts of K: each finishes some units, and
        // has the others' sums of those brought to where its operands were.
        cluster_barrier();  // every pair's MMAs are complete: no operand is in use any more
        if (ok) {
          tc_fence_after();
          for (int j0 = way * kPart; j0 < tl.rows; j0 += kWays * kPart) {
            const int to = owner(j0 / kPart);
            if (to == part) continue;
            int a[kPart];
            if constexpr (kLaneIsChannel) {
              tmem_ld_32x16(taddr + j0, a);
            } else {
              int b[2][16];
              tmem_ld_16x32(taddr + j0, b[0]);
              tmem_ld_16x32(taddr + (16u << 16) + j0, b[1]);
              tmem_ld_wait(b[0], b[1]);
#pragma unroll
              for (int i = 0; i < kPart; ++i) a[i] = b[i / 16][i % 16];
            }
            const uint32_t dst = cluster_addr(part_sums(j0 / kPart, part - (part > to ? 1 : 0)), 2 * to + rank);
#pragma unroll
            for (int i = 0; i < kPart; i += 4) st_cluster_v4(dst + i * 128, a[i], a[i + 1], a[i + 2], a[i + 3]);
          }
        }
        cluster_barrier();
      }
      if (!ok) continue;
      tc_fence_after();
      // The other pairs' sums of a unit of this one, added to its own.
      auto add_parts = [&](int unit, int* a, int first, int n) {
        for (int src = 0; src < kS - 1; ++src) {
          const int4* in = reinterpret_cast<const int4*>(part_sums(unit, src)) + first / 4 * 32;
#pragma unroll
          for (int i = 0; i < n / 4; ++i) {
            const int4 v = in[i * 32];
            a[4 * i] += v.x, a[4 * i + 1] += v.y, a[4 * i + 2] += v.z, a[4 * i + 3] += v.w;
          }
        }
      };
      auto release = [&] {  // this warp has read its last columns: the accumulator may be written again
        if (kS > 1) return;  // there is no further tile
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(cluster_addr(&sh.acc_empty[acc], leader));
      };
      if (t + step < total) next = fetch(local + 1);
      if constexpr (kLaneIsChannel) {
        const int64_t pitch = p.ldy * 4;
        if (way * kRows32 >= tl.rows) release();
        for (int j0 = way * kRows32; j0 < tl.rows; j0 += kWays * kRows32) {
          if (kS > 1 && owner(j0 / kPart) != part) continue;
          // (The slot's values, a unit ago, have been read by the whole warp.)
          fetch_residual(j0 + (kSlots - 1) * kWays * kRows32, ahead(kSlots - 1));
          int a[kRows32];
          tmem_ld_32x16(taddr + j0, a);
          if constexpr (kS > 1) add_parts(j0 / kPart, a, 0, kRows32);
          if (j0 + kWays * kRows32 >= tl.rows) release();
          float v[kRows32];
#pragma unroll
          for (int i = 0; i < kRows32; i += 4) {
            const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&sh.x_scale[acc][j0 + i]);
            scale_pair(a[i], a[i + 1], s.x, ws[0], v[i], v[i + 1]);
            scale_pair(a[i + 2], a[i + 3], s.y, ws[0], v[i + 2], v[i + 3]);
          }
          if (has_bias) {
#pragma unroll
            for (int i = 0; i < kRows32; ++i) v[i] += cur.bias[0];
          }
          const int nr = c < p.n ? tl.rows - j0 : 0;
          if (tma_residual && whole_unit(j0)) {
            if (!mbar_wait(&sh.residual[e][slot], (slot_phase >> slot) & 1))
              raise_error(p.err, kDevWaitTimeout, 89, t, j0);
            slot_phase ^= 1u << slot;
            const float* in = reinterpret_cast<const float*>(stg + slot * kSlotBytes) + lane;
#pragma unroll
            for (int i = 0; i < kRows32; ++i) v[i] += in[i * 32];
          } else if (has_residual) {
            const float* res = static_cast<const float*>(p.residual) + (static_cast<int64_t>(tl.row0) + j0) * p.ldr + c;
#pragma unroll
            for (int i = 0; i < kRows32; ++i)
              if (i < nr) v[i] += res[i * p.ldr];
          }
          char* out = static_cast<char*>(p.y) + ((static_cast<int64_t>(tl.row0) + j0) * p.ldy + c) * 4;
          if (nr >= kRows32) {
#pragma unroll
            for (int i = 0; i < kRows32; ++i, out += pitch) *reinterpret_cast<float*>(out) = v[i];
          } else {
#pragma unroll
            for (int i = 0; i < kRows32; ++i, out += pitch)
              if (i < nr) *reinterpret_cast<float*>(out) = v[i];
          }
          __syncwarp();
          slot = ahead(1);
        }
        continue;
      } else {
        if (way * kUnit >= tl.rows) release();
        for (int j0 = way * kUnit; j0 < tl.rows; j0 += kWays * kUnit) {
          if (kS > 1 && owner(j0 / kPart) != part) continue;
          int a[2][16];  // [16 lanes][the four blocks' four values]
          tmem_ld_16x32(taddr + j0, a[0]);
          tmem_ld_16x32(taddr + (16u << 16) + j0, a[1]);
          const int64_t row = tl.row0 + j0;
          const int nr = tl.rows - j0;
          tmem_ld_wait(a[0], a[1]);
          if constexpr (kS > 1) {
            add_parts(j0 / kPart, a[0], 0, 16);
            add_parts(j0 / kPart, a[1], 16, 16);
          }
          if (j0 + kWays * kUnit >= tl.rows) release();
          xbuf ^= 1;
          const bool whole = nr >= kUnit && c0 + 32 <= p.n;
          Block v[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint64_t s = *reinterpret_cast<const uint64_t*>(&sh.x_scale[acc][j0 + 8 * b + tc]);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              scale_pair(a[q >> 1][4 * b + 2 * (q & 1)], a[q >> 1][4 * b + 2 * (q & 1) + 1], s, ws[q], v[b][2 * q],
                         v[b][2 * q + 1]);
          }
          // Blocks first .. first + kOut - 1 of the unit are this warp's to store.
          constexpr int kOut = kGated ? 2 : 4;
          int first = 0;
          if (kGated) {
            // The gate's warp finishes the unit's first two blocks, the up's warp the others.
            first = gate ? 0 : 2;
            float4* give = xch + xbuf * (kXchBytes / 16);
            const float4* take = xch_other + xbuf * (kXchBytes / 16);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const Block& o = gate ? v[2 + b] : v[b];
                give[(2 * b + h) * 32 + lane] = make_float4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
              }
            named_bar_sync(2 + (quarter & 1) + 2 * way, 64);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float4 w4 = take[(2 * b + h) * 32 + lane];
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float own = gate ? v[b][4 * h + i] : v[2 + b][4 * h + i];
                  v[b][4 * h + i] = silu_mul(gate ? own : w[i], gate ? w[i] : own);
                }
              }
          } else {
            if (has_bias) {
#pragma unroll
              for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[b][i] += cur.bias[i / 2];
            }
            if (has_residual) {
              const T* res = static_cast<const T*>(p.residual) + (row + tc) * p.ldr + c;
              Block r[4];
              if (whole) {
#pragma unroll
                for (int b = 0; b < 4; ++b) load_block(r[b], res + 8 * b * p.ldr, p.ldr);
              } else {
#pragma unroll
                for (int b = 0; b < 4; ++b) load_block(r[b], res + 8 * b * p.ldr, p.ldr, nr - tc - 8 * b, nc);
              }
#pragma unroll
              for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[b][i] += r[b][i];
            }
          }
          if (kBf16 && args.tma_store && nr >= 8 * (first + kOut)) {
            // The buffers alternate with the groups that are committed: a unit
            // stored directly (a tile's partial end) commits none and takes none,
            // else the wait would let the one store still pending be this buffer's.
            obuf ^= 1;
            unsigned char* out = stg + obuf * (kOut * 8 * 64);
            if (elect_one()) bulk_wait_read<1>();  // the store before the last has read this buffer
            __syncwarp();
#pragma unroll
            for (int b = 0; b < kOut; ++b) stage_block(v[b], out, b, lane);
            fence_proxy_async_smem();
            __syncwarp();
            if (elect_one()) {
              if (c0 < p.n) tma_store_2d(&args.y, static_cast<int>(c0), static_cast<int>(row) + 8 * first, out);
              bulk_commit();
            }
          } else {
            T* dst = y + (row + 8 * first + tc) * p.ldy + c;
            if (whole) {
#pragma unroll
              for (int b = 0; b < kOut; ++b) store_block(v[b], dst + 8 * b * p.ldy, p.ldy);
            } else {
#pragma unroll
              for (int b = 0; b < kOut; ++b)
                store_block(v[b], dst + 8 * b * p.ldy, p.ldy, nr - tc - 8 * (first + b), nc);
            }
          }
        }
      }
    }
    if (elect_one()) bulk_wait_read<0>();
  }
  __syncwarp();
  if (kS > 1 && warp < 4) {  // the epilogue's two meetings
    cluster_barrier();
    cluster_barrier();
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // the pair's MMAs are complete: no operand, accumulator or barrier is in use any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  __syncthreads();
  cluster_barrier();
}

// Clusters that run at the same time on the current device.
template <bool kGated, bool kBf16, int kS>
cudaError_t resident_clusters(int* clusters) {
  static std::mutex mu;
  static int known[kMaxDevices] = {};
  int dev = 0;
  cudaError_t st = cudaGetDevice(&dev);
  if (st != cudaSuccess) return st;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev] == 0) {
    const auto kernel = w8a8_gemm_kernel<kGated, kBf16, kS>;
    st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<kGated, kBf16>);
    if (st != cudaSuccess) return st;
    int sms = 0;
    if ((st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return st;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(sms / (2 * kS) * 2 * kS));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem<kGated, kBf16>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * kS;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if ((st = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg)) != cudaSuccess) return st;
    if (n <= 0 && kS == 1) return cudaErrorNotSupported;
    known[dev] = n > 0 ? n : -1;  // a device may hold no larger cluster: K then stays whole
  }
  *clusters = known[dev];
  return cudaSuccess;
}

// Tokens per tile: the width that ends first; of equals the widest, or in a
// single wave the narrowest, which spreads the larger groups over idle pairs
// (154 rows in 16 uneven groups 6.3 us at 64, 7.2 at 256). A pair's
// time for a slice of K is its copies', 128 weight rows and half of the tokens
// in each SM, so a tile of n tokens costs n + 256 and the tiles come in waves.
// Measured in us, the width taken against 256: dense, 64 x 2048 x 2048 7.4 / 8.1
// (32); 200 rows 8.2 / 10.6 (32); 500 x 4096 x 2048 8.5 / 10.5 (128); 3000 x 2048
// x 2048 14.8 / 15.8 (192); 4096 x 2048 x 2048 stays at 256: 20.0, at 160 21.3.
// Groups' sizes are known on the device only: as if even, half a tile of each
// lost, and halved widths alone, since a narrower guess that breaks a group
// once more costs a wave. 2 groups of 200 rows, 2048 x 1024: 7.1 / 8.3 (64); 4
// of 128 gated stay at 256: 12.3, at 64 16.0; 8 of 150 8.4, at 128 10.1.
int choose_tokens(int64_t rows, int64_t groups, int c_tiles, int pairs, int64_t* best_cost) {
  const int64_t parts = groups < rows ? groups : rows, even = (rows + parts - 1) / parts;
  const int narrowest = groups > 1 ? 64 : 32;
  int best = kMaxN;
  *best_cost = INT64_MAX;
  for (int bn = kMaxN; bn >= narrowest; bn = groups > 1 ? bn / 2 : bn - 32) {
    int64_t tiles = (rows + bn - 1) / bn, width = (rows + tiles - 1) / tiles;
    if (groups > 1) {
      tiles = std::max(parts, rows / bn + parts / 2);
      width = std::min<int64_t>(bn, even);
    }
    const int64_t waves = (tiles * c_tiles + pairs - 1) / pairs, cost = waves * ((width + 31) / 32 * 32 + 256);
    if (cost < *best_cost || (cost == *best_cost && waves == 1)) {
      *best_cost = cost;
      best = bn;
    }
  }
  return best;
}

// K in `parts` parts where that costs less than `cost`, all tiles' clusters at
// the same time (a second wave of clusters starts 6 us late): tiles as narrow as
// lets them. A slice of K of 32 tokens is 288 in the cost and takes 0.19 us, on one
// pair as on 74; the exchange takes 1.5 us at 32 tokens and 5 at 256. Measured
// in us, in two parts or four / whole: 64 x 2048 x 8192 9.7 (4) / 16.7; 64 x 4096
// x 8192 14.6 (2) / 19.2; 64 x 2048 x 2048 7.2 (4) / 7.4; 128 x 300 x 2048 6.6
// (4) / 7.4; 500 x 300 x 5000 9.9 (4) / 12.7; 256 x 4096 x 4096 11.1 (2) / 12.4;
// whole stay 128 x 2048 x 2048 7.7 (2) / 7.5, 256 x 2048 x 2048 8.3 (2) / 8.0
// and 500 x 4096 x 4096 15.1 (2) / 13.7.
void split_tokens(int64_t rows, Args& a, int parts, int clusters, int64_t* cost, int* chosen) {
  if (a.k_blocks < parts) return;
  for (int bn = 32; bn <= kMaxN; bn += 32) {
    if ((rows + bn - 1) / bn * a.c_tiles > clusters) continue;
    const int64_t split = static_cast<int64_t>((a.k_blocks + parts - 1) / parts) * (bn + 256) + 1800 + 16 * bn;
    if (split < *cost) {
      *cost = split;
      *chosen = parts;
      a.tokens_per_tile = bn;
    }
    return;
  }
}

// The rows that row_index names, one after another at a pitch of `chunks` 16-byte
// pieces; zeros where x has no such row. A warp a row, four pieces of it in
// flight a lane. The rows are taken from `stripes` ranges in turn (as many as
// there are groups): a group's rows are in token order, so that the groups come
// to the same tokens at about the same time, while L2 holds their rows (196608
// rows of 2048 bytes, 64 even groups: 92 us with 80 MB of x read from memory,
// 111 us and 299 MB in the rows' own order; skewed groups 110 us, 237 MB).
__global__ void __launch_bounds__(256) gather_rows_kernel(const int8_t* x, int64_t ldx, int64_t x_rows,
                                                          const int* row_index, int rows, int stripes, int chunks,
                                                          uint4* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const int per = (rows + stripes - 1) / stripes;
  const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x / 32);
  for (int i = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < per * stripes; i += warps) {
    const int r = i % stripes * per + i / stripes;
    if (r >= rows) continue;
    const int64_t src = row_index[r];
    const bool in = src >= 0 && src < x_rows;
    const uint4* from = reinterpret_cast<const uint4*>(x + (in ? src : 0) * ldx);
    uint4* to = out + static_cast<int64_t>(r) * chunks;
    for (int c0 = lane; c0 < chunks; c0 += 128) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        v[u] = in && c0 + 32 * u < chunks ? from[c0 + 32 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + 32 * u < chunks) to[c0 + 32 * u] = v[u];
    }
  }
}

template <bool kGated, bool kBf16>
cudaError_t launch(const W8a8& p, cudaStream_t stream) {
  int pairs = 0;
  cudaError_t st = resident_clusters<kGated, kBf16, 1>(&pairs);
  if (st != cudaSuccess) return st;
  const int8_t* x = p.x;
  int64_t ldx = p.ldx;
  if (p.row_index != nullptr) {
    ldx = (p.k + 15) / 16 * 16;
    const int64_t blocks = (p.rows + 7) / 8, most = static_cast<int64_t>(pairs) * 2 * 8;
    st = launch_pdl(gather_rows_kernel, static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream, p.x,
                    p.ldx, p.x_rows, p.row_index, static_cast<int>(p.rows), static_cast<int>(p.groups),
                    static_cast<int>(ldx / 16), reinterpret_cast<uint4*>(p.workspace));
    if (st != cudaSuccess) return st;
    x = p.workspace;
  }
  Args a{};
  a.p = p;
  a.channels = kGated ? kBM : 2 * kBM;
  a.c_tiles = static_cast<int>((p.n + a.channels - 1) / a.channels);
  a.k_blocks = static_cast<int>((p.k + kBK - 1) / kBK);
  int64_t cost = 0;
  a.tokens_per_tile = choose_tokens(p.rows, p.groups, a.c_tiles, pairs, &cost);
  int parts = 1;  // of K
  if constexpr (!kGated) {
    if (p.starts == nullptr) {  // dense: the tiles are known here
      cost *= a.k_blocks;
      int clusters = 0;
      if ((st = resident_clusters<kGated, kBf16, 2>(&clusters)) != cudaSuccess) return st;
      split_tokens(p.rows, a, 2, clusters, &cost, &parts);
      if ((st = resident_clusters<kGated, kBf16, 4>(&clusters)) != cudaSuccess) return st;
      split_tokens(p.rows, a, 4, clusters, &cost, &parts);
    }
  }
  // Boxes that no tile can need are left unset: a map costs the call 0.15 us.
  const bool ok = make_int8_tmap(&a.x, x, p.rows, p.k, ldx, kBoxRows) &&
                  (a.tokens_per_tile < 128 || make_int8_tmap(&a.x_wide, x, p.rows, p.k, ldx, 64)) &&
                  (a.tokens_per_tile < kMaxN || make_int8_tmap(&a.x_half, x, p.rows, p.k, ldx, kMaxN / 2)) &&
                  make_int8_tmap(&a.w, p.w, p.groups * p.n, p.k, p.ldw, kGated ? kBM / 2 : kBM) &&
                  (!kGated || make_int8_tmap(&a.up, p.w_up, p.groups * p.n, p.k, p.ldw, kBM / 2));
  if (!ok) return cudaErrorInvalidValue;
  auto aligned = [](const void* base, int64_t ld) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld * (kBf16 ? 2 : 4) % 16 == 0;
  };
  a.tma_store = kBf16 && aligned(p.y, p.ldy);
  // (With K in parts a warp's units do not follow one another as the residual's slots do.)
  a.tma_residual = !kBf16 && !kGated && parts == 1 && p.residual != nullptr && aligned(p.residual, p.ldr);
  if (a.tma_store && !make_tile_tmap(&a.y, p.y, true, p.rows, p.n, p.ldy, kGated ? kUnit / 2 : kUnit))
    return cudaErrorInvalidValue;
  if (a.tma_residual && !make_tile_tmap(&a.residual, p.residual, false, p.rows, p.n, p.ldr, kRows32))
    return cudaErrorInvalidValue;
  if constexpr (!kGated) {
    const unsigned tiles = static_cast<unsigned>((p.rows + a.tokens_per_tile - 1) / a.tokens_per_tile * a.c_tiles);
    if (parts == 2)
      return launch_pdl(w8a8_gemm_kernel<kGated, kBf16, 2>, tiles * 4, kThreads, kSmem<kGated, kBf16>, stream, a);
    if (parts == 4)
      return launch_pdl(w8a8_gemm_kernel<kGated, kBf16, 4>, tiles * 8, kThreads, kSmem<kGated, kBf16>, stream, a);
  }
  const int64_t most =
      (p.rows / a.tokens_per_tile + (p.groups < p.rows ? p.groups : p.rows)) * static_cast<int64_t>(a.c_tiles);
  const unsigned blocks = 2u * static_cast<unsigned>(most < pairs ? most : pairs);
  return launch_pdl(w8a8_gemm_kernel<kGated, kBf16, 1>, blocks, kThreads, kSmem<kGated, kBf16>, stream, a);
}

}  // namespace

namespace {
// Which kernel: w8a8_rows.cu reads the weights once per 8 rows (dense: up to 32)
// of a group, with little to set up; the kernel above takes 5.6 us or more.
// Measured in us, rows against this one. Dense, n x k: 1 row 2048 x 2048 2.9 / 6.4,
// 102400 x 2048 36 / 39; 8 rows 8192 x 2048 6.1 / 7.4, 4096 x 8192 11.0 / 13.4; 16
// rows 2048 x 2048 4.1 / 6.3, 4096 x 4096 7.4 / 8.4, 2048 x 8192 11.8 / 8.7, 8192
// x 1024 7.2 / 5.8, 8192 x 2048 8.3 / 7.4; 32 rows 1000 x 1000 4.8 / 6.2, 2048 x
// 2048 6.4 / 6.4, 4096 x 2048 7.2 / 7.4, 2048 x 4096 10.5 / 7.2. Groups: 64 of 2 x 1024 x 2048 gated, 6
// rows 7.6 / 12.1, 60 rows 37 / 38, 240 rows 46 / 52; 64 of 2048 x 1024, 6 rows
// 6.2 / 9.7, 96 rows 23.5 / 25.7, 240 rows 30.5 / 29.7; 16 of 1024 x 2048, 32
// rows 9.7 / 11.5, 128 rows 14.8 / 11.5; 8 of those, 30 rows 7.7 / 9.8, 60 9.8 / 9.9.
// These groups were routed at random. The rule has only their mean size, the sizes
// being on the device, and that kernel reads a group's weights again for every 8
// of its rows. 64 groups of 2048 x 1024, then gated ones of 1024 x 2048 with a row
// index: 96 rows, all groups alike, 29.0 / 25.7 and 45.0 / 52.0, in four groups
// 16.0 / 7.2 and 35.4 / 12.9, in one 43.8 / 7.5 and 111 / 13.9; 256 rows in one
// group 112 / 8.9 and 274 / 16.4.
// Dense gated products (a layer's shared expert) have no form for more than 8
// rows at a time there: a layer with one of 2 x 2048 x 2048 takes 121.7 us at 17 rows and
// 155.2 at 32, with that product here 116.6 and 146.2.
bool few_rows_grouped(int64_t rows, int64_t groups) { return rows <= 256 && rows <= 4 * groups; }
bool few_rows(const W8a8& p) {
  if (p.starts != nullptr) return few_rows_grouped(p.rows, p.groups);
  return p.rows <= 8 || (p.n <= 4096 && ((p.rows <= 16 && p.k <= 4096) || (p.rows <= 32 && p.k <= 2048)));
}
}  // namespace

size_t w8a8_gather_bytes(int64_t rows, int64_t groups, int64_t k) {
  return few_rows_grouped(rows, groups) ? 0 : static_cast<size_t>(rows) * static_cast<size_t>((k + 15) / 16 * 16);
}

cudaError_t prepare_w8a8() {
  int n = 0;
  cudaError_t st = resident_clusters<false, false, 1>(&n);
  if (st == cudaSuccess) st = resident_clusters<false, true, 1>(&n);
  if (st == cudaSuccess) st = resident_clusters<true, false, 1>(&n);
  if (st == cudaSuccess) st = resident_clusters<true, true, 1>(&n);
  if (st == cudaSuccess) st = resident_clusters<false, false, 2>(&n);
  if (st == cudaSuccess) st = resident_clusters<false, true, 2>(&n);
  if (st == cudaSuccess) st = resident_clusters<false, false, 4>(&n);
  if (st == cudaSuccess) st = resident_clusters<false, true, 4>(&n);
  return st;
}

cudaError_t launch_w8a8(const W8a8& p, cudaStream_t stream) {
  if (p.rows == 0 || p.n == 0) return cudaSuccess;
  if (few_rows(p)) return launch_w8a8_rows(p, stream);
  if (p.w_up != nullptr) return p.y_bf16 ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
  return p.y_bf16 ? launch<false, true>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace uocr_b200
