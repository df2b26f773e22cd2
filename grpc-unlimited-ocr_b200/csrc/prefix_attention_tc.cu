// Attention behind shared prefixes for many rows, on the tensor cores
// (uocr_prefix_attention; prefix_attention.cu chooses).
//
// A block takes 256 rows (a row and a query head of one key/value head each) as
// two tiles of 128 and runs the prefix's keys past them, 128 at a time:
//   S = Q K^T   tcgen05.mma, Q and K in shared memory, S in TMEM
//   P = exp2(S - m), in registers; the sum l; P in bf16 over S in TMEM
//   O += P V    tcgen05.mma, P in TMEM, V in shared memory, O in TMEM
// One warp brings keys and values by TMA, one lane issues the MMAs, and one
// warpgroup a tile does the exponentials, a thread a row, so that a row's maximum
// and sum need no exchange. The two tiles take turns: while one is exponentiated
// the other is multiplied.
//
// m is the maximum of the tiles seen when it last had to move: O and l are
// rescaled only where a later score exceeds it by more than 2^8, which fp32 and
// bf16 hold without loss, and which hardly happens after the first tile.
//
// Work is cut by units of one tile pair and 128 keys, counted through over
// prefixes, heads and rows, the same number for every block, whatever the
// lengths: a block's share may begin and end inside a range of keys, and the
// parts of a row meet in the join's slots.
#include <algorithm>

#include "prefix_attention.cuh"
#include "tc.cuh"
#include "tc_gemm.h"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kTcRows = kAttentionTcRows;  // of a block: two tiles
constexpr int kTileRows = kTcRows / 2;
constexpr int kTcKeys = 128;
constexpr int kSlots = 4;        // shared-memory slots of 128 keys or values
constexpr int kTcThreads = 384;  // a warpgroup for copies and MMAs, two of rows
constexpr float kSlack = 8.0f;   // log2 of what a score may exceed m by
// The register file's shares, a thread's, after the launch's 168 of each: 128 * 56 + 256 * 224 = 384 * 168.
constexpr int kLaunchRegs = 168, kFewRegs = 56, kManyRegs = 224;
constexpr uint32_t kTmemAll = 512;

// O of N = kDim columns (+)= P in TMEM . V in shared memory (K = 16 keys).
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Values [128 keys][64 dims] per 16 KB as TMA leaves them, as the B operand with
// N = dims contiguous (MN-major, 128-byte swizzle): 64-dim chunks 16 KB apart
// (the leading offset), 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(kTcKeys * 128 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
constexpr uint32_t kBMajorMn = 1u << 16;  // instruction descriptor: B is MN-major

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_addr(bar))
      : "memory");
}

// 32 columns of this warp's lanes, without the wait.
__device__ __forceinline__ void tmem_ld32_async(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// The wait; what was loaded passes through it, so that no use of it moves above.
template <int kCount>
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[kCount]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < kCount; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two values in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

struct __align__(8) TcBarriers {
  uint64_t full[kSlots];
  uint64_t empty[kSlots];
  uint64_t s_full[2];  // a tile's scores are there, and all MMAs before them are done
  uint64_t p_half[2];  // the weights of its first 64 keys are there
  uint64_t p_full[2];  // the others'
  uint64_t o_done;     // a segment's MMAs are done
  uint64_t drain;
};

// A run of a block's units within one range of keys.
struct Segment {
  int first_row, start, count;  // rows: vr = row * group + head of the prefix's rows, `count` from `start`
  int prefix, kv_head;
  int tile0, tile1, tiles;      // of 128 keys: [tile0, tile1) of `tiles`
  int len;
  int slot, used;               // of the join; how many the range's rows use
};                              // tile0 == tile1: there is none

struct TcArgs {
  CUtensorMap k, v;
  Attention a;
};

// A prefix: its rows and keys.
struct Prefix {
  int rows, first_row, len;
  int pairs, tiles;  // of 256 rows, of 128 keys
};
// The units of prefix p: (key/value heads) x (row tile pairs) x (key tiles).
__device__ __forceinline__ unsigned units_of(const Attention& a, int p, Prefix* x) {
  if (p >= a.prefixes) return 0;
  x->rows = prefix_rows_of(a, p, &x->first_row);
  x->len = prefix_len_of(a, p);
  x->pairs = (x->rows * a.group + kTcRows - 1) / kTcRows;
  x->tiles = max(1, (x->len + kTcKeys - 1) / kTcKeys);  // an empty prefix still has a part: no keys
  return static_cast<unsigned>(a.kv_heads) * x->pairs * x->tiles;
}
__device__ __forceinline__ unsigned warp_scan(unsigned v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const unsigned other = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += other;
  }
  return v;
}

// What the scheduling warp keeps: the first 32 prefixes, which mostly are all.
struct Schedule {
  Prefix mine;
  unsigned units, upto;  // of this lane's prefix, inclusive sum
  unsigned unit, end, share;
};

__device__ __forceinline__ Schedule make_schedule(const Attention& a) {
  const int lane = threadIdx.x & 31;
  Schedule c{};
  c.units = units_of(a, lane, &c.mine);
  c.upto = warp_scan(c.units);
  unsigned total = __shfl_sync(0xffffffffu, c.upto, 31);
  int most = c.mine.pairs > 0 ? c.mine.tiles : 1;
  for (int p = 32 + lane; p < (a.prefixes + 31) / 32 * 32; p += 32) {
    Prefix x{};
    total += __reduce_add_sync(0xffffffffu, units_of(a, p, &x));
    if (x.pairs > 0) most = max(most, x.tiles);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  // No range of keys meets more than prefix_slots blocks.
  c.share = max(max((total + gridDim.x - 1) / gridDim.x, (most + a.prefix_slots - 2u) / (a.prefix_slots - 1u)), 1u);
  c.unit = min(total, blockIdx.x * c.share);
  c.end = min(total, c.unit + c.share);
  return c;
}

// By the scheduling warp: the block's next segment.
__device__ __forceinline__ void next_segment(const Attention& a, Schedule& c, Segment* s) {
  const int lane = threadIdx.x & 31;
  if (c.unit >= c.end) {
    if (lane == 0) s->tile0 = s->tile1 = 0;
    __syncwarp();
    return;
  }
  unsigned before = 0;
  for (int p0 = 0; p0 < a.prefixes; p0 += 32) {
    Prefix x = c.mine;
    unsigned n = c.units, upto = c.upto;
    if (p0 > 0) {
      n = units_of(a, p0 + lane, &x);
      upto = before + warp_scan(n);
    }
    if (c.unit < upto && c.unit >= upto - n) {
      const unsigned local = c.unit - (upto - n), range = local / x.tiles, tile0 = local - range * x.tiles;
      const unsigned first = c.unit - tile0, head = range / x.pairs;  // first: the range's first unit
      s->prefix = p0 + lane;
      s->kv_head = static_cast<int>(head);
      s->first_row = x.first_row;
      s->start = static_cast<int>(range - head * x.pairs) * kTcRows;
      s->count = min(kTcRows, x.rows * a.group - s->start);
      s->tiles = x.tiles;
      s->tile0 = static_cast<int>(tile0);
      s->tile1 = static_cast<int>(tile0 + min(x.tiles - tile0, c.end - c.unit));
      s->len = x.len;
      const unsigned block0 = first / c.share;
      s->slot = static_cast<int>(blockIdx.x - block0);
      s->used = static_cast<int>((first + x.tiles - 1) / c.share - block0) + 1;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
    if (c.unit < before) break;
  }
  __syncwarp();
  c.unit += s->tile1 - s->tile0;
}

template <int kDim>
__global__ void __launch_bounds__(kTcThreads, 1) attention_tc_kernel(const __grid_constant__ TcArgs args) {
  constexpr int kHalves = kDim / 64;
  constexpr uint32_t kHalfBytes = kTcKeys * 128;           // 128 rows x 64 dims
  constexpr uint32_t kSlotBytes = kHalves * kHalfBytes;
  extern __shared__ unsigned char dyn_raw[];
  __shared__ TcBarriers bars;
  __shared__ Segment segs[2];  // the one that is worked on, and the one after it
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;
  const Attention& a = args.a;
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_tiles = smem;                        // [2][kSlotBytes]
  unsigned char* slots = smem + 2 * kSlotBytes;         // [kSlots][kSlotBytes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_half[t], kTileRows);
      mbar_init(&bars.p_full[t], kTileRows);
    }
    mbar_init(&bars.o_done, 1);
    mbar_init(&bars.drain, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&tmem_holder, kTmemAll);
  pdl_wait();
  pdl_launch_dependents();
  Schedule schedule{};
  if (warp == 2) {
    schedule = make_schedule(a);
    next_segment(a, schedule, &segs[0]);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  // Counters that run on over the segments: a slot's or a tile's use number gives its barrier's phase. The two kinds
  // of warpgroup keep to code of their own from here on, with the same barriers in it: their registers differ.
  uint32_t fills = 0, rounds[2] = {0, 0}, segments = 0;
  uint32_t issued = 0;  // fills that have been asked for
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    uint32_t ahead = 0;  // fills of the segment that were asked for before it began
    for (;; ++segments) {
      const Segment s = segs[segments & 1];
      const int tiles = s.tile1 - s.tile0, pair = s.count > kTileRows ? 2 : 1;
      if (tiles == 0 || abort_flag != 0) break;
      if (warp == 0) {
        // ---- keys and values: K, V, K, V, ... The last tile ends with the prefix: it begins among keys that were there
        // before, which are masked, and nothing behind the prefix is read. ----
        auto fill = [&](const Segment& of, uint32_t first, uint32_t k) {
          const uint32_t n = first + k, slot = n % kSlots;
          if (!mbar_wait(&bars.empty[slot], (n / kSlots & 1) ^ 1)) {
            raise_error(a.err, kDevWaitTimeout, 90, of.prefix, static_cast<int>(k));
            abort_flag = 1;
            return false;
          }
          const int tile = of.tile0 + static_cast<int>(k / 2);
          const int key = tile == of.tiles - 1 ? of.len - kTcKeys : tile * kTcKeys;
          mbar_arrive_expect_tx(&bars.full[slot], kSlotBytes);
          issued = n + 1;
          for (int h = 0; h < kHalves; ++h)
            tma_load_4d(slots + slot * kSlotBytes + h * kHalfBytes, k % 2 == 0 ? &args.k : &args.v, h * 64, key,
                        of.kv_head, of.prefix, &bars.full[slot]);
          return true;
        };
        bool ok = true;
        if (lane == 0)
          for (uint32_t k = ahead; k < 2u * tiles && ok; ++k) ok = fill(s, fills, k);
        __syncwarp();
        named_bar_sync(1, 64);  // the segment after this is known
        const Segment next = segs[(segments + 1) & 1];
        // Its first fills wait for no more than this one's products.
        ahead = min(2u * (next.tile1 - next.tile0), static_cast<uint32_t>(kSlots));
        if (lane == 0)
          for (uint32_t k = 0; k < ahead && ok; ++k) ok = fill(next, fills + 2 * tiles, k);
        __syncwarp();
      } else if (warp == 2) {
        next_segment(a, schedule, &segs[(segments + 1) & 1]);
        named_bar_sync(1, 64);
      }
      if (warp == 1) named_bar_sync(2, 32 + 256);  // its Q is there
      if (warp == 1 && lane == 0) {
        // ---- MMAs. Those of one thread run in the order of their issue: the scores of a tile's next keys, written
        // where its weights lie, come behind the product that reads these. ----
        constexpr uint32_t kScores = bf16_idesc(kTileRows, kTcKeys);
        constexpr uint32_t kOutput = bf16_idesc(kTileRows, kDim) | kBMajorMn;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
          if (ok && !mbar_wait(bar, parity)) {
            raise_error(a.err, kDevWaitTimeout, site, s.prefix, static_cast<int>(parity));
            abort_flag = 1;
            ok = false;
          }
          tc_fence_after();
        };
        auto landed = [&](uint32_t n) { wait(&bars.full[n % kSlots], n / kSlots & 1, 91); };
        auto scores = [&](int t, uint32_t n) {
          const uint32_t ks = smem_addr(slots + n % kSlots * kSlotBytes);
          const uint32_t qs = smem_addr(q_tiles + t * kSlotBytes);
#pragma unroll
          for (int k = 0; k < kDim / 16; ++k) {
            const uint32_t off = (k / 4) * kHalfBytes + (k % 4) * 32;
            umma_bf16(tmem + t * kTcKeys, sw128_kmajor_desc(qs + off), sw128_kmajor_desc(ks + off), kScores, k != 0);
          }
          umma_commit(&bars.s_full[t]);
        };
        landed(fills);
        if (ok) {
          for (int t = 0; t < pair; ++t) scores(t, fills);
          umma_commit(&bars.empty[fills % kSlots]);
        }
        for (int i = 0; i < tiles && ok; ++i) {
          const uint32_t v = fills + 2 * i + 1, next_k = v + 1;
          landed(v);
          if (i + 1 < tiles) landed(next_k);
          for (int t = 0; t < pair && ok; ++t) {
            const uint32_t vs = smem_addr(slots + v % kSlots * kSlotBytes);
            for (int half = 0; half < 2; ++half) {
              wait(half == 0 ? &bars.p_half[t] : &bars.p_full[t], (rounds[t] + i) & 1, 92);
              if (!ok) break;
#pragma unroll
              for (int k = half * kTcKeys / 32; k < (half + 1) * kTcKeys / 32; ++k)
                umma_bf16_ts(tmem + 2 * kTcKeys + t * kDim, tmem + t * kTcKeys + k * 8,
                             sw128_mnmajor_desc(vs + k * 16 * 128), kOutput, (i | k) != 0);
            }
            if (!ok) break;
            if (t == pair - 1) umma_commit(&bars.empty[v % kSlots]);
            if (i + 1 < tiles) {
              scores(t, next_k);
              if (t == pair - 1) umma_commit(&bars.empty[next_k % kSlots]);
            }
          }
        }
        umma_commit(&bars.o_done);
      }
      fills += 2 * tiles;
      rounds[0] += tiles;
      if (pair == 2) rounds[1] += tiles;
      __syncwarp();
      __syncthreads();  // its TMEM and Q have been read
      tc_fence_after();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    for (;; ++segments) {
      const Segment& s = segs[segments & 1];
      const int tiles = s.tile1 - s.tile0, pair = s.count > kTileRows ? 2 : 1;
      if (tiles == 0 || abort_flag != 0) break;
      {
        // Q, swizzled like the copies of K: neighbouring threads bring a row's 16-byte pieces.
        constexpr int kPieces = kDim / 8, kStep = 256 / kPieces;
        const int thread = threadIdx.x - 128, c = thread % kPieces;
        uint4 v[kTcRows / kStep];
#pragma unroll
        for (int i = 0; i < kTcRows / kStep; ++i) {
          const int r = i * kStep + thread / kPieces, vr = s.start + r;
          const __nv_bfloat16* src = a.q + static_cast<int64_t>(s.first_row + vr / a.group) * a.ldq +
                                     (s.kv_head * a.group + vr % a.group) * kDim;
          v[i] = r < s.count ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kTcRows / kStep; ++i) {
          const int r = i * kStep + thread / kPieces, in_tile = r % kTileRows;
          if (r < pair * kTileRows)
            *reinterpret_cast<uint4*>(q_tiles + (r / kTileRows) * kSlotBytes + (c / 8) * kHalfBytes + in_tile * 128 +
                                      ((c ^ in_tile) & 7) * 16) = v[i];
        }
        fence_proxy_async_smem();
      }
      named_bar_sync(2, 32 + 256);  // its Q is there
      // ---- a row: its scores to weights ----
      const int t = (warp - 4) / 4, r = threadIdx.x - 128;
      if (t < pair) {
        const uint32_t at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_at = at + t * kTcKeys, o_at = at + 2 * kTcKeys + t * kDim;
        float m = -INFINITY, l = 0.0f;  // m: of the raw scores
        const int skip_last = s.tile1 == s.tiles ? s.tiles * kTcKeys - s.len : 0;
        bool ok = true;
        for (int i = 0; i < tiles; ++i) {
          if (!__all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], (rounds[0] + i) & 1))) {
            raise_error(a.err, kDevWaitTimeout, 93, s.prefix, i);
            abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t x[kTcKeys];
#pragma unroll
          for (int c = 0; c < kTcKeys; c += 32) tmem_ld32_async(s_at + c, x + c);
          tmem_ld_done(x);
          const int skip = i == tiles - 1 ? skip_last : 0;
          if (skip > 0) {
#pragma unroll
            for (int c = 0; c < kTcKeys; ++c)
              if (c < skip) x[c] = __float_as_uint(-INFINITY);
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kTcKeys; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              top[e] = fmaxf(top[e], fmaxf(__uint_as_float(x[c + e]), __uint_as_float(x[c + 4 + e])));
          const float peak = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          if (i == 0) {
            m = peak;
          } else {
            const bool moves = (peak - m) * a.scale_log2 > kSlack;  // also where m is -inf
            if (__any_sync(0xffffffffu, moves)) {
              const float to = fmaxf(m, peak);
              const float f = to == m ? 1.0f : exp2_fast((m - to) * a.scale_log2);
              m = to;
              l *= f;
#pragma unroll
              for (int c = 0; c < kDim; c += 32) {
                uint32_t o[32];
                tmem_ld32_async(o_at + c, o);
                tmem_ld_done(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(o_at + c, o);
              }
            }
          }
          const float shift = m == -INFINITY ? 0.0f : m * a.scale_log2;
          const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), shift2 = make_float2(-shift, -shift);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // The products with the first half's values start while the second half is exponentiated.
            uint32_t p[kTcKeys / 4];
#pragma unroll
            for (int c = 0; c < kTcKeys / 2; c += 2) {
              const int at = half * (kTcKeys / 2) + c;
              float2 e = fma2(make_float2(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), scale2, shift2);
              e.x = exp2_fast(e.x);
              e.y = exp2_fast(e.y);
              sum[c / 2 % 2] = add2(sum[c / 2 % 2], e);
              p[c / 2] = pack2(e.x, e.y);
            }
            tmem_st32(s_at + half * (kTcKeys / 4), p);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(half == 0 ? &bars.p_half[t] : &bars.p_full[t]);
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&bars.o_done, segments & 1))) {
          raise_error(a.err, kDevWaitTimeout, 94, s.prefix, 0);
          abort_flag = 1;
          ok = false;
        }
        tc_fence_after();
        const int vr = s.start + r;
        const int64_t cell =
            (static_cast<int64_t>(s.first_row + vr / a.group) * a.heads + s.kv_head * a.group + vr % a.group) * a.slots;
        const bool mine = r < s.count && ok;
        if (mine) {
          a.part_ml[cell + s.slot] = make_float2(m == -INFINITY ? m : m * a.scale_log2, l);
          if (s.tile0 == 0)  // the slots that no block comes to
            for (int k = s.used; k < a.prefix_slots; ++k) a.part_ml[cell + k] = make_float2(-INFINITY, 0.0f);
        }
        // 32 columns at a time through 4 KB of the tile's Q, which is done with, so that a store instruction covers whole
        // lines: four rows of 128 bytes.
        unsigned char* stage = q_tiles + t * kSlotBytes + (warp & 3) * 4096;
        const int64_t mine_at = mine ? (cell + s.slot) * kDim : -1;
#pragma unroll 1
        for (int c = 0; c < kDim; c += 32) {
          uint32_t o[32];
          tmem_ld32_async(o_at + c, o);
          tmem_ld_done(o);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int row = k * 4 + lane / 8, e = lane & 7;
            const int64_t to = __shfl_sync(0xffffffffu, mine_at, row);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((e ^ (row & 7)) << 4));
            if (to >= 0) *reinterpret_cast<uint4*>(a.part_o + to + c + e * 4) = v;
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      if ((warp - 4) / 4 < pair) rounds[0] += tiles;  // of this warp's tile
      __syncthreads();  // its TMEM and Q have been read
    }
  }
  if (abort_flag != 0 && lane == 0) {
    // A wait gave up: nothing may be in flight when the block ends.
    if (warp == 0)
      for (uint32_t n = issued > kSlots ? issued - kSlots : 0; n < issued; ++n)
        mbar_wait(&bars.full[n % kSlots], n / kSlots & 1);
    if (warp == 1) {
      umma_commit(&bars.drain);
      mbar_wait(&bars.drain, 0);
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemAll);
  }
}

template <int kDim>
cudaError_t launch(const TcArgs& t, unsigned blocks, cudaStream_t stream) {
  constexpr size_t kSmem = static_cast<size_t>(2 + kSlots) * kTcKeys * kDim * 2 + 1024;
  static bool done[kMaxDevices] = {};
  int dev = 0;
  cudaError_t st = cudaGetDevice(&dev);
  if (st != cudaSuccess) return st;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!done[dev]) {
    // The shares of the register file have to add up to the launch's.
    cudaFuncAttributes attr{};
    if ((st = cudaFuncGetAttributes(&attr, attention_tc_kernel<kDim>)) != cudaSuccess) return st;
    if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidKernelImage;
    if ((st = allow_max_dynamic_smem(attention_tc_kernel<kDim>)) != cudaSuccess) return st;
    done[dev] = true;
  }
  return launch_pdl(attention_tc_kernel<kDim>, blocks, kTcThreads, kSmem, stream, t);
}

}  // namespace

cudaError_t launch_attention_tc(const Attention& a, int dim, unsigned blocks, cudaStream_t stream) {
  TcArgs t{};
  t.a = a;
  if (!make_cache_tmap(&t.k, a.prefix_k, dim, a.prefix_capacity, a.kv_heads, a.prefixes, a.prefix_head_stride,
                       a.prefix_stride, kTcKeys) ||
      !make_cache_tmap(&t.v, a.prefix_v, dim, a.prefix_capacity, a.kv_heads, a.prefixes, a.prefix_head_stride,
                       a.prefix_stride, kTcKeys))
    return cudaErrorInvalidValue;
  return dim == 64 ? launch<64>(t, blocks, stream) : launch<128>(t, blocks, stream);
}

}  // namespace uocr_b200
