// Attention behind shared prefixes for many rows, on the tensor cores
// (uocr_prefix_attention; prefix_attention.cu chooses).
//
// A block takes rows (a row and a query head of one key/value head each) in two
// tiles of 128 and runs the prefix's keys past them, 128 at a time:
//   S = Q K^T   tcgen05.mma, Q and K in shared memory, S in TMEM
//   P = exp2(S - m), in registers; the sum l; P in bf16 over S in TMEM
//   O += P V    tcgen05.mma, P in TMEM, V in shared memory, O in TMEM
// One warp brings keys and values by TMA, one lane issues the MMAs, and one
// warpgroup a tile does the exponentials, a thread a row, so that a row's maximum
// and sum need no exchange. The two tiles take turns: while one is exponentiated
// the other is multiplied. With many rows the tiles are 256 rows and see the same
// keys. With up to 128 they are the same rows, and see every other 128 keys each:
// their two parts of a row meet in the join like those of two blocks.
//
// m is the maximum of the tiles seen when it last had to move: O and l are
// rescaled only where a later score exceeds it by more than 2^8, which fp32 and
// bf16 hold without loss, and which hardly happens after the first tile. Scores far
// from 0 are taken from a base of their row (`base` below).
//
// Work is cut by units of the tiles' rows and 128 keys, counted through over
// prefixes, heads and rows, the same number for every block, whatever the
// lengths: a block's share may begin and end inside a range of keys, and the
// parts of a row meet in the join's slots. What a range costs a block besides its
// keys (bringing Q, the first scores, the way out of O) counts as units before its
// first key, so that a block with two ranges has fewer keys.
#include <algorithm>
#include <type_traits>

#include "prefix_attention.cuh"
#include "tc.cuh"
#include "tc_gemm.h"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kTileRows = kAttentionTcRows;
// What a range costs besides its keys, in units: 128 keys take 1.8 us for two tiles of rows, 0.6 (the memory's rate) where
// the tiles split them. With 4, 6, 8 and 12 for the latter sixteen pages take 53.3, 53.6, 54.3 and 55.3 us, with 2, 3 and
// 4 for the former prompts on a page 108.6, 108.4 and 108.4, a document 51.3, 51.2 and 52.1.
__host__ __device__ __forceinline__ unsigned range_units(const Attention& a) { return a.split ? 4 : 3; }
constexpr int kTcKeys = 128;
constexpr int kSlots = 4;        // shared-memory slots of 128 keys or values
constexpr int kTcThreads = 384;  // a warpgroup for copies and MMAs, two of rows
constexpr float kSlack = 8.0f;   // log2 of what a score may exceed m by
// The register file's shares, a thread's, after the launch's 168 of each: 128 * 56 + 256 * 224 = 384 * 168.
constexpr int kLaunchRegs = 168, kFewRegs = 56, kManyRegs = 224;
constexpr uint32_t kTmemAll = 512;

// Shared-memory matrix descriptors in halves: the low word names the address and
// the leading offset and is what moves from product to product; one lane issues
// them all, and every operation on a descriptor is time between two products.
// Keys and Q: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart. Values
// [128 keys][64 dims] per 16 KB as TMA leaves them: B with N = dims contiguous
// (MN-major), 64-dim chunks 16 KB apart (the leading offset), 8-key groups 1024
// bytes apart.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // group stride, version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t kmajor_low(uint32_t saddr) { return (saddr >> 4 & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t mnmajor_low(uint32_t saddr) {
  return (saddr >> 4 & 0x3FFFu) | (static_cast<uint32_t>(kTcKeys * 128 >> 4) << 16);
}
constexpr uint32_t kBMajorMn = 1u << 16;  // instruction descriptor: B is MN-major

// The MMA warp runs as a whole and one lane's predicate lets the instruction
// through, so that its operands stay uniform registers.
// D in TMEM (+)= A in shared memory . B in shared memory, K = 16.
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t d_tmem, uint32_t a_low, uint32_t b_low,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh), "r"(leader)
      : "memory");
}
// D in TMEM (+)= A in TMEM . B in shared memory, K = 16.
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

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

// The greatest of three; NaN where one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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
  int ranges, tiles;  // of rows (a head's), of 128 keys
};
// The units of prefix p: (key/value heads) x (ranges) x (key tiles and what a range costs).
__device__ __forceinline__ unsigned units_of(const Attention& a, int p, Prefix* x) {
  if (p >= a.prefixes) return 0;
  x->rows = prefix_rows_of(a, p, &x->first_row);
  x->len = prefix_len_of(a, p);
  const int of_range = a.split ? kTileRows : 2 * kTileRows;
  x->ranges = (x->rows * a.group + of_range - 1) / of_range;
  x->tiles = max(1, (x->len + kTcKeys - 1) / kTcKeys);  // an empty prefix still has a part: no keys
  return static_cast<unsigned>(a.kv_heads) * x->ranges * (x->tiles + range_units(a));
}
__device__ __forceinline__ unsigned warp_scan(unsigned v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const unsigned other = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v = add_saturated(v, other);
  }
  return v;
}

// Where a segment's key tile i and its values lie among the fills. Same keys for both tiles: K0 V0 K1 V1 ...; every
// other one: K0 K1 V0 K2 V1 K3 ... V.
__device__ __forceinline__ uint32_t key_fill(bool split, int i) { return split ? (i < 2 ? i : 2 * i - 1) : 2 * i; }
__device__ __forceinline__ uint32_t value_fill(bool split, int i, int tiles) {
  return split ? (i == tiles - 1 ? 2 * i + 1 : 2 * i + 2) : 2 * i + 1;
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
  int most = c.mine.ranges > 0 ? c.mine.tiles : 1;
  for (int p = 32 + lane; p < (a.prefixes + 31) / 32 * 32; p += 32) {
    Prefix x{};
    total = add_saturated(total, __shfl_sync(0xffffffffu, warp_scan(units_of(a, p, &x)), 31));
    if (x.ranges > 0) most = max(most, x.tiles);
  }
  if (total > a.tc_units) total = 0;  // row offsets out of order: recorded
  most = __reduce_max_sync(0xffffffffu, most);
  // No range of keys meets more blocks than there are slots for (two of a block that splits the keys).
  const unsigned blocks = a.split ? a.prefix_slots / 2 : a.prefix_slots;
  c.share = max(max((total + gridDim.x - 1) / gridDim.x, (most + blocks - 2) / (blocks - 1)), 2u);
  c.unit = min(total, blockIdx.x * c.share);
  c.end = min(total, c.unit + c.share);
  return c;
}

// By the scheduling warp: the block's next segment.
__device__ __forceinline__ void next_segment(const Attention& a, Schedule& c, Segment* s) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) s->tile0 = s->tile1 = 0;
  __syncwarp();
  unsigned before = 0;
  for (int p0 = 0; p0 < a.prefixes && c.unit < c.end; p0 += 32) {
    Prefix x = c.mine;
    unsigned n = c.units, upto = c.upto;
    if (p0 > 0) {
      n = units_of(a, p0 + lane, &x);
      upto = before + warp_scan(n);
    }
    const bool mine = c.unit < upto && c.unit >= upto - n;
    unsigned to = 0;
    if (mine) {
      const unsigned each = x.tiles + range_units(a);
      const unsigned local = c.unit - (upto - n), range = local / each, at = local - range * each;
      const unsigned first = c.unit - at + range_units(a), head = range / x.ranges;  // first: the unit of the first keys
      const int of_range = a.split ? kTileRows : 2 * kTileRows;
      to = min(c.unit - at + each, c.end);
      s->prefix = p0 + lane;
      s->kv_head = static_cast<int>(head);
      s->first_row = x.first_row;
      s->start = static_cast<int>(range - head * x.ranges) * of_range;
      s->count = min(of_range, x.rows * a.group - s->start);
      s->tiles = x.tiles;
      s->tile0 = static_cast<int>(max(c.unit, first) - first);
      s->tile1 = static_cast<int>(max(to, first) - first);  // none where the share ends before the first keys
      s->len = x.len;
      const unsigned block0 = first / c.share;
      s->slot = static_cast<int>(blockIdx.x - block0);
      s->used = static_cast<int>((first + x.tiles - 1) / c.share - block0) + 1;
    }
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    before = __shfl_sync(0xffffffffu, upto, 31);
    if (who != 0) {
      c.unit = __shfl_sync(0xffffffffu, to, __ffs(who) - 1);
      break;
    }
  }
  __syncwarp();
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
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
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
  if (threadIdx.x == 32 * 3) {  // parameters of the launch, there before any grid has ended
    prefetch_tmap(&args.k);
    prefetch_tmap(&args.v);
  }
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
  const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(tmem_holder)));
  // Counters that run on over the segments: a slot's or a tile's use number gives its barrier's phase. The two kinds
  // of warpgroup keep to code of their own from here on, with the same barriers in it: their registers differ.
  uint32_t fills = 0, rounds[2] = {0, 0}, segments = 0;
  uint32_t issued = 0;  // fills that have been asked for
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    const uint32_t leader = elect_one() ? 1u : 0u;
    uint32_t ahead = 0;  // fills of the segment that were asked for before it began
    for (;; ++segments) {
      const Segment s = segs[segments & 1];
      const int tiles = uniform(s.tile1 - s.tile0), pair = uniform(s.count) > kTileRows ? 2 : 1;
      if (tiles == 0 || abort_flag != 0) break;
      if (warp == 0) {
        // ---- keys and values, in the order in which the products take them (key_fill, value_fill). The last tile ends
        // with the prefix: it begins among keys that the tile before it has too, and nothing behind the prefix is read. ----
        auto fill = [&](const Segment& of, uint32_t first, uint32_t k) {
          const uint32_t n = first + k, slot = n % kSlots;
          if (!mbar_wait(&bars.empty[slot], (n / kSlots & 1) ^ 1)) {
            raise_error(a.err, kDevWaitTimeout, 90, of.prefix, static_cast<int>(k));
            abort_flag = 1;
            return false;
          }
          const uint32_t all = of.tile1 - of.tile0;
          uint32_t j = k / 2;
          bool keys = k % 2 == 0;
          if (a.split && all > 1) {
            keys = k < 2 || (k % 2 == 1 && k < 2 * all - 2);
            j = k < 2 ? k : keys ? k / 2 + 1 : k == 2 * all - 1 ? all - 1 : k / 2 - 1;
          }
          const int tile = of.tile0 + static_cast<int>(j);
          const int key = tile == of.tiles - 1 ? of.len - kTcKeys : tile * kTcKeys;
          mbar_arrive_expect_tx(&bars.full[slot], kSlotBytes);
          issued = n + 1;
          for (int h = 0; h < kHalves; ++h)
            tma_load_4d(slots + slot * kSlotBytes + h * kHalfBytes, keys ? &args.k : &args.v, h * 64, key,
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
      if (warp == 1) {
        named_bar_sync(2, 32 + 256);  // its Q is there
        // ---- MMAs. Those of one thread run in the order of their issue: the scores of a tile's next keys, written
        // where its weights lie, come behind the product that reads these. ----
        constexpr uint32_t kScores = bf16_idesc(kTileRows, kTcKeys);
        constexpr uint32_t kOutput = bf16_idesc(kTileRows, kDim) | kBMajorMn;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
          if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity))) {
            if (leader) raise_error(a.err, kDevWaitTimeout, site, s.prefix, static_cast<int>(parity));
            abort_flag = 1;
            ok = false;
          }
          tc_fence_after();
        };
        auto landed = [&](uint32_t n) { wait(&bars.full[n % kSlots], n / kSlots & 1, 91); };
        const uint32_t q_low = kmajor_low(smem_addr(q_tiles)), k_low = kmajor_low(smem_addr(slots)),
                       v_low = mnmajor_low(smem_addr(slots));
        auto scores = [&](auto tile, uint32_t n) {
          constexpr int t = decltype(tile)::value;
          const uint32_t k0 = k_low + n % kSlots * (kSlotBytes >> 4);
          const uint32_t q0 = q_low + (t == 0 || a.split ? 0u : kSlotBytes >> 4);
#pragma unroll
          for (int k = 0; k < kDim / 16; ++k) {
            const uint32_t off = ((k / 4) * kHalfBytes + (k % 4) * 32) >> 4;
            umma_ss(leader, tmem + t * kTcKeys, q0 + off, k0 + off, kScores, k != 0);
          }
          umma_commit_by(leader, &bars.s_full[t]);
        };
        // A tile's turn: the output of its keys `i`, then the scores of its next ones.
        auto turn = [&](auto tile, int i, uint32_t round) {
          constexpr int t = decltype(tile)::value;
          const bool last_use = a.split || t == pair - 1;
          const uint32_t v = fills + value_fill(a.split, i, tiles);
          landed(v);
          const uint32_t v0 = v_low + v % kSlots * (kSlotBytes >> 4);
          for (int half = 0; half < 2; ++half) {
            wait(half == 0 ? &bars.p_half[t] : &bars.p_full[t], (rounds[t] + round) & 1, 92);
            if (!ok) return;
#pragma unroll
            for (int k = 0; k < kTcKeys / 32; ++k)
              umma_ts(leader, tmem + 2 * kTcKeys + t * kDim, tmem + t * kTcKeys + half * (kTcKeys / 4) + k * 8,
                      v0 + half * (kTcKeys / 2 * 128 >> 4) + (k * 16 * 128 >> 4), kOutput, round | half | k);
          }
          if (last_use) umma_commit_by(leader, &bars.empty[v % kSlots]);
          const int next = a.split ? i + 2 : i + 1;
          if (next >= tiles) return;
          const uint32_t n = fills + key_fill(a.split, next);
          landed(n);
          if (!ok) return;
          scores(tile, n);
          if (last_use) umma_commit_by(leader, &bars.empty[n % kSlots]);
        };
        constexpr std::integral_constant<int, 0> k0{};
        constexpr std::integral_constant<int, 1> k1{};
        landed(fills);
        if (ok) scores(k0, fills);
        if (a.split) {
          umma_commit_by(leader, &bars.empty[fills % kSlots]);
          if (tiles > 1) {
            landed(fills + 1);
            if (ok) scores(k1, fills + 1);
            umma_commit_by(leader, &bars.empty[(fills + 1) % kSlots]);
          }
        } else {
          if (ok && pair == 2) scores(k1, fills);
          umma_commit_by(leader, &bars.empty[fills % kSlots]);
        }
        const int step = a.split ? 2 : 1;
        for (int i = 0, round = 0; i < tiles && ok; i += step, ++round) {
          turn(k0, i, round);
          if (ok && (a.split ? i + 1 < tiles : pair == 2)) turn(k1, a.split ? i + 1 : i, round);
        }
        umma_commit_by(leader, &bars.o_done);
      }
      fills += 2 * tiles;
      rounds[0] += a.split ? (tiles + 1) / 2 : tiles;
      rounds[1] += a.split ? tiles / 2 : pair == 2 ? tiles : 0;
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
        // Q, swizzled like the copies of K: neighbouring threads bring a row's 16-byte pieces, all of them under way at
        // once. In a loop and without a division a row: unrolled, with the rows in registers, the first of these
        // instructions were what a block waited for (4.2 us before the first scores of a document, now 2.7).
        constexpr int kPieces = kDim / 8, kStep = 256 / kPieces;
        const int thread = threadIdx.x - 128, c = thread % kPieces;
        const int per_row = kStep / a.group, per_head = kStep % a.group;
        int r = thread / kPieces, row = (s.start + r) / a.group, head = (s.start + r) % a.group;
#pragma unroll 1
        for (; r < pair * kTileRows; r += kStep) {
          const int in_tile = r % kTileRows;
          const __nv_bfloat16* src = a.q + static_cast<int64_t>(s.first_row + row) * a.ldq + (s.kv_head * a.group + head) * kDim + c * 8;
          cp_async16_or_zero(q_tiles + (r / kTileRows) * kSlotBytes + (c / 8) * kHalfBytes + in_tile * 128 +
                                 ((c ^ in_tile) & 7) * 16,
                             r < s.count ? src : a.q, r < s.count);
          row += per_row;
          head += per_head;
          if (head >= a.group) {
            head -= a.group;
            ++row;
          }
        }
        cp_async_commit();
        cp_async_wait_all();
        fence_proxy_async_smem();
      }
      named_bar_sync(2, 32 + 256);  // its Q is there
      // ---- a row: its scores to weights ----
      const int t = (warp - 4) / 4, in_tile = (threadIdx.x - 128) % kTileRows, r = a.split ? in_tile : threadIdx.x - 128;
      const int my_rounds = a.split ? (tiles + 1 - t) / 2 : t < pair ? tiles : 0;
      if (my_rounds > 0 || a.split) {
        const uint32_t at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_at = at + t * kTcKeys, o_at = at + 2 * kTcKeys + t * kDim;
        float m = -INFINITY, l = 0.0f;  // m: of the raw scores
        const bool has_rows = r - lane < s.count;  // of this warp
        // Rounds times two, where the tiles split the keys: of the prefix's last tile but one, if it shares keys with the
        // last. (An empty prefix is told apart below.)
        const int doubled = a.split ? 1 : 0;
        const int shared_from = s.len % kTcKeys != 0 ? s.tiles - 2 - s.tile0 - (a.split ? t : 0) : 1 << 30;
        // The exponents are fma(x, scale, -m scale). What the rounding of m scale is off by, all weights of a row have in
        // common: up to 2^-14 where it is at most 1024, but from 2^31 on more than their range. A row whose m is farther
        // off takes it from its scores (`base`), and the tile is read anew.
        float base = 0.0f;
        bool based = false;  // one of the warp's rows
        auto is_far = [&](float m) { return fabsf(m * a.scale_log2) > 1024.0f && m != -INFINITY; };
        bool ok = true;
        for (int i = 0; i < my_rounds; ++i) {
          if (!__all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], (rounds[0] + i) & 1))) {
            raise_error(a.err, kDevWaitTimeout, 93, s.prefix, i);
            abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          if (!has_rows) {
            mbar_arrive(&bars.p_half[t]);
            mbar_arrive(&bars.p_full[t]);
            continue;
          }
          uint32_t x[kTcKeys];
          for (bool again = true; again;) {
            again = false;
#pragma unroll
            for (int c = 0; c < kTcKeys; c += 32) tmem_ld32_async(s_at + c, x + c);
            tmem_ld_done(x);
            // A key that the prefix's last two tiles both have counts half in each. (Not 0 in one of them: an infinite value
            // times 0 is NaN.) In a single tile they lie before the first key, where the copy brings zeros, and are none.
            if (based || (i << doubled) >= shared_from) {
              const int twice = -s.len & (kTcKeys - 1);
              const float less = s.tiles == 1 ? INFINITY : 1.0f / a.scale_log2;
              if (based) {
#pragma unroll
                for (int c = 0; c < kTcKeys; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) - base);
              }
              if ((i << doubled) > shared_from) {  // the last
#pragma unroll
                for (int c = 0; c < kTcKeys; ++c)
                  if (c < twice) x[c] = __float_as_uint(__uint_as_float(x[c]) - less);
              } else if ((i << doubled) == shared_from) {
#pragma unroll
                for (int c = 0; c < kTcKeys; ++c)
                  if (c >= kTcKeys - twice) x[c] = __float_as_uint(__uint_as_float(x[c]) - less);
              }
            }
            float top[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = __uint_as_float(x[e]);
#pragma unroll
            for (int c = 4; c < kTcKeys; c += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                top[e] = max3_nan(top[e], __uint_as_float(x[c + e]),
                                  __uint_as_float(x[c + 4 + e < kTcKeys ? c + 4 + e : c + e]));
            const float peak = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]);
            if (i == 0) {
              m = peak;
              again = __any_sync(0xffffffffu, is_far(m));
            } else {
              const bool moves = !((peak - m) * a.scale_log2 <= kSlack) && peak != m;  // also where m is -inf or one is NaN
              if (__any_sync(0xffffffffu, moves)) {
                const float to = max3_nan(m, peak, peak);  // NaN: every weight of the row becomes one
                const float f = to == m ? 1.0f : exp2_fast((m - to) * a.scale_log2);
                m = to;
                l *= f;
                again = __any_sync(0xffffffffu, is_far(m));
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
            if (again) {
              tmem_st_wait();  // O may be rescaled once more
              based = true;
              if (is_far(m)) {
                base += m;
                m = l == 0.0f ? -INFINITY : 0.0f;
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
        const int slot = a.split ? 2 * s.slot + t : s.slot;
        const bool mine = r < s.count && ok;
        if (mine) {
          a.part_ml[cell + slot] = m == -INFINITY || s.len == 0
                                       ? make_float2(-INFINITY, 0.0f)
                                       : make_float2(__fmul_rn(base, a.scale_log2) + m * a.scale_log2, l);
          if (s.tile0 == 0 && (t == 0 || !a.split))  // the slots that no block comes to
            for (int k = a.split ? 2 * s.used : s.used; k < a.prefix_slots; ++k)
              a.part_ml[cell + k] = make_float2(-INFINITY, 0.0f);
        }
        // 32 columns at a time through 4 KB of the tile's Q, which is done with, so that a store instruction covers whole
        // lines: four rows of 128 bytes.
        unsigned char* stage = q_tiles + t * kSlotBytes + (warp & 3) * 4096;
        const int64_t mine_at = mine ? (cell + slot) * kDim : -1;
#pragma unroll 1
        for (int c = 0; c < (has_rows && my_rounds > 0 ? kDim : 0); c += 32) {
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
      rounds[0] += my_rounds;  // of this warp's tile
      __syncthreads();  // its TMEM and Q have been read
    }
  }
  if (abort_flag != 0) {
    // A wait gave up: nothing may be in flight when the block ends.
    if (warp == 0 && lane == 0)
      for (uint32_t n = issued > kSlots ? issued - kSlots : 0; n < issued; ++n)
        mbar_wait(&bars.full[n % kSlots], n / kSlots & 1);
    if (warp == 1) {  // by the lane that issued the MMAs
      umma_commit_by(elect_one() ? 1u : 0u, &bars.drain);
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
  // The shares of the register file have to add up to the launch's.
  static const int registers = [] {
    cudaFuncAttributes attr{};
    return cudaFuncGetAttributes(&attr, attention_tc_kernel<kDim>) == cudaSuccess ? attr.numRegs : 0;
  }();
  if (registers != kLaunchRegs) return cudaErrorInvalidKernelImage;
  const cudaError_t st = allow_max_dynamic_smem_once<attention_tc_kernel<kDim>>();
  if (st != cudaSuccess) return st;
  return launch_pdl(attention_tc_kernel<kDim>, blocks, kTcThreads, kSmem, stream, t);
}

}  // namespace

cudaError_t launch_attention_tc(const Attention& a, int dim, unsigned blocks, cudaStream_t stream) {
  TcArgs t{};
  t.a = a;
  const int64_t of_range = a.split ? kTileRows : 2 * kTileRows, tiles = (a.prefix_capacity + kTcKeys - 1) / kTcKeys;
  const int64_t ranges = static_cast<int64_t>(a.rows) * a.group / of_range + std::min(a.prefixes, a.rows);
  t.a.tc_units = static_cast<unsigned>(a.kv_heads * ranges * (tiles + range_units(a)));
  if (!make_cache_tmap(&t.k, a.prefix_k, dim, a.prefix_capacity, a.kv_heads, a.prefixes, a.prefix_head_stride,
                       a.prefix_stride, kTcKeys) ||
      !make_cache_tmap(&t.v, a.prefix_v, dim, a.prefix_capacity, a.kv_heads, a.prefixes, a.prefix_head_stride,
                       a.prefix_stride, kTcKeys))
    return cudaErrorInvalidValue;
  return dim == 64 ? launch<64>(t, blocks, stream) : launch<128>(t, blocks, stream);
}

}  // namespace uocr_b200
