// Attention of sequences that share prefixes (uocr_prefix_attention): the
// kernel for few rows, the join of partial results, and the choice of parts.
//
// With the rows of all sequences behind a prefix in one tile, the prefix's keys
// and values are read once for all of them. A softmax over a set of keys is the
// join of softmaxes over parts of it: from (m_i, l_i, o_i), the parts' maxima,
// sums of exp(s - m_i) and unnormalised outputs,
//   m = max m_i,  l = sum l_i exp(m_i - m),  o = sum o_i exp(m_i - m) / l.
// So prefixes and own keys are cut into as many shares as the card holds blocks,
// and a second kernel joins a row's parts.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "prefix_attention.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kThreads = 128;
constexpr int kKeys = 64;    // of a stage
constexpr int kStages = 2;
constexpr int kBlocks = 3;   // of an SM
// Stages of a block at least: with 2, 3, 4 and 6 the four rows of a page take 13.1, 14.0, 12.8 and 15.3 us, the parts
// that fewer make costing the join more than the blocks save.
constexpr int kMinShare = 4;
constexpr int kMaxSlots = 160;  // of a row: the most that a plan gives its prefix and its own keys
constexpr int kMaxPrefixSlots = 64, kMaxOwnSlots = 32, kMaxTcSlots = 128;
static_assert(kMaxPrefixSlots + kMaxOwnSlots <= kMaxSlots && kMaxTcSlots + kMaxOwnSlots <= kMaxSlots, "");

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p))
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p))
               : "memory");
}
// An 8 x 8 matrix of 16-bit elements in a warp's registers, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// A run of a block's units within one range of keys: rows x heads of one
// key/value head (vr = row * group + head, `count` of them from `start`).
struct Segment {
  int first_row, start, count;
  int kv_head;
  int of;                // the prefix or sequence
  bool own;
  int key0, key1;        // the block's part
  int limit0;            // keys the row at first_row sees; each row after it sees one more (own keys), or the same
  int all_see;           // keys that every row of the tile sees
  int slot, used, slots;  // of the join: this one, how many the range's blocks use, how many there are
  bool first;            // the range's first block
  int stages;            // of the block's share
};

// The work is counted through in units of a tile of rows and a stage of keys,
// over the prefixes (where this kernel has them), then the sequences' own keys,
// and every block takes the same number of units, whatever the lengths.
struct Grid {
  int prefixes, sequences;  // that this launch has to do with
  unsigned most_units;      // there can be
  // 1: launched behind a kernel of the same call, which this one takes nothing from. That kernel lets this one start
  // when it has itself waited for all work before the call, so the wait for it can come last.
  int late_wait;
};

// A prefix or a sequence (index e, the prefixes first): its rows and keys.
struct Source {
  int rows, first_row, keys;
  int tiles, stages;
};

template <int kPrefixRows, int kOwnRows>
__device__ __forceinline__ unsigned source_units(const Attention& a, const Grid& g, int e, Source* s) {
  if (e >= g.prefixes + g.sequences) return 0;
  const bool own = e >= g.prefixes;
  s->rows = own ? rows_of(a, e - g.prefixes, &s->first_row) : prefix_rows_of(a, e, &s->first_row);
  s->keys = own ? len_of(a, e - g.prefixes) : prefix_len_of(a, e);
  const int of_tile = own ? kOwnRows : kPrefixRows;
  s->tiles = (s->rows * a.group + of_tile - 1) / of_tile;
  s->stages = max(1, (s->keys + kKeys - 1) / kKeys);  // without keys there still is a part: none
  return static_cast<unsigned>(a.kv_heads) * s->tiles * s->stages;
}

// Inclusive sums over the block's threads; *total over all. `part`: a sum a warp.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* part, unsigned* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const unsigned other = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v = add_saturated(v, other);
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  *total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) v = add_saturated(v, part[w]);
    *total = add_saturated(*total, part[w]);
  }
  return v;
}

// A segment's keys and values into the ring of padded stages, by cp.async. A thread
// copies 16 bytes of every kStep-th key of a stage. Where its keys lie (with
// ancestry: in any of the caches) is read a fill ahead of the copies, all keys at
// once.
template <int kDim>
struct Feed {
  static constexpr int kPitch = kDim + 8;  // padded: fragment loads without bank conflicts
  static constexpr int kStage = 2 * kKeys * kPitch;
  static constexpr int kStep = kThreads / (kDim / 8), kCopies = kKeys / kStep;
  const Attention& a;
  const Segment& w;
  __nv_bfloat16* ring;
  const __nv_bfloat16* keys;  // of key 0 (with ancestry: in cache 0)
  const __nv_bfloat16* values;
  bool gathers;
  int from[kCopies];

  __device__ __forceinline__ Feed(const Attention& attention, const Segment& segment, unsigned char* raw)
      : a(attention), w(segment), ring(reinterpret_cast<__nv_bfloat16*>(raw)) {
    const int64_t base = w.own ? (a.ancestry != nullptr ? 0 : w.of * a.cache_stride) + w.kv_head * a.head_stride
                               : w.of * a.prefix_stride + w.kv_head * a.prefix_head_stride;
    keys = (w.own ? a.k : a.prefix_k) + base;
    values = (w.own ? a.v : a.prefix_v) + base;
    gathers = w.own && a.ancestry != nullptr;
  }
  __device__ __forceinline__ void look_up(int key) {
    if (!gathers) return;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = key + static_cast<int>(threadIdx.x) / (kDim / 8) + i * kStep;
      from[i] = at < w.key1 ? a.ancestry[w.of * a.ld_ancestry + at] : 0;
    }
  }
  __device__ __forceinline__ void fill(int stage, int key) {
    const int copy_key = threadIdx.x / (kDim / 8), col = threadIdx.x % (kDim / 8) * 8;
    __nv_bfloat16* ks = ring + stage * kStage + copy_key * kPitch + col;
    __nv_bfloat16* vs = ks + kKeys * kPitch;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = key + copy_key + i * kStep;
      const bool valid = at < w.key1;
      int64_t off = valid ? static_cast<int64_t>(at) * kDim + col : 0;
      if (gathers) {
        int cache = from[i];
        if (valid && (cache < 0 || cache >= a.caches)) {
          raise_error(a.err, kDevBadIndex, kSiteAncestor, w.of, cache);
          cache = w.of < a.caches ? w.of : 0;
        }
        off += cache * a.cache_stride;
      }
      cp_async16_or_zero(ks + i * kStep * kPitch, keys + off, valid);
      cp_async16_or_zero(vs + i * kStep * kPitch, values + off, valid);
    }
  }
  __device__ __forceinline__ void start() {
    look_up(w.key0);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (w.key0 + s * kKeys < w.key1) fill(s, w.key0 + s * kKeys);
      cp_async_commit();
      look_up(w.key0 + (s + 1) * kKeys);
    }
  }
  // While the stage with `key` is worked on.
  __device__ __forceinline__ void next(int key, int stage) {
    const int ahead = key + (kStages - 1) * kKeys;
    if (ahead < w.key1) fill((stage + kStages - 1) % kStages, ahead);
    cp_async_commit();
    look_up(ahead + kKeys);
  }
};

// The end of a block that has all own keys of its rows: their kAlong parts, which
// the warps leave in the ring's place, and the prefix's are joined and the rows
// written.
template <int kDim, int kRows, int kAlong, int kBlock = kThreads>  // kBlock: threads
struct LastJoin {
  float* os;        // [kAlong][kRows][kDim]
  float2* mls;      // [kAlong][kRows]
  float* own;       // [kAlong][kRows] factors
  float* scales;    // [kRows] 1 / sum
  float2* factors;  // [kRows][prefix_slots] the parts' maxima and sums, then their factors in the maxima's place
  __device__ __forceinline__ explicit LastJoin(unsigned char* raw) {
    os = reinterpret_cast<float*>(raw);
    mls = reinterpret_cast<float2*>(os + kAlong * kRows * kDim);
    own = reinterpret_cast<float*>(mls + kAlong * kRows);
    scales = own + kAlong * kRows;
    factors = reinterpret_cast<float2*>(scales + kRows);
  }
  static constexpr size_t bytes(int prefix_slots) {
    return kAlong * kRows * (kDim * 4 + 8 + 4) + kRows * (4 + prefix_slots * 8);
  }
  // live: a word of shared memory that nobody else uses by now
  __device__ __forceinline__ void run(const Attention& a, const Segment& w, uint32_t* live, bool late_wait) const {
    auto cell = [&](int r) {  // of the tile's row r
      const int vr = w.start + r;
      const int64_t row = w.first_row + vr / a.group;
      return row * a.heads + w.kv_head * a.group + vr % a.group;
    };
    if (late_wait) pdl_wait();  // the prefix's parts
    __syncthreads();
    for (int c0 = threadIdx.x; c0 < w.count * a.prefix_slots; c0 += 8 * kBlock) {
      float2 ml[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = c0 + k * kBlock;
        if (c < w.count * a.prefix_slots) ml[k] = a.part_ml[cell(c / a.prefix_slots) * a.slots + c % a.prefix_slots];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + k * kBlock < w.count * a.prefix_slots) factors[c0 + k * kBlock] = ml[k];
    }
    if (threadIdx.x == 0) *live = 0;  // from here on: one more than the last slot with keys
    __syncthreads();
    {
      // All rows at once, kLanes neighbouring threads each.
      constexpr int kLanes = kBlock / kRows;
      const int r = threadIdx.x / kLanes, at = threadIdx.x % kLanes;
      float2* ml = factors + r * a.prefix_slots;
      const int slots = r < w.count ? a.prefix_slots : 0;
      float top = -INFINITY;
      for (int i = at; i < kAlong; i += kLanes) top = fmaxf(top, mls[i * kRows + r].x);
      for (int s = at; s < slots; s += kLanes) top = fmaxf(top, ml[s].x);
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float shift = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      int used = 0;
      for (int i = at; i < kAlong; i += kLanes) {
        const float2 p = mls[i * kRows + r];
        const float f = exp2_fast(p.x - shift);
        sum = fmaf(p.y, f, sum);
        own[i * kRows + r] = f;
      }
      for (int s = at; s < slots; s += kLanes) {
        const float2 p = ml[s];
        const float f = exp2_fast(p.x - shift);
        sum = fmaf(p.y, f, sum);
        // A part without keys has no output: its factor is told apart from one that has underflowed.
        ml[s].x = p.x == -INFINITY ? -1.0f : f;
        if (p.x != -INFINITY) used = s + 1;
      }
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (used > 0) atomicMax(live, static_cast<uint32_t>(used));
      if (at == 0 && r < w.count) {
        scales[r] = sum != 0.0f ? 1.0f / sum : 0.0f;
        if (a.lse != nullptr)
          a.lse[cell(r)] = sum != 0.0f ? (top + log2f(sum)) * 0.69314718055994530942f : -INFINITY;
      }
    }
    __syncthreads();
    const int live_slots = static_cast<int>(*live);
    // 16 pieces of parts under way at a time: of four rows where there are many, of one where there are few.
    auto join_rows = [&](auto rows_at_once) {
      constexpr int kR = decltype(rows_at_once)::value, kAhead = 16 / kR;
      constexpr int kPieces = kDim / 4, kGroups = kBlock / kPieces;
      const int col = threadIdx.x % kPieces * 4;
      for (int r0 = threadIdx.x / kPieces * kR; r0 < w.count; r0 += kGroups * kR) {
        float4 acc[kR];
        const float* parts[kR];
        auto add = [](float4& sum, const float4& v, float f) {
          sum.x = fmaf(v.x, f, sum.x), sum.y = fmaf(v.y, f, sum.y);
          sum.z = fmaf(v.z, f, sum.z), sum.w = fmaf(v.w, f, sum.w);
        };
#pragma unroll
        for (int k = 0; k < kR; ++k) {
          acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          parts[k] = a.part_o + cell(r0 + k) * a.slots * kDim + col;
        }
        for (int s0 = 0; s0 < live_slots; s0 += kAhead) {
          float4 v[kR][kAhead];
          float f[kR][kAhead];
#pragma unroll
          for (int k = 0; k < kR; ++k)
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
              f[k][s] = r0 + k < w.count && s0 + s < live_slots ? factors[(r0 + k) * a.prefix_slots + s0 + s].x : -1.0f;
              v[k][s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (!(f[k][s] < 0.0f)) v[k][s] = *reinterpret_cast<const float4*>(parts[k] + (s0 + s) * kDim);
            }
#pragma unroll
          for (int k = 0; k < kR; ++k)
#pragma unroll
            for (int s = 0; s < kAhead; ++s) add(acc[k], v[k][s], f[k][s]);
        }
#pragma unroll
        for (int k = 0; k < kR; ++k) {
          const int r = r0 + k;
          if (r >= w.count) break;
#pragma unroll
          for (int i = 0; i < kAlong; ++i)
            add(acc[k], *reinterpret_cast<const float4*>(os + (i * kRows + r) * kDim + col), own[i * kRows + r]);
          const int vr = w.start + r;
          const float scale = scales[r];
          __nv_bfloat16* out = a.out + static_cast<int64_t>(w.first_row + vr / a.group) * a.ldo +
                               (w.kv_head * a.group + vr % a.group) * kDim + col;
          *reinterpret_cast<uint2*>(out) =
              make_uint2(pack2(acc[k].x * scale, acc[k].y * scale), pack2(acc[k].z * scale, acc[k].w * scale));
        }
      }
    };
    if (w.count > 16)
      join_rows(std::integral_constant<int, 4>{});
    else
      join_rows(std::integral_constant<int, 1>{});
  }
};

// A segment. 4 warps: kWarpRows of them side by side along the rows (16 each),
// the others along a stage's keys, each with its own running maximum, sum and
// output in registers; keys and values in a ring of padded stages filled by
// cp.async. mma.sync and not tcgen05: a tile has 16 to 64 rows, of which a tcgen05
// tile would use an eighth to a half.
// With kLast the block has all own keys of its rows: it joins the prefix's parts
// to them (behind the wait for the kernel that makes them, with late_wait) and
// writes the rows; else it writes its part.
template <int kDim, int kWarpRows, bool kLast>
__device__ __forceinline__ void attend(const Attention& a, const Segment& seg, unsigned char* raw, uint32_t* odd_keys,
                                       bool late_wait) {
  const Segment w = seg;  // in registers
  constexpr int kRows = 16 * kWarpRows, kWarpKeys = kKeys / (4 / kWarpRows);
  constexpr int kPitch = kDim + 8;  // padded: fragment loads without bank conflicts
  constexpr int kStage = 2 * kKeys * kPitch;
  __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, tq = lane & 3;
  const int row0 = warp % kWarpRows * 16, warp_key = warp / kWarpRows * kWarpKeys;

  Feed<kDim> feed(a, w, raw);
  feed.start();

  // This thread's two rows of the warp's tile, and the warp's queries as A fragments.
  int limit[2];
  const __nv_bfloat16* src[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int vr = w.start + row0 + gr + 8 * i;
    const bool valid = row0 + gr + 8 * i < w.count;
    const int row = vr / a.group, head = w.kv_head * a.group + vr % a.group;
    limit[i] = !valid ? 0 : w.own ? w.limit0 + row : w.limit0;
    src[i] = valid ? a.q + (w.first_row + row) * a.ldq + head * kDim : nullptr;
  }
  uint32_t qa[kDim / 16][4];
#pragma unroll
  for (int kk = 0; kk < kDim / 16; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qa[kk][i] = src[i & 1] != nullptr
                      ? *reinterpret_cast<const uint32_t*>(src[i & 1] + kk * 16 + (i >> 1) * 8 + 2 * tq)
                      : 0u;
  float o[kDim / 8][4];
#pragma unroll
  for (int d = 0; d < kDim / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  int stage = 0;
  for (int key = w.key0; key < w.key1; key += kKeys) {
    cp_async_wait<kStages - 2>();
    __syncthreads();  // the stage has landed for all, and the one filled next has been read by all
    feed.next(key, stage);
    const __nv_bfloat16* ks = ring + stage * kStage + warp_key * kPitch;
    const __nv_bfloat16* vs = ks + kKeys * kPitch;
    stage = (stage + 1) % kStages;
    float s[kWarpKeys / 8][4];
#pragma unroll
    for (int nt = 0; nt < kWarpKeys / 8; nt += 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = s[nt + 1][e] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < kDim / 16; ++kk) {
        // matrices: keys nt * 8 .. + 7 at dims 0-7 and 8-15, then the next 8 keys
        uint32_t b[4];
        ldmatrix_x4(b, ks + (nt * 8 + (lane & 7) + (lane >> 4) * 8) * kPitch + kk * 16 + (lane >> 3 & 1) * 8);
        mma_bf16(s[nt], qa[kk], b[0], b[1]);
        mma_bf16(s[nt + 1], qa[kk], b[2], b[3]);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < kWarpKeys / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = key + warp_key + nt * 8 + 2 * tq + (e & 1);
        s[nt][e] = at < min(limit[e >> 1], w.key1) ? s[nt][e] * a.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[nt][e]);
      }
    float alpha[2], shift[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      top[i] = fmaxf(m[i], top[i]);
      shift[i] = top[i] == -INFINITY ? 0.0f : top[i];  // no key yet: 2^(-inf - 0) = 0
      alpha[i] = exp2_fast(m[i] - shift[i]);
      m[i] = top[i];
      l[i] *= alpha[i];
    }
#pragma unroll
    for (int nt = 0; nt < kWarpKeys / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = exp2_fast(s[nt][e] - shift[e >> 1]);
        l[e >> 1] += s[nt][e];
      }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {  // the maxima soon stay
#pragma unroll
      for (int d = 0; d < kDim / 8; ++d) {
        o[d][0] *= alpha[0];
        o[d][1] *= alpha[0];
        o[d][2] *= alpha[1];
        o[d][3] *= alpha[1];
      }
    }
    // A key that only some of the tile's rows see has the weight 0 in the others, which an infinite or NaN value
    // would turn into a NaN: such values are added apart, where they are seen, and are 0 in the products.
    if (key + kKeys > w.all_see && w.all_see < w.key1) {
      __nv_bfloat16* whole = ring + ((stage + kStages - 1) % kStages) * kStage + kKeys * kPitch;
      if (threadIdx.x < kKeys / 32) odd_keys[threadIdx.x] = 0;
      __syncthreads();
      bool odd = false;
#pragma unroll 4
      for (int c = threadIdx.x; c < kKeys * (kDim / 8); c += kThreads) {
        const int r = c / (kDim / 8);
        const uint4 u = *reinterpret_cast<const uint4*>(whole + r * kPitch + c % (kDim / 8) * 8);
        // An exponent of ones, plus one in its last place, carries into the sign's.
        auto ones = [](uint32_t x) { return (x & 0x7f807f80u) + 0x00800080u; };
        if (((ones(u.x) | ones(u.y) | ones(u.z) | ones(u.w)) & 0x80008000u) != 0) {
          atomicOr(&odd_keys[r / 32], 1u << (r & 31));
          odd = true;
        }
      }
      if (__syncthreads_or(odd)) {
        // p * v of an infinite or NaN v is v, whatever p > 0.
#pragma unroll 1
        for (int r = warp_key; r < warp_key + kWarpKeys; ++r) {
          if ((odd_keys[r / 32] >> (r & 31) & 1) == 0) continue;
#pragma unroll
          for (int d = 0; d < kDim / 8; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = __bfloat162float(whole[r * kPitch + d * 8 + 2 * tq + (e & 1)]);
              if (!isfinite(v) && key + r < limit[e >> 1]) o[d][e] += v;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < kKeys * kDim; c += kThreads) {
          __nv_bfloat16* v = whole + c / kDim * kPitch + c % kDim;
          if (!isfinite(__bfloat162float(*v))) *v = __float2bfloat16_rn(0.0f);
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int kk = 0; kk < kWarpKeys / 16; ++kk) {
      // The weights as the tensor cores take them: rounded to bf16, like the values they meet.
      const uint32_t p[4] = {pack2(s[2 * kk][0], s[2 * kk][1]), pack2(s[2 * kk][2], s[2 * kk][3]),
                             pack2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int d = 0; d < kDim / 8; d += 2) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, vs + (kk * 16 + (lane & 15)) * kPitch + d * 8 + (lane >> 4) * 8);
        mma_bf16(o[d], p, b[0], b[1]);
        mma_bf16(o[d + 1], p, b[2], b[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  auto cell = [&](int r) {  // of the tile's row r
    const int vr = w.start + r;
    const int64_t row = w.first_row + vr / a.group;
    return row * a.heads + w.kv_head * a.group + vr % a.group;
  };
  if constexpr (kLast) {
    using Join = LastJoin<kDim, kRows, 4 / kWarpRows>;
    const Join join(raw);
    cp_async_wait_all();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = warp / kWarpRows * kRows + row0 + gr + 8 * i;
      if (tq == 0) join.mls[r] = make_float2(m[i], l[i]);
#pragma unroll
      for (int d = 0; d < kDim / 8; ++d)
        *reinterpret_cast<float2*>(join.os + r * kDim + d * 8 + 2 * tq) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
    }
    join.run(a, w, odd_keys, late_wait);
  } else {
    if (w.first)  // the slots that no block comes to
      for (int c = threadIdx.x; c < w.count * (w.slots - w.used); c += kThreads)
        a.part_ml[cell(c % w.count) * a.slots + w.used + c / w.count] = make_float2(-INFINITY, 0.0f);
    if (w.key0 >= w.key1) {
      for (int r = threadIdx.x; r < w.count; r += kThreads) a.part_ml[cell(r) * a.slots + w.slot] = make_float2(-INFINITY, 0.0f);
      return;
    }
    if constexpr (kWarpRows == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + gr + 8 * i;
        if (r >= w.count) continue;
        const int64_t at = cell(r) * a.slots + w.slot;
        if (tq == 0) a.part_ml[at] = make_float2(m[i], l[i]);
#pragma unroll
        for (int d = 0; d < kDim / 8; ++d)
          *reinterpret_cast<float2*>(a.part_o + at * kDim + d * 8 + 2 * tq) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
      }
    } else {
      // The warps along the keys are joined in shared memory, in the ring's place.
      constexpr int kAlong = 4 / kWarpRows;
      float* os = reinterpret_cast<float*>(raw);                    // [kAlong][kRows][kDim]
      float2* mls = reinterpret_cast<float2*>(os + kAlong * kRows * kDim);  // [kAlong][kRows]
      cp_async_wait_all();
      __syncthreads();
      const int along = warp / kWarpRows;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + gr + 8 * i;
        if (tq == 0) mls[along * kRows + r] = make_float2(m[i], l[i]);
#pragma unroll
        for (int d = 0; d < kDim / 8; ++d)
          *reinterpret_cast<float2*>(os + (along * kRows + r) * kDim + d * 8 + 2 * tq) =
              make_float2(o[d][2 * i], o[d][2 * i + 1]);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < w.count * (kDim / 4); c += kThreads) {
        const int r = c / (kDim / 4), col = c % (kDim / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kAlong; ++i) top = fmaxf(top, mls[i * kRows + r].x);
        const float shift = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kAlong; ++i) {
          const float2 ml = mls[i * kRows + r];
          const float f = exp2_fast(ml.x - shift);
          const float4 v = *reinterpret_cast<const float4*>(os + (i * kRows + r) * kDim + col);
          sum = fmaf(ml.y, f, sum);
          acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
        }
        const int64_t at = cell(r) * a.slots + w.slot;
        if (col == 0) a.part_ml[at] = make_float2(top, sum);
        *reinterpret_cast<float4*>(a.part_o + at * kDim + col) = acc;
      }
    }
  }
}

// At most 8 rows that all see the same own keys (a token's heads): the keys are the
// rows of the tensor-core tiles and the 8 rows their columns, S^T = K Q^T and
// O^T = V^T P^T, half the products and registers of 16 padded rows. Each warp takes
// 16 of a round's keys and brings them itself, into three slots of its own for 16
// keys or values (K V K, then V K V): no barrier before the join, and with 52 KB a
// block of four warps four blocks an SM, so that 512 ranges of own keys are under
// way at once (with three some have to wait for the end of others: sixteen pages
// 58.7 against 53.3 us). A lane reads one key's ancestor, and the copies are a loop: the
// first instructions of a kernel come from memory like its data. Blocks that have an SM to themselves take eight warps and half the
// rounds: four beams 13.9 against 12.8 us.
template <int kDim, int kWarps>
struct FewRing {
  static constexpr int kSlot = 16 * (kDim + 8), kSlots = 3;
  static constexpr size_t kBytes = static_cast<size_t>(kWarps) * kSlots * kSlot * 2;
};
template <int kDim, int kWarps>
__device__ __forceinline__ void attend_few(const Attention& a, unsigned char* raw, uint32_t* free_word, bool late_wait) {
  constexpr int kPitch = kDim + 8, kRows = 8, kRound = 16 * kWarps;
  constexpr int kStep = 32 / (kDim / 8), kCopies = 16 / kStep;  // a lane copies 16 bytes of every kStep-th key
  using Ring = FewRing<kDim, kWarps>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, tq = lane & 3;
  const bool gathers = a.ancestry != nullptr;
  const int copy_key = warp * 16 + lane / (kDim / 8), col = lane % (kDim / 8) * 8;
  Segment w{};  // a sequence's row and a key/value head
  w.of = w.first_row = blockIdx.x / a.kv_heads;
  w.kv_head = blockIdx.x % a.kv_heads;
  w.count = a.group;
  const int64_t base = (gathers ? 0 : w.of * a.cache_stride) + w.kv_head * a.head_stride;
  __nv_bfloat16* const ring = reinterpret_cast<__nv_bfloat16*>(raw) + warp * Ring::kSlots * Ring::kSlot;
  int from = 0;  // the cache of this lane's key of the next round, read ahead of the copies
  auto look_up = [&](int key, int end) {
    const int at = key + warp * 16 + lane;
    if (gathers) from = lane < 16 && at < end ? a.ancestry[w.of * a.ld_ancestry + at] : 0;
  };
  look_up(0, a.capacity);  // beside the length, not behind it: what is no key's is not used
  if (a.capacity > 0) {
    const int n = a.lens[w.of];
    if ((n < 0 || n > a.capacity) && threadIdx.x == 0) raise_error(a.err, kDevBadIndex, kSiteLength, w.of, n);
    w.key1 = min(max(n, 0), a.capacity);
  }
  auto check = [&](int key) {
    if (!gathers || (from >= 0 && from < a.caches)) return;
    if (key + warp * 16 + lane < w.key1) raise_error(a.err, kDevBadIndex, kSiteAncestor, w.of, from);
    from = w.of < a.caches ? w.of : 0;
  };
  auto copy = [&](const __nv_bfloat16* of, int slot, int key) {  // by the whole warp
    __nv_bfloat16* to = ring + slot * Ring::kSlot + lane / (kDim / 8) * kPitch + col;
#pragma unroll 2
    for (int i = 0; i < kCopies; ++i) {
      const int at = key + copy_key + i * kStep;
      const bool valid = at < w.key1;
      int64_t off = valid ? static_cast<int64_t>(at) * kDim + col : 0;
      if (gathers) {
        const int64_t cache = __shfl_sync(0xffffffffu, from, lane / (kDim / 8) + i * kStep);
        off += valid ? cache * a.cache_stride : 0;
      }
      cp_async16_or_zero(to + i * kStep * kPitch, of + base + off, valid);
    }
  };
  check(0);
  if (w.key1 > 0) copy(a.k, 0, 0);
  cp_async_commit();
  if (w.key1 > 0) copy(a.v, 1, 0);
  cp_async_commit();
  look_up(kRound, w.key1);
  uint32_t q[kDim / 16][2];  // row gr
  const __nv_bfloat16* src =
      a.q + static_cast<int64_t>(w.first_row) * a.ldq + (w.kv_head * a.group + w.start + gr) * kDim;
#pragma unroll
  for (int kk = 0; kk < kDim / 16; ++kk)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q[kk][i] = gr < w.count ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + i * 8 + 2 * tq) : 0u;
  float o[kDim / 16][4];
#pragma unroll
  for (int d = 0; d < kDim / 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // rows 2 tq and 2 tq + 1
  int slot = 0;  // of the keys; the values' is the one after it, the next keys' the third
  for (int key = 0; key < w.key1; key += kRound) {
    const int next = key + kRound, slot1 = (slot + 1) % 3, slot2 = (slot + 2) % 3;
    cp_async_wait<1>();
    __syncwarp();  // the keys have landed, the values before them have been read
    check(next);
    if (next < w.key1) copy(a.k, slot2, next);
    cp_async_commit();
    const __nv_bfloat16* ks = ring + slot * Ring::kSlot;
    const __nv_bfloat16* vs = ring + slot1 * Ring::kSlot;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // keys gr, gr + 8 x rows 2 tq, + 1
#pragma unroll
    for (int kk = 0; kk < kDim / 16; ++kk) {
      uint32_t k[4];
      ldmatrix_x4(k, ks + (lane & 15) * kPitch + kk * 16 + (lane >> 4) * 8);
      mma_bf16(s, k, q[kk][0], q[kk][1]);
    }
    const int at = key + warp * 16 + gr;
    float alpha[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = at < w.key1 ? s[i] * a.scale_log2 : -INFINITY;
      s[2 + i] = at + 8 < w.key1 ? s[2 + i] * a.scale_log2 : -INFINITY;
      float top = fmaxf(s[i], s[2 + i]);
#pragma unroll
      for (int off = 4; off < 32; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      top = fmaxf(top, m[i]);
      const float shift = top == -INFINITY ? 0.0f : top;
      alpha[i] = exp2_fast(m[i] - shift);
      m[i] = top;
      s[i] = exp2_fast(s[i] - shift);
      s[2 + i] = exp2_fast(s[2 + i] - shift);
      l[i] = fmaf(l[i], alpha[i], s[i] + s[2 + i]);
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int d = 0; d < kDim / 16; ++d) {
        o[d][0] *= alpha[0];
        o[d][1] *= alpha[1];
        o[d][2] *= alpha[0];
        o[d][3] *= alpha[1];
      }
    }
    const uint32_t p0 = transpose_8x8(pack2(s[0], s[1])), p1 = transpose_8x8(pack2(s[2], s[3]));
    cp_async_wait<1>();
    __syncwarp();  // the values have landed, the keys have been read
    if (next < w.key1) copy(a.v, slot, next);
    cp_async_commit();
    look_up(next + kRound, w.key1);
    slot = slot2;
#pragma unroll
    for (int d = 0; d < kDim / 16; ++d) {
      uint32_t v[4];
      ldmatrix_x4_trans(v, vs + ((lane & 7) + (lane >> 4) * 8) * kPitch + d * 16 + (lane >> 3 & 1) * 8);
      mma_bf16(o[d], v, p0, p1);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int off = 4; off < 32; off *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
  const LastJoin<kDim, kRows, kWarps, 32 * kWarps> join(raw);
  cp_async_wait_all();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = warp * kRows + 2 * tq + i;
    if (gr == 0) join.mls[r] = make_float2(m[i], l[i]);
#pragma unroll
    for (int d = 0; d < kDim / 16; ++d) {
      join.os[r * kDim + d * 16 + gr] = o[d][i];
      join.os[r * kDim + d * 16 + gr + 8] = o[d][2 + i];
    }
  }
  join.run(a, w, free_word, late_wait);
}

template <int kDim, int kPrefixWarps, int kOwnWarps>
__global__ void __launch_bounds__(kThreads, kBlocks) attention_rows_kernel(Attention a, Grid g) {
  constexpr int kPrefixRows = 16 * kPrefixWarps, kOwnRows = 16 * kOwnWarps;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint32_t odd_keys[kKeys / 32];  // keys of the stage with a value that is no finite number
  __shared__ Segment seg;
  __shared__ unsigned part[2][kThreads / 32];
  __shared__ int most[2];  // stages of the longest prefix and sequence
  if (threadIdx.x < 2) most[threadIdx.x] = 1;
  if (!g.late_wait) {
    pdl_wait();
    pdl_launch_dependents();
  }
  __syncthreads();
  const int sources = g.prefixes + g.sequences;
  Source mine{};  // of this thread in the first round, which for few sources is the only one
  const unsigned my_units = source_units<kPrefixRows, kOwnRows>(a, g, threadIdx.x, &mine);
  if (mine.tiles > 0) atomicMax(&most[static_cast<int>(threadIdx.x) >= g.prefixes], mine.stages);
  unsigned rest = 0;
  for (int e = kThreads + threadIdx.x; e < sources; e += kThreads) {
    Source s{};
    rest = add_saturated(rest, source_units<kPrefixRows, kOwnRows>(a, g, e, &s));
    if (s.tiles > 0) atomicMax(&most[e >= g.prefixes], s.stages);
  }
  unsigned first_round, total;
  const unsigned my_upto = block_scan(my_units, part[0], &first_round);
  total = first_round;
  if (sources > kThreads) {
    unsigned others;
    block_scan(rest, part[1], &others);
    total = add_saturated(total, others);
  }
  if (total > g.most_units) total = 0;  // row offsets out of order: recorded
  // No range of keys meets more blocks than there are slots for it.
  const int own_slots = a.slots - a.prefix_slots;
  unsigned share = max((total + gridDim.x - 1) / gridDim.x, static_cast<unsigned>(kMinShare));
  if (g.prefixes > 0) share = max(share, (most[0] + a.prefix_slots - 2u) / (a.prefix_slots - 1u));
  if (g.sequences > 0) share = max(share, (most[1] + own_slots - 2u) / (own_slots - 1u));
  unsigned unit = blockIdx.x * share;
  const unsigned end = min(total, unit + share);
  while (unit < end) {
    unsigned before = 0;
    for (int e0 = 0; e0 < sources; e0 += kThreads) {
      const int e = e0 + threadIdx.x;
      Source s = mine;
      unsigned n = my_units, upto = my_upto, in_round = first_round;
      if (e0 > 0) {
        __syncthreads();  // the sums of the round before have been read
        n = source_units<kPrefixRows, kOwnRows>(a, g, e, &s);
        upto = before + block_scan(n, part[1], &in_round);
      }
      if (unit < upto && unit >= upto - n) {
        const unsigned local = unit - (upto - n), range = local / s.stages, stage0 = local - range * s.stages;
        const unsigned first = unit - stage0, head = range / s.tiles;  // first: the range's first unit
        const int tile = static_cast<int>(range - head * s.tiles);
        const int of_tile = e >= g.prefixes ? kOwnRows : kPrefixRows;
        seg.own = e >= g.prefixes;
        seg.of = seg.own ? e - g.prefixes : e;
        seg.kv_head = static_cast<int>(head);
        seg.first_row = s.first_row;
        seg.start = tile * of_tile;
        seg.count = min(of_tile, s.rows * a.group - seg.start);
        seg.stages = static_cast<int>(min(s.stages - stage0, end - unit));
        int keys = s.keys;
        seg.limit0 = seg.all_see = s.keys;
        if (seg.own) {
          seg.limit0 = s.keys - s.rows + 1;
          seg.all_see = seg.limit0 + seg.start / a.group;
          keys = max(0, seg.limit0 + (seg.start + seg.count - 1) / a.group);  // the tile's last row sees the most
        }
        seg.key0 = min(keys, static_cast<int>(stage0) * kKeys);
        seg.key1 = min(keys, (static_cast<int>(stage0) + seg.stages) * kKeys);
        seg.first = stage0 == 0;
        const unsigned block0 = first / share;
        const int slot0 = seg.own ? a.prefix_slots : 0;
        seg.slot = static_cast<int>(blockIdx.x - block0) + slot0;
        seg.used = static_cast<int>((first + s.stages - 1) / share - block0) + 1 + slot0;
        seg.slots = seg.own ? a.slots : a.prefix_slots;
      }
      before += in_round;
      if (unit < before) break;
    }
    __syncthreads();  // the segment is known
    unit += seg.stages;
    if (kPrefixWarps == kOwnWarps || seg.own)
      attend<kDim, kOwnWarps, false>(a, seg, raw, odd_keys, false);
    else
      attend<kDim, kPrefixWarps, false>(a, seg, raw, odd_keys, false);
    __syncthreads();  // the segment and the ring have been read
  }
  if (g.late_wait) pdl_wait();
}

// A block for all own keys of a tile of a sequence's rows, which also joins the
// prefix's parts and writes the rows. Blocks: tiles of all sequences x heads.
template <int kDim, int kWarps>
__global__ void __launch_bounds__(kThreads, kBlocks) attention_last_kernel(Attention a, int late_wait) {
  constexpr int kRows = 16 * kWarps;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint32_t odd_keys[kKeys / 32];
  __shared__ Segment seg;
  if (!late_wait) pdl_wait();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int tile = blockIdx.x / a.kv_heads;
    if (lane == 0) seg.count = 0;
    __syncwarp();
    auto take = [&](int b, int rows, int first_row, int local) {
      const int len = a.capacity > 0 ? len_of(a, b) : 0;
      seg.own = true;
      seg.of = b;
      seg.kv_head = blockIdx.x % a.kv_heads;
      seg.first_row = first_row;
      seg.start = local * kRows;
      seg.count = min(kRows, rows * a.group - seg.start);
      seg.limit0 = len - rows + 1;
      seg.all_see = seg.limit0 + seg.start / a.group;
      seg.key0 = 0;
      seg.key1 = max(0, seg.limit0 + (seg.start + seg.count - 1) / a.group);  // the tile's last row sees the most
    };
    if (a.row_offsets == nullptr) {
      const int each = (a.group + kRows - 1) / kRows;
      if (lane == 0) take(tile / each, 1, tile / each, tile % each);
    } else {
      for (int b0 = 0; b0 < a.sequences; b0 += 32) {
        int first = 0;
        const int rows = b0 + lane < a.sequences ? rows_of(a, b0 + lane, &first) : 0;
        const int tiles = (rows * a.group + kRows - 1) / kRows;
        int upto = tiles;
#pragma unroll
        for (int off = 1; off < 32; off *= 2) {
          const int other = __shfl_up_sync(0xffffffffu, upto, off);
          if (lane >= off) upto += other;
        }
        const bool mine = tile < upto && tile >= upto - tiles;
        if (mine) take(b0 + lane, rows, first, tile - (upto - tiles));
        if (__any_sync(0xffffffffu, mine)) break;
        tile -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
  }
  __syncthreads();
  if (seg.count == 0) {
    if (late_wait) pdl_wait();
  } else {
    attend<kDim, kWarps, true>(a, seg, raw, odd_keys, late_wait != 0);
  }
}

// The same for one row a sequence and at most 8 heads to a key/value head. Blocks: sequences x key/value heads.
template <int kDim, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps) attention_few_kernel(Attention a, int late_wait) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint32_t free_word;
  if (!late_wait) pdl_wait();
  // The next grid waits for this one, which waits for the one before it. Among attention calls its early start makes
  // little difference (four beams 12.8 us with and 13.0 without it, sixteen pages, which go without, 53.1 and 53.3).
  if (kWarps == 8) pdl_launch_dependents();
  attend_few<kDim, kWarps>(a, raw, &free_word, late_wait != 0);
}

// kWarps warps join the parts of a (row, head): first all maxima and sums, a lane a part, then the outputs of the parts
// that hold keys, warp by warp every kWarps-th one, eight under way at a time.
template <int kDim, int kWarps>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(Attention a) {
  constexpr int kEach = kDim / 32, kCells = kThreads / 32 / kWarps;
  __shared__ float factors[kCells][kMaxSlots];
  __shared__ float sums[kCells][kWarps][kDim];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, local = warp / kWarps, along = warp % kWarps;
  const int64_t cell = static_cast<int64_t>(blockIdx.x) * kCells + local;
  bool live = cell < static_cast<int64_t>(a.rows) * a.heads;
  const int64_t row = live ? cell / a.heads : 0;
  const int head = static_cast<int>(cell % a.heads);
  if (live && a.row_offsets != nullptr) live = row >= a.row_offsets[0] && row < a.row_offsets[a.sequences];
  const float2* ml = a.part_ml + cell * a.slots;
  float2 mine[kMaxSlots / 32];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxSlots / 32; ++i) {
    const int s = i * 32 + lane;
    mine[i] = live && s < a.slots ? ml[s] : make_float2(-INFINITY, 0.0f);
    top = fmaxf(top, mine[i].x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float shift = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxSlots / 32; ++i) {
    const int s = i * 32 + lane;
    const float f = exp2_fast(mine[i].x - shift);
    sum = fmaf(mine[i].y, f, sum);
    // A part without keys has no output: its factor is told apart from one that has underflowed.
    if (along == 0 && s < a.slots) factors[local][s] = mine[i].x == -INFINITY ? -1.0f : f;
  }
  sum = warp_sum(sum);
  if (kWarps > 1)
    __syncthreads();
  else
    __syncwarp();
  float acc[kEach] = {};
  const float* o = a.part_o + cell * a.slots * kDim + lane * kEach;
  constexpr int kAhead = 8;
  for (int s0 = along; live && s0 < a.slots; s0 += kAhead * kWarps) {
    float v[kAhead][kEach];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * kWarps;
      const bool has = s < a.slots && factors[local][s] >= 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) v[k][i] = 0.0f;
      if (has) {
        if constexpr (kEach == 4) {
          const float4 x = *reinterpret_cast<const float4*>(o + static_cast<int64_t>(s) * kDim);
          v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(o + static_cast<int64_t>(s) * kDim);
          v[k][0] = x.x, v[k][1] = x.y;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * kWarps;
      const float f = s < a.slots ? fmaxf(factors[local][s], 0.0f) : 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) acc[i] = fmaf(v[k][i], f, acc[i]);
    }
  }
  if (kWarps > 1) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) sums[local][along][lane * kEach + i] = acc[i];
    __syncthreads();
    if (along != 0) return;
#pragma unroll
    for (int w = 1; w < kWarps; ++w)
#pragma unroll
      for (int i = 0; i < kEach; ++i) acc[i] += sums[local][w][lane * kEach + i];
  }
  if (!live) return;
  // A NaN sum (of NaN scores) stays one.
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  __nv_bfloat16* out = a.out + row * a.ldo + head * kDim + lane * kEach;
  if constexpr (kEach == 4)
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(out) = pack2(acc[0] * inv, acc[1] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[cell] = sum != 0.0f ? (top + log2f(sum)) * 0.69314718055994530942f : -INFINITY;
}

// The parts that the prefixes and the own keys are cut into, and the kernels.
struct Plan {
  bool tc, split;  // the prefixes by the tensor-core kernel, its tiles the same rows
  int prefix_slots, own_slots;
  int prefix_warps, own_warps;  // of the kernel for few rows: warps side by side along the rows of a tile
  unsigned blocks;
  int64_t units;      // of that kernel's work, there can be
  bool whole_own;     // the own keys of a tile of rows by one block, which joins the prefix's parts to them
  int64_t own_tiles;  // there can be
};

constexpr int kSms = 148;  // blocks of the tensor-core kernel, one an SM; correct on any number of SMs

// A prefix with many rows is arithmetic, for the tensor-core kernel: from more than 16 on, where the other kernel's tiles
// grow (us, this one's and the other's, 60 own keys; a page of 100, 256, 1024 and 4096 keys, then sixteen such pages):
//   16 rows  11.1 13.3  11.8 10.9  12.0 11.0  13.7 12.7    13.0 15.6  13.7 12.8  18.8 18.3  34.2 36.1
//   20 rows  11.3 15.1  11.8 12.5  12.0 12.7  13.8 14.7    13.2 17.3  14.1 14.4  19.1 20.7  34.8 38.9
//   24 rows  11.3 15.3  12.0 12.7  12.2 12.8  13.8 14.8    16.4 17.6  17.4 14.6  21.4 21.3  35.1 39.7
//   32 rows  11.5 15.7  12.1 12.9  12.3 13.0  14.2 15.3    17.1 18.3  18.0 17.3  22.4 21.8  36.4 41.5
//   64 rows  11.7 20.0  12.2 16.1  12.5 16.6  14.4 20.9    22.2 29.6  23.4 25.7  28.7 35.4  44.0 63.8
// So it loses a little between 16 pages of 256 and 1024 keys at 24 and 32 rows, and at 7 sequences of 37 rows of heads of
// 64 behind 1001 keys (16.5 against 13.5).
bool many_rows(const uocr_prefix_attention_args& a) {
  return a.prefix_capacity > 0 && a.rows * (a.heads / a.kv_heads) / a.prefixes > 16;
}
// Whether that kernel takes the call's scale, which it divides by, and strides, for its tensor maps.
bool tc_takes(const uocr_prefix_attention_args& a) {
  auto far = [](int64_t stride) { return stride <= 0 || stride >= (int64_t{1} << 39); };
  return a.scale >= FLT_MIN && !(a.kv_heads > 1 && far(a.prefix_head_stride)) && !(a.prefixes > 1 && far(a.prefix_stride));
}

Plan plan_of(const uocr_prefix_attention_args& a, bool tc) {
  Plan p{};
  p.tc = tc;
  const int64_t group = a.heads / a.kv_heads;
  // Rows of a tile by those of a prefix, of a sequence.
  auto warps_for = [](int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; };
  p.prefix_warps = warps_for(a.rows * group / a.prefixes);
  p.own_warps = warps_for(a.rows * group / std::max<int64_t>(a.sequences, 1));
  // The units there can be, by the capacities; with row offsets each sequence's (prefix's) last tile may be part empty.
  auto tiles = [&](int64_t count, int64_t each, int warps) {
    const int64_t tile = 16 * warps;
    return a.row_offsets == nullptr ? count * ((each * group + tile - 1) / tile)
                                    : a.rows * group / tile + std::min(count, a.rows);
  };
  const int64_t prefix_stages = (a.prefix_capacity + kKeys - 1) / kKeys, own_stages = (a.capacity + kKeys - 1) / kKeys;
  p.own_tiles = tiles(a.sequences, 1, p.own_warps);
  // Own keys in parts only where few blocks would have many: a join less, and own parts that are not written and read.
  // Four sequences of 300, 512 and 1024 own keys take 12.6, 14.0 and 21.9 us whole, 15.4, 16.4 and 16.5 in parts.
  p.whole_own = p.own_tiles * a.kv_heads >= kSms || own_stages <= 8;
  const int64_t units = p.units =
      a.kv_heads * ((p.tc ? 0 : tiles(a.prefixes, a.sequences / a.prefixes, p.prefix_warps) * prefix_stages) +
                    (p.whole_own ? 0 : p.own_tiles * own_stages));
  p.blocks = static_cast<unsigned>(std::min<int64_t>(units, kBlocks * kSms));
  // A range of keys meets as many blocks as shares fit into it, and one more; half as many again for lengths that differ.
  const int64_t share = std::max<int64_t>((units + kBlocks * kSms - 1) / (kBlocks * kSms), kMinShare);
  auto slots = [&](int64_t stages, int most) {
    return static_cast<int>(stages == 0 ? 0 : std::min<int64_t>((stages + share - 1) / share * 3 / 2 + 2, most));
  };
  p.prefix_slots = slots(prefix_stages, kMaxPrefixSlots);
  p.own_slots = p.whole_own ? 0 : slots(own_stages, kMaxOwnSlots);
  if (p.tc) {
    p.split = a.rows * group <= kAttentionTcRows * a.prefixes;
    const int64_t of_range = kAttentionTcRows * (p.split ? 1 : 2);
    const int64_t ranges = a.kv_heads * std::max((a.rows * group + of_range - 1) / of_range, p.split ? a.prefixes : 1);
    // Blocks a range can meet: as many as there are for each, and no more than its keys make (two tiles a block at least).
    const int64_t tiles = (a.prefix_capacity + 127) / 128;
    const int64_t blocks = std::max<int64_t>(std::min(kSms / ranges + 3, tiles / 2 + 2), 3);
    p.prefix_slots = static_cast<int>(std::min<int64_t>(blocks * (p.split ? 2 : 1), kMaxTcSlots));
  }
  return p;
}

template <int kDim, int kPrefixWarps, int kOwnWarps>
cudaError_t launch_rows(const Attention& a, const Grid& g, unsigned blocks, cudaStream_t stream) {
  constexpr size_t kRing = static_cast<size_t>(kStages) * 2 * kKeys * (kDim + 8) * 2;
  // 4 / w warps along the keys, 16 w rows
  constexpr size_t kJoin = static_cast<size_t>(64) * (kDim * 4 + 8);
  static_assert(kJoin <= kRing, "the join takes the ring's place");
  cudaError_t st = allow_max_dynamic_smem_once<attention_rows_kernel<kDim, kPrefixWarps, kOwnWarps>>();
  if (st != cudaSuccess) return st;
  return launch_pdl(attention_rows_kernel<kDim, kPrefixWarps, kOwnWarps>, blocks, kThreads, kRing, stream, a, g);
}

template <int kDim, int kWarps>
cudaError_t launch_last(const Attention& a, unsigned blocks, int late_wait, cudaStream_t stream) {
  constexpr size_t kRing = static_cast<size_t>(kStages) * Feed<kDim>::kStage * 2;
  const size_t join = LastJoin<kDim, 16 * kWarps, 4 / kWarps>::bytes(a.prefix_slots);
  const cudaError_t st = allow_max_dynamic_smem_once<attention_last_kernel<kDim, kWarps>>();
  if (st != cudaSuccess) return st;
  return launch_pdl(attention_last_kernel<kDim, kWarps>, blocks, kThreads, std::max(kRing, join), stream, a, late_wait);
}
template <int kDim, int kWarps>
cudaError_t launch_few(const Attention& a, unsigned blocks, int late_wait, cudaStream_t stream) {
  const size_t join = LastJoin<kDim, 8, kWarps, 32 * kWarps>::bytes(a.prefix_slots);
  const cudaError_t st = allow_max_dynamic_smem_once<attention_few_kernel<kDim, kWarps>>();
  if (st != cudaSuccess) return st;
  return launch_pdl(attention_few_kernel<kDim, kWarps>, blocks, 32 * kWarps, std::max(FewRing<kDim, kWarps>::kBytes, join),
                    stream, a, late_wait);
}

template <int kDim>
cudaError_t launch(const uocr_prefix_attention_args& args, const Attention& a, const Plan& p, cudaStream_t stream) {
  Grid g{};
  g.prefixes = p.tc || args.prefix_capacity == 0 ? 0 : a.prefixes;
  g.sequences = args.capacity == 0 || p.whole_own ? 0 : a.sequences;
  g.late_wait = p.tc;
  g.most_units = static_cast<unsigned>(p.units);
  cudaError_t st = p.tc ? launch_attention_tc(a, kDim, kSms, stream) : cudaSuccess;
  if (st == cudaSuccess && p.blocks > 0) {
    const int own = g.sequences == 0 ? p.prefix_warps : p.own_warps;
    switch ((g.prefixes == 0 ? own : p.prefix_warps) * 8 + own) {
      case 8 + 1: st = launch_rows<kDim, 1, 1>(a, g, p.blocks, stream); break;
      case 16 + 1: st = launch_rows<kDim, 2, 1>(a, g, p.blocks, stream); break;
      case 16 + 2: st = launch_rows<kDim, 2, 2>(a, g, p.blocks, stream); break;
      case 32 + 1: st = launch_rows<kDim, 4, 1>(a, g, p.blocks, stream); break;
      case 32 + 2: st = launch_rows<kDim, 4, 2>(a, g, p.blocks, stream); break;
      default: st = launch_rows<kDim, 4, 4>(a, g, p.blocks, stream);
    }
  }
  if (st != cudaSuccess) return st;
  if (p.whole_own) {
    const int late = p.tc || p.blocks > 0;
    const unsigned n = static_cast<unsigned>(p.own_tiles * a.kv_heads);
    if (a.row_offsets == nullptr && a.group <= 8)  // as many tiles: one a sequence
      return n <= kSms ? launch_few<kDim, 8>(a, n, late, stream) : launch_few<kDim, 4>(a, n, late, stream);
    return p.own_warps == 1   ? launch_last<kDim, 1>(a, n, late, stream)
           : p.own_warps == 2 ? launch_last<kDim, 2>(a, n, late, stream)
                              : launch_last<kDim, 4>(a, n, late, stream);
  }
  // Few rows: all warps of a block on one, for the round trips of its parts.
  const int64_t cells = args.rows * args.heads, each = kThreads / 32;
  if (cells <= 4 * kSms)
    return launch_pdl(attention_join_kernel<kDim, 4>, static_cast<unsigned>(cells), kThreads, 0, stream, a);
  return launch_pdl(attention_join_kernel<kDim, 1>, static_cast<unsigned>((cells + each - 1) / each), kThreads, 0,
                    stream, a);
}

}  // namespace

bool prefix_attention_counts(const uocr_prefix_attention_args& a) {
  // Units are counted in 32 bits; the tensor-core kernel has at most five for each of these.
  const double stages = static_cast<double>((a.prefix_capacity + kKeys - 1) / kKeys + (a.capacity + kKeys - 1) / kKeys);
  return (static_cast<double>(a.rows) * a.heads / 16 + a.kv_heads * static_cast<double>(a.sequences)) * stages < 8.0e8;
}

size_t prefix_attention_bytes(const uocr_prefix_attention_args& a) {
  // By the sizes alone: room for either kernel where the scale or the strides may decide.
  const Plan few = plan_of(a, false);
  int slots = few.prefix_slots + few.own_slots;
  if (many_rows(a)) {
    const Plan many = plan_of(a, true);
    slots = std::max(slots, many.prefix_slots + many.own_slots);
  }
  return static_cast<size_t>(a.rows * a.heads) * slots * (a.head_dim * 4 + sizeof(float2));
}

cudaError_t launch_prefix_attention(const uocr_prefix_attention_args& args, ErrorWord* err, cudaStream_t stream) {
  const Plan p = plan_of(args, many_rows(args) && tc_takes(args));
  Attention a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(args.q);
  a.prefix_k = reinterpret_cast<const __nv_bfloat16*>(args.prefix_k);
  a.prefix_v = reinterpret_cast<const __nv_bfloat16*>(args.prefix_v);
  a.prefix_lens = args.prefix_lens;
  a.k = reinterpret_cast<const __nv_bfloat16*>(args.k);
  a.v = reinterpret_cast<const __nv_bfloat16*>(args.v);
  a.lens = args.lens, a.ancestry = args.ancestry, a.row_offsets = args.row_offsets;
  a.out = reinterpret_cast<__nv_bfloat16*>(args.out);
  a.lse = args.lse;
  a.ldq = args.ldq, a.ldo = args.ldo, a.ld_ancestry = args.ld_ancestry;
  a.prefix_stride = args.prefix_stride, a.prefix_head_stride = args.prefix_head_stride;
  a.cache_stride = args.cache_stride, a.head_stride = args.head_stride;
  a.rows = static_cast<int>(args.rows), a.sequences = static_cast<int>(args.sequences);
  a.prefixes = static_cast<int>(args.prefixes), a.caches = static_cast<int>(args.caches);
  a.heads = static_cast<int>(args.heads), a.kv_heads = static_cast<int>(args.kv_heads);
  a.group = a.heads / a.kv_heads;
  a.per = static_cast<int>(args.sequences / args.prefixes);
  a.prefix_capacity = static_cast<int>(args.prefix_capacity), a.capacity = static_cast<int>(args.capacity);
  a.prefix_slots = p.prefix_slots;
  a.split = p.split;
  a.slots = p.prefix_slots + p.own_slots;
  a.scale_log2 = args.scale * kLog2e;
  a.part_o = static_cast<float*>(args.workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + args.rows * args.heads * a.slots * args.head_dim);
  a.err = err;
  return args.head_dim == 64 ? launch<64>(args, a, p, stream) : launch<128>(args, a, p, stream);
}

}  // namespace uocr_b200
