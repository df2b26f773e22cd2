// The best continuations of a group of beams (uocr_beam_select).
//
// score(b, t) = scores[b] + (logit - m) - log sum exp(logit - m): within a beam
// the order is the logits' own, so one pass over a row is enough: a block goes
// through a part of a row, keeps the maximum, the sum of exponentials and the
// `select` best logits; a second kernel joins a group's parts. Bound: the one
// read of the logits; for few rows two launches and their rounds. 128 rows of 102400
// logits take 23.1 us (2.3 TB/s: instructions and barriers, 8.0 at the copy rate),
// four rows 7.9; with all but 100 tokens masked 54.8 (-inf: 44.2) and 12.6, since
// what equals the bound then reaches it.
//
// The best of a part without sorting it: the threads' own maxima, sorted within
// warps, bound the select-th best of all from below. What
// reaches the bound goes on a list; where that grows the bound is drawn anew from
// it, higher, so that soon hardly an element passes; what is left at the end, a
// few dozen, is ranked. Keys are unique (value, then the lower index), so the
// result is the exact one, ties included, in every case.
#include <algorithm>

#include "beam.h"
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// 2^x to 2 ulp; 2^-inf = 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kEach = 16;     // elements of a thread and round
constexpr int kRound = kThreads * kEach;
constexpr int kRanked = 512;  // as many keys are ranked against one another; more are thinned out first
constexpr int kList = kRound + 2 * UOCR_BEAM_MAX + 64;  // what a round may leave (list_limit), and one round
__device__ __forceinline__ int list_limit(int select) { return 2 * select + 64; }

// Floats in their order as unsigned integers, -0 as 0; 0 stands for no candidate.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float f, uint32_t index) {
  return f > -INFINITY ? static_cast<uint64_t>(ordered(f)) << 32 | (0xffffffffu - index) : 0;
}

// The warp's keys in descending order over its lanes.
template <typename Key>
__device__ __forceinline__ Key sort_lanes(Key key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const Key other = __shfl_xor_sync(0xffffffffu, key, step);
      const bool keep_high = ((lane & size) == 0) == ((lane & step) == 0);
      key = (other > key) == keep_high ? other : key;
    }
  return key;
}

// A lower bound on the select-th best of the block's elements, from each
// thread's best: for j = 1, 2, 4 and 8 groups of warps, every group has a warp with
// ceil(select / j) elements that reach the group's best such warp's last one, and so
// j ceil(select / j) >= select elements reach the least of the groups'. (The 16th
// of 4096 is reached by 16, this by some 35, the best of the warps' 16th, j = 1, by
// 116.) All threads call it; `shared`: 4 * kWarps keys.
template <typename Key>
__device__ __forceinline__ Key bound_of(Key best, int select, uint64_t* shared) {
  static_assert(kWarps == 8, "four kinds of groups, a lane each of their warps");
  const Key sorted = sort_lanes(best);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kind = lane / kWarps;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane == ((select - 1) >> k)) shared[k * kWarps + warp] = sorted;  // ceil(select / 2^k) - 1
  __syncthreads();
  Key bound = static_cast<Key>(shared[lane]);
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    const Key other = __shfl_xor_sync(0xffffffffu, bound, 1 << step);
    bound = step < 3 - kind ? max(bound, other) : min(bound, other);
  }
  bound = max(bound, __shfl_xor_sync(0xffffffffu, bound, 8));
  bound = max(bound, __shfl_xor_sync(0xffffffffu, bound, 16));
  return max(bound, static_cast<Key>(1));
}

// e^(f - m) for f <= m, m above -inf. The difference comes first: from 2^24 on the rounding of a product m log2 e is
// more than 1, and of the lowest floats, which mask tokens, the product is -inf.
__device__ __forceinline__ float exp_of(float f, float m) { return exp2_fast((f - m) * kLog2e); }

struct Select {
  const void* logits;
  const float* scores;
  const int* finished;
  int64_t ld;
  int vocab, beams, select;
  int parts, part;  // of a row; elements of a part, a multiple of kRound
  bool vec;         // rows allow 16 bytes at a time
  float2* sums;     // [rows, parts]: maximum m, and sum of exp(f - m)
  uint64_t* best;   // [rows, parts, select] keys, descending
};

// Cuts the list to its `select` best, in order, and returns the last of them (1:
// there are fewer), which all that still can be among the best reach. All threads
// call it, behind a barrier. `best`: UOCR_BEAM_MAX keys.
__device__ uint64_t cut(uint64_t* list, int* count, int* next, int select, uint64_t* bounds, uint64_t* best) {
  int n = *count;
  // Many: those that reach a bound, drawn like the first one, unless that removes next to nothing. In place: what a
  // thread keeps it has in registers.
  for (int before = 2 * n; n > kRanked && n * 5 < before * 4;) {
    constexpr int kMost = (kList + kThreads - 1) / kThreads;
    uint64_t mine[kMost];
    uint64_t high = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int at = i * kThreads + static_cast<int>(threadIdx.x);
      mine[i] = at < n ? list[at] : 0;
      high = max(high, mine[i]);
    }
    if (threadIdx.x == 0) *next = 0;
    const uint64_t bound = bound_of(high, select, bounds);
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (mine[i] >= bound) list[atomicAdd(next, 1)] = mine[i];
    __syncthreads();
    before = n;
    n = *next;
    __syncthreads();
  }
#pragma unroll 1
  for (int i = threadIdx.x / 2; i < (n + 15) / 16 * 16; i += kThreads / 2) {  // two neighbouring threads a key; whole warps
    const uint64_t key = i < n ? list[i] : ~0ull;
    int rank = 0;
#pragma unroll 8
    for (int j = threadIdx.x & 1; j < n; j += 2) rank += list[j] > key;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    if (i < n && rank < select) best[rank] = key;
  }
  __syncthreads();
  n = min(n, select);
  if (static_cast<int>(threadIdx.x) < n) list[threadIdx.x] = best[threadIdx.x];
  if (threadIdx.x == 0) *count = n;
  const uint64_t last = n == select ? best[select - 1] : 1;
  __syncthreads();
  return last;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) beam_parts_kernel(Select a) {
  constexpr int kVec = 16 / sizeof(T);
  extern __shared__ uint64_t list[];  // [kList]
  __shared__ uint64_t bounds[4 * kWarps];
  __shared__ float2 warp_sums[kWarps];
  __shared__ uint64_t best[UOCR_BEAM_MAX];
  __shared__ int count, next;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const bool ended = a.finished != nullptr && a.finished[row] != 0;
  const float score = a.scores[row];
  const T* src = static_cast<const T*>(a.logits) + row * a.ld;
  const int begin = part * a.part, end = min(a.vocab, begin + a.part);
  // A round's elements of this thread, as they lie in memory: kVec side by side, then those kThreads * kVec further on.
  struct Raw {
    uint4 v[kEach / kVec];
  };
  auto index = [&](int base, int i) {
    return base + (i / kVec * kThreads + static_cast<int>(threadIdx.x)) * kVec + i % kVec;
  };
  auto load = [&](int base) {
    Raw r;
    if (a.vec && base + kRound <= end) {
      const uint4* p = reinterpret_cast<const uint4*>(src + base) + threadIdx.x;
#pragma unroll
      for (int j = 0; j < kEach / kVec; ++j) r.v[j] = p[j * kThreads];
      return r;
    }
#pragma unroll
    for (int j = 0; j < kEach / kVec; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          const int at = index(base, j * kVec + i);
          w[i] = at < end ? __float_as_uint(src[at]) : 0xff800000u;
        } else {
          const int at = index(base, j * kVec + 2 * i);
          const unsigned short* of = reinterpret_cast<const unsigned short*>(src);
          w[i] = (at < end ? of[at] : 0xff80u) | (at + 1 < end ? of[at + 1] : 0xff80u) << 16;
        }
      }
      r.v[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
  };
  auto value_of = [](const Raw& r, int i) {
    const uint4& u = r.v[i / kVec];
    const int at = i % kVec;
    const int word = sizeof(T) == 4 ? at : at / 2;
    const uint32_t w = word == 0 ? u.x : word == 1 ? u.y : word == 2 ? u.z : u.w;
    return __uint_as_float(sizeof(T) == 4 ? w : at % 2 == 0 ? w << 16 : w & 0xffff0000u);
  };
  Raw ahead = load(begin);
  // The second kernel asks for nothing of a beam that has ended or does not exist. Found out with the first loads under
  // way, not before them: one round trip less where the beam goes on.
  if (ended || !(score > -INFINITY)) return;
  if (threadIdx.x == 0) count = 0;
  float m = -INFINITY, sum = 0.0f;  // of this thread
  uint64_t bound = 0;
  float at_least = -INFINITY;
  for (int base = begin; base < end; base += kRound) {
    float f[kEach];
    float peak = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      f[i] = value_of(ahead, i);
      peak = fmaxf(peak, f[i]);  // of no NaN
    }
    if (base + kRound < end) ahead = load(base + kRound);
    if (peak > m) {
      sum *= exp_of(m, peak);  // of no element yet: 0 * 0
      m = peak;
    }
    const float shift = m > -INFINITY ? m : 0.0f;
    float2 of_round = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
      const float2 x = fma2(add2(make_float2(f[i], f[i + 1]), make_float2(-shift, -shift)),
                            make_float2(kLog2e, kLog2e), make_float2(0.0f, 0.0f));
      of_round = add2(of_round, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
    }
    float added = of_round.x + of_round.y;
    if (added != added) {  // NaN counts as -inf; beside +inf the sum is not asked for
      added = 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) added += exp_of(fmaxf(f[i], -INFINITY), shift);
    }
    sum += added;
    if (bound == 0) {
      // By the values alone, in half the steps: of equal ones the first cut tells the best.
      const uint32_t value = max(bound_of(ordered(peak), a.select, bounds), ordered(-INFINITY));
      bound = static_cast<uint64_t>(value) << 32;
      at_least = unordered(value);
    }
    bool many = base == begin && base + kRound < end;
    if (peak >= at_least) {
      unsigned reach = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) reach |= f[i] >= at_least ? 1u << i : 0u;
      while (reach != 0) {  // few threads have any, and those mostly one
        const int i = __ffs(reach) - 1;
        reach &= reach - 1;
        float v[kEach / 2];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (i & 8) != 0 ? f[k + 8] : f[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (i & 4) != 0 ? v[k + 4] : v[k];
        const float lo = (i & 2) != 0 ? v[2] : v[0], hi = (i & 2) != 0 ? v[3] : v[1];
        const uint64_t key = key_of((i & 1) != 0 ? hi : lo, static_cast<uint32_t>(index(base, i)));
        if (key < bound) continue;
        const int at = atomicAdd(&count, 1);
        list[at] = key;
        many |= at >= list_limit(a.select);
      }
    }
    // The bound is drawn anew after the first round, from when on few elements pass, and when the list grows.
    if (__syncthreads_or(many)) {
      bound = max(bound, cut(list, &count, &next, a.select, bounds, best));
      at_least = unordered(max(static_cast<uint32_t>(bound >> 32), ordered(-INFINITY)));
    }
  }
  // The block's maximum and sum.
  float top = m;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  sum = warp_sum(m > -INFINITY ? sum * exp_of(m, top) : 0.0f);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = make_float2(top, sum);
  __syncthreads();
  const int64_t cell = row * a.parts + part;
  if (threadIdx.x == 0) {
    float2 all = warp_sums[0];
    for (int w = 1; w < kWarps; ++w) {
      const float2 p = warp_sums[w];
      const float high = fmaxf(all.x, p.x);
      if (high == -INFINITY) continue;
      all = make_float2(high, all.y * exp_of(all.x, high) + p.y * exp_of(p.x, high));
    }
    a.sums[cell] = all;
  }
  cut(list, &count, &next, a.select, bounds, best);
  if (static_cast<int>(threadIdx.x) < a.select)
    a.best[cell * a.select + threadIdx.x] = static_cast<int>(threadIdx.x) < count ? list[threadIdx.x] : 0;
}

struct Join {
  Select s;
  int* tokens;
  int* parents;
  float* new_scores;
  int* new_finished;
  int eos;
  int depth;  // 1 .. select
};

// A candidate in the order of the selection: the score, then the lower beam, within
// a beam the higher logit (scores far from 0 can no longer tell those apart), then
// the lower token. The 64-bit score as an integer in the same order, which compares
// in two instructions where doubles took ten times as long; 0: no candidate.
struct Cand {
  uint64_t score;
  uint64_t flat;  // beam << 52 | inverted ordered logit << 20 | token
};
constexpr int kTokenBits = 20, kBeamAt = 52;
static_assert(UOCR_BEAM_MAX <= 1 << (64 - kBeamAt), "");
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));  // -0 as 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ float score_of(const Cand& c) {
  const uint64_t u = c.score >> 63 ? c.score & 0x7fffffffffffffffull : ~c.score;
  return static_cast<float>(__longlong_as_double(static_cast<long long>(u)));
}
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  return (a.score > b.score) | ((a.score == b.score) & (a.flat < b.flat));  // no branch
}

constexpr int kJoinThreads = 512;
constexpr int kLanes = 4;  // neighbouring threads that rank a candidate

// How many of the n candidates are better than `mine`.
__device__ __forceinline__ int rank_of(const Cand& mine, const Cand* of, int n) {
  int rank = 0;
#pragma unroll 4
  for (int j = threadIdx.x % kLanes; j < n; j += kLanes) rank += better(of[j], mine) ? 1 : 0;
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  return rank + __shfl_xor_sync(0xffffffffu, rank, 2);
}

// A block joins a group, whose lists (parts) are in descending order. The `depth`
// first entries of each are ranked against one another: further entries of a list
// are candidates only where the last of those is among the `select` best, and then
// only the ones that are not below the select-th best. (With the first entries alone
// 200 candidates were left of sixteen pages' 24 lists, and 3.7 us for their ranks.)
// Everything of the group is read in one round, the keys too where they fit (kStage).
template <bool kStaged>
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(Join a) {
  extern __shared__ Cand heads[];  // [beams * parts * depth], then [select * select], then the keys
  __shared__ double log_sums[UOCR_BEAM_MAX];  // log sum exp(f - top); INFINITY: no candidates
  __shared__ float tops[UOCR_BEAM_MAX];
  __shared__ float scores[UOCR_BEAM_MAX];
  __shared__ int ended[UOCR_BEAM_MAX];
  __shared__ Cand worst;
  __shared__ int lists[UOCR_BEAM_MAX];
  __shared__ int chosen, count;
  const Select& s = a.s;
  const int n = s.beams * s.parts, depth = a.depth;
  Cand* left = heads + n * depth;
  uint64_t* staged = reinterpret_cast<uint64_t*>(left + s.select * s.select);
  pdl_wait();
  pdl_launch_dependents();
  const int64_t group = blockIdx.x, first = group * s.beams;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t* keys = s.best + first * s.parts * s.select;
  if (kStaged)
    for (int i = threadIdx.x; i < n * s.select; i += kJoinThreads) staged[i] = keys[i];
  if (threadIdx.x == 0) chosen = count = 0;
  for (int b = warp; b < s.beams; b += kJoinThreads / 32) {
    const float score = s.scores[first + b];
    const bool done = s.finished != nullptr && s.finished[first + b] != 0;
    double value = INFINITY;
    float m = -INFINITY;
    if (!done && score > -INFINITY) {
      double sum = 0.0;
      for (int c0 = 0; c0 < s.parts; c0 += 32) {
        const float2 p = c0 + lane < s.parts ? s.sums[(first + b) * s.parts + c0 + lane] : make_float2(-INFINITY, 0.0f);
        float high = fmaxf(m, p.x);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, off));
        if (high == -INFINITY) continue;
        const double top = static_cast<double>(high);
        double all = p.x > -INFINITY ? static_cast<double>(p.y) * exp(static_cast<double>(p.x) - top) : 0.0;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        sum = all + (m > -INFINITY ? sum * exp(static_cast<double>(m) - top) : 0.0);
        m = high;
      }
      if (m > -INFINITY && m < INFINITY) value = log(sum);
    }
    if (lane == 0) {
      log_sums[b] = value;
      tops[b] = m;
      scores[b] = score;
      ended[b] = done;
    }
  }
  __syncthreads();
  // Entry `at` of list `i` (a beam's part, or the one candidate of a beam that has ended).
  auto entry = [&](int i, int at) {
    const int b = i / s.parts;
    const float score = scores[b];
    Cand e{0, ~0ull};
    if (ended[b]) {
      if (i == b * s.parts && at == 0 && score > -INFINITY) {
        e.score = ordered64(score);
        e.flat = static_cast<uint64_t>(b) << kBeamAt | static_cast<uint32_t>(max(a.eos, 0));
      }
    } else if (log_sums[b] < INFINITY) {
      const uint64_t key = kStaged ? staged[i * s.select + at] : keys[static_cast<int64_t>(i) * s.select + at];
      // The maximum first: far from 0 it and the sum's log have no number in common.
      const double logit = static_cast<double>(unordered(static_cast<uint32_t>(key >> 32)));
      const double v = static_cast<double>(score) + ((logit - static_cast<double>(tops[b])) - log_sums[b]);
      if (key != 0 && static_cast<float>(v) > -INFINITY) {  // as it is handed out
        e.score = ordered64(v);
        e.flat = static_cast<uint64_t>(b) << kBeamAt | static_cast<uint64_t>(~static_cast<uint32_t>(key >> 32)) << kTokenBits |
                 (0xffffffffu - static_cast<uint32_t>(key));
      }
    }
    return e;
  };
  // Entry `at` of all lists, then the next one's: neighbouring threads have different lists.
  for (int i = threadIdx.x; i < n * depth; i += kJoinThreads) heads[i] = entry(i % n, i / n);
  __syncthreads();
  for (int i0 = 0; i0 < n * depth; i0 += kJoinThreads / kLanes) {
    const int i = i0 + threadIdx.x / kLanes;
    const Cand mine = i < n * depth ? heads[i] : Cand{0, ~0ull};
    const int rank = rank_of(mine, heads, n * depth);
    if (mine.score == 0 || threadIdx.x % kLanes != 0 || rank >= s.select) continue;
    left[atomicAdd(&count, 1)] = mine;
    if (rank == s.select - 1) worst = mine;
    if (i >= n * (depth - 1)) lists[atomicAdd(&chosen, 1)] = i % n;
  }
  __syncthreads();
  const bool full = count == s.select;
  const int further = s.select - depth, deep = chosen;  // at most select / depth lists: `left` has room for them
  __syncthreads();
  for (int i = threadIdx.x; i < deep * further; i += kJoinThreads) {
    const Cand e = entry(lists[i / further], depth + i % further);
    if (e.score != 0 && !(full && better(worst, e))) left[atomicAdd(&count, 1)] = e;
  }
  __syncthreads();
  const int m = count;
  auto put = [&](int rank, int token, int parent, float score, bool done) {
    const int64_t at = group * s.select + rank;
    a.tokens[at] = token;
    a.parents[at] = parent;
    a.new_scores[at] = score;
    if (a.new_finished != nullptr) a.new_finished[at] = done ? 1 : 0;
  };
  for (int i0 = 0; i0 < m; i0 += kJoinThreads / kLanes) {
    const int i = i0 + threadIdx.x / kLanes;
    const Cand mine = i < m ? left[i] : Cand{0, ~0ull};
    const int rank = rank_of(mine, left, m);
    if (mine.score == 0 || threadIdx.x % kLanes != 0 || rank >= s.select) continue;
    const int b = static_cast<int>(mine.flat >> kBeamAt), token = static_cast<int>(mine.flat & ((1u << kTokenBits) - 1));
    put(rank, token, b, score_of(mine), ended[b] || token == a.eos);
  }
  for (int i = m + threadIdx.x; i < s.select; i += kJoinThreads) put(i, max(a.eos, 0), 0, -INFINITY, true);
}

// Elements of a part, whole rounds: as many parts as there are blocks on the SMs at a time (three each), so that none
// waits for another.
int part_of(const uocr_beam_select_args& a) {
  const int64_t rows = std::max<int64_t>(a.batch * a.beams, 1);
  const int64_t parts = std::max<int64_t>(3 * 148 / rows, 1);
  const int64_t rounds = (a.vocab + kRound - 1) / kRound;
  return static_cast<int>((rounds + parts - 1) / parts) * kRound;
}
int parts_of(const uocr_beam_select_args& a) {
  const int64_t part = part_of(a);
  return static_cast<int>((a.vocab + part - 1) / part);
}

template <typename T>
cudaError_t launch(const uocr_beam_select_args& a, const Join& j, cudaStream_t stream) {
  const size_t keys = static_cast<size_t>(j.s.beams) * j.s.parts * j.s.select * sizeof(uint64_t);
  const size_t join_smem = (static_cast<size_t>(j.s.beams) * j.s.parts * j.depth + j.s.select * j.s.select) * sizeof(Cand);
  const bool staged = keys <= 64 * 1024;
  cudaError_t st = allow_max_dynamic_smem_once<beam_parts_kernel<T>>();
  if (st == cudaSuccess) st = allow_max_dynamic_smem_once<beam_join_kernel<true>>();
  if (st == cudaSuccess) st = allow_max_dynamic_smem_once<beam_join_kernel<false>>();
  if (st == cudaSuccess)
    st = launch_pdl(beam_parts_kernel<T>, static_cast<unsigned>(a.batch * a.beams * j.s.parts), kThreads,
                    kList * sizeof(uint64_t), stream, j.s);
  if (st == cudaSuccess)
    st = launch_pdl(staged ? beam_join_kernel<true> : beam_join_kernel<false>, static_cast<unsigned>(a.batch), kJoinThreads,
                    join_smem + (staged ? keys : 0), stream, j);
  return st;
}

}  // namespace

size_t beam_select_bytes(const uocr_beam_select_args& a) {
  return static_cast<size_t>(a.batch * a.beams) * parts_of(a) * (sizeof(float2) + a.select * sizeof(uint64_t));
}

cudaError_t launch_beam_select(const uocr_beam_select_args& a, cudaStream_t stream) {
  Join j{};
  Select& s = j.s;
  s.logits = a.logits, s.scores = a.scores, s.finished = a.finished;
  s.ld = a.ld_logits;
  s.vocab = static_cast<int>(a.vocab), s.beams = static_cast<int>(a.beams), s.select = static_cast<int>(a.select);
  s.parts = parts_of(a);
  s.part = part_of(a);
  const size_t eb = a.dtype == UOCR_DTYPE_BF16 ? 2 : 4;
  s.vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld_logits * eb % 16 == 0;
  const size_t cells = static_cast<size_t>(a.batch * a.beams) * s.parts;
  s.best = static_cast<uint64_t*>(a.workspace);
  s.sums = reinterpret_cast<float2*>(s.best + cells * a.select);
  j.tokens = a.tokens, j.parents = a.parents, j.new_scores = a.new_scores, j.new_finished = a.new_finished;
  j.eos = a.eos;
  // As many entries as the block ranks in one go.
  j.depth = std::clamp(kJoinThreads / kLanes / (s.beams * s.parts), 1, s.select);
  return a.dtype == UOCR_DTYPE_BF16 ? launch<__nv_bfloat16>(a, j, stream) : launch<float>(a, j, stream);
}

}  // namespace uocr_b200
