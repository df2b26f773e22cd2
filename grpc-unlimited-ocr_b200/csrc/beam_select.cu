// The best continuations of a group of beams (uocr_beam_select).
//
// score(b, t) = scores[b] + logit - (m + log sum exp(logit - m)): within a beam
// the order is the logits' own, so one pass over a row is enough: a block keeps
// a chunk of a row in registers, takes its maximum, its sum of exponentials and
// its `select` best logits; a second kernel joins a group's chunks. Bound: the
// one read of the logits; for few rows two launches and their rounds.
//
// The best of a chunk without sorting it: the select-th best of the threads'
// own maxima, taken warp by warp, bounds the select-th best of all from below,
// which leaves a few dozen elements to rank against one another. Keys are
// unique (value, then the lower index), so the result is the exact one, ties
// included, in every case.
#include "beam.h"
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRefine = 256;  // survivors above this are thinned out once more before they are ranked

// Floats in their order as unsigned integers; 0 stands for no candidate.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float f, uint32_t index) {
  return f > -INFINITY ? static_cast<uint64_t>(ordered(f)) << 32 | (0xffffffffu - index) : 0;
}

// The warp's keys in descending order over its lanes.
__device__ __forceinline__ uint64_t sort_lanes(uint64_t key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, step);
      const bool keep_high = ((lane & size) == 0) == ((lane & step) == 0);
      key = (other > key) == keep_high ? other : key;
    }
  return key;
}

// A lower bound on the select-th best of the block's elements, from each
// thread's best: the best of the warps' select-th ones. All threads call it;
// *top receives the best of all. `shared`: 2 * kWarps keys.
__device__ uint64_t bound_of(uint64_t best, int select, uint64_t* shared, uint64_t* top) {
  const uint64_t sorted = sort_lanes(best);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == select - 1) shared[warp] = sorted;
  if (lane == 0) shared[kWarps + warp] = sorted;
  __syncthreads();
  uint64_t bound = 1, first = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    bound = max(bound, shared[w]);
    first = max(first, shared[kWarps + w]);
  }
  *top = first;
  return bound;
}

struct Select {
  const void* logits;
  const float* scores;
  const int* finished;
  int64_t ld;
  int vocab, beams, select, chunks;
  bool vec;         // rows allow 16 bytes at a time
  float2* sums;     // [rows, chunks]: maximum and sum of exponentials
  uint64_t* best;   // [rows, chunks, select] keys, descending
};

template <typename T, int kEach>
__global__ void __launch_bounds__(kThreads) beam_chunks_kernel(Select a) {
  constexpr int kVec = 16 / sizeof(T);
  extern __shared__ uint64_t list[];  // [kWarps * select * kEach]: no warp has more than `select` threads at the bound
  __shared__ uint64_t bounds[2 * kWarps];
  __shared__ float part[kWarps];
  __shared__ int count, next;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks;
  // The second kernel asks for nothing of a beam that has ended or does not exist.
  if ((a.finished != nullptr && a.finished[row] != 0) || !(a.scores[row] > -INFINITY)) return;
  if (threadIdx.x == 0) count = 0;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld;
  const int base = chunk * (kThreads * kEach);
  float f[kEach];
  float peak = -INFINITY;
  int peak_at = 0;
#pragma unroll
  for (int j = 0; j < kEach / kVec; ++j) {
    const int at = base + (j * kThreads + static_cast<int>(threadIdx.x)) * kVec;
    float* g = f + j * kVec;
    if (a.vec && at + kVec <= a.vocab) {
      const uint4 u = *reinterpret_cast<const uint4*>(src + at);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < kVec; ++i) g[i] = to_f32(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) g[i] = at + i < a.vocab ? to_f32(src[at + i]) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (!(f[i] > -INFINITY)) f[i] = -INFINITY;  // NaN
    if (f[i] > peak) {
      peak = f[i];
      peak_at = i;
    }
  }
  auto index = [&](int i) {
    return static_cast<uint32_t>(base + (i / kVec * kThreads + static_cast<int>(threadIdx.x)) * kVec + i % kVec);
  };
  uint64_t top;
  uint64_t bound = bound_of(key_of(peak, index(peak_at)), a.select, bounds, &top);
  const float m = top != 0 ? unordered(static_cast<uint32_t>(top >> 32)) : 0.0f;
  const float at_least = unordered(max(static_cast<uint32_t>(bound >> 32), ordered(-INFINITY)));
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    sum += __expf(f[i] - m);
    if (f[i] >= at_least) {
      const uint64_t key = key_of(f[i], index(i));
      if (key >= bound) list[atomicAdd(&count, 1)] = key;
    }
  }
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  int n = count;
  const int64_t cell = row * a.chunks + chunk;
  if (threadIdx.x == 0) {
    float s = 0.0f;
    for (int w = 0; w < kWarps; ++w) s += part[w];
    a.sums[cell] = make_float2(top != 0 ? m : -INFINITY, top != 0 ? s : 0.0f);
  }
  // Many survivors (large values side by side in few threads): dealt out anew, bounded again. In place: what a
  // thread keeps it has in registers. Ends when a round removes less than a fifth.
  for (int before = n + n; n > kRefine && n * 5 < before * 4; ) {
    constexpr int kMost = kEach;  // list entries a thread: kWarps * 32 * kEach / kThreads
    uint64_t mine[kMost];
    uint64_t high = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int at = i * kThreads + static_cast<int>(threadIdx.x);
      mine[i] = at < n ? list[at] : 0;
      high = max(high, mine[i]);
    }
    if (threadIdx.x == 0) next = 0;
    __syncthreads();
    bound = bound_of(high, a.select, bounds, &top);
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (mine[i] >= bound) list[atomicAdd(&next, 1)] = mine[i];
    __syncthreads();
    before = n;
    n = next;
    __syncthreads();
  }
  uint64_t* out = a.best + cell * a.select;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n && rank < a.select; ++j) rank += list[j] > key;
    if (rank < a.select) out[rank] = key;
  }
  for (int i = n + threadIdx.x; i < a.select; i += kThreads) out[i] = 0;
}

struct Join {
  Select s;
  int* tokens;
  int* parents;
  float* new_scores;
  int* new_finished;
  int eos;
};

// A candidate in the order of the selection: the score, then the lower beam and token.
struct Cand {
  double score;
  uint64_t flat;  // beam << 32 | token
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  return a.score > b.score || (a.score == b.score && a.flat < b.flat);
}

// A block joins a group. Only the chunks with the `select` best first entries
// can hold any of the `select` best candidates, and of those only the entries
// that are not below the select-th best first entry.
__global__ void __launch_bounds__(kThreads) beam_join_kernel(Join a) {
  extern __shared__ Cand heads[];  // [beams * chunks], then [select * select]
  __shared__ double lse[UOCR_BEAM_MAX];
  __shared__ Cand worst;
  __shared__ int lists[UOCR_BEAM_MAX];
  __shared__ int chosen, count;
  const Select& s = a.s;
  const int n = s.beams * s.chunks;
  Cand* left = heads + n;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t group = blockIdx.x, first = group * s.beams;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) chosen = count = 0;
  for (int b = warp; b < s.beams; b += kWarps) {
    const float score = s.scores[first + b];
    const bool ended = s.finished != nullptr && s.finished[first + b] != 0;
    double value = INFINITY;  // no candidates
    if (!ended && score > -INFINITY) {
      float m = -INFINITY;
      for (int c = lane; c < s.chunks; c += 32) m = fmaxf(m, s.sums[(first + b) * s.chunks + c].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      double sum = 0.0;
      for (int c = lane; c < s.chunks; c += 32) {
        const float2 p = s.sums[(first + b) * s.chunks + c];
        if (p.x > -INFINITY) sum += static_cast<double>(p.y) * exp(static_cast<double>(p.x) - m);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      value = m > -INFINITY && m < INFINITY ? m + log(sum) : INFINITY;
    }
    if (lane == 0) lse[b] = value;
  }
  __syncthreads();
  // Entry `at` of list `i` (a beam's chunk, or the one candidate of a beam that has ended).
  auto entry = [&](int i, int at) {
    const int b = i / s.chunks, c = i % s.chunks;
    const float score = s.scores[first + b];
    Cand e{-INFINITY, ~0ull};
    if (s.finished != nullptr && s.finished[first + b] != 0) {
      if (c == 0 && at == 0 && score > -INFINITY) {
        e.score = score;
        e.flat = static_cast<uint64_t>(b) << 32 | static_cast<uint32_t>(max(a.eos, 0));
      }
    } else if (lse[b] < INFINITY) {
      const uint64_t key = s.best[((first + b) * s.chunks + c) * s.select + at];
      const double v = static_cast<double>(score) + (static_cast<double>(unordered(static_cast<uint32_t>(key >> 32))) - lse[b]);
      if (key != 0 && v > -INFINITY) {
        e.score = v;
        e.flat = static_cast<uint64_t>(b) << 32 | (0xffffffffu - static_cast<uint32_t>(key));
      }
    }
    return e;
  };
  for (int i = threadIdx.x; i < n; i += kThreads) heads[i] = entry(i, 0);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const Cand mine = heads[i];
    if (mine.flat == ~0ull) continue;
    int rank = 0;
    for (int j = 0; j < n && rank < s.select; ++j) rank += better(heads[j], mine);
    if (rank < s.select) lists[atomicAdd(&chosen, 1)] = i;
    if (rank == s.select - 1) worst = mine;
  }
  __syncthreads();
  const bool full = chosen == s.select;
  for (int i = threadIdx.x; i < chosen * s.select; i += kThreads) {
    const Cand e = entry(lists[i / s.select], i % s.select);
    if (e.flat != ~0ull && !(full && better(worst, e))) left[atomicAdd(&count, 1)] = e;
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
  for (int i = threadIdx.x; i < m; i += kThreads) {
    const Cand mine = left[i];
    int rank = 0;
    for (int j = 0; j < m && rank < s.select; ++j) rank += better(left[j], mine);
    if (rank >= s.select) continue;
    const int b = static_cast<int>(mine.flat >> 32), token = static_cast<int>(mine.flat & 0xffffffffu);
    const bool ended = s.finished != nullptr && s.finished[first + b] != 0;
    put(rank, token, b, static_cast<float>(mine.score), ended || token == a.eos);
  }
  for (int i = m + threadIdx.x; i < s.select; i += kThreads) put(i, max(a.eos, 0), 0, -INFINITY, true);
}

constexpr int kEachMost = 32;

int chunk_each(const uocr_beam_select_args& a) {
  // Few rows: smaller chunks, so that more SMs read.
  return a.batch * a.beams * ((a.vocab + kThreads * 16 - 1) / (kThreads * 16)) <= 592 ? 16 : kEachMost;
}

int chunks_of(const uocr_beam_select_args& a) {
  const int64_t each = static_cast<int64_t>(chunk_each(a)) * kThreads;
  return static_cast<int>((a.vocab + each - 1) / each);
}

template <typename T, int kEach>
cudaError_t launch(const uocr_beam_select_args& a, const Join& j, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kWarps) * j.s.select * kEach * sizeof(uint64_t);
  const size_t join_smem = (static_cast<size_t>(j.s.beams) * j.s.chunks + j.s.select * j.s.select) * sizeof(Cand);
  cudaError_t st = allow_max_dynamic_smem(beam_chunks_kernel<T, kEach>);
  if (st == cudaSuccess) st = allow_max_dynamic_smem(beam_join_kernel);
  if (st == cudaSuccess)
    st = launch_pdl(beam_chunks_kernel<T, kEach>, static_cast<unsigned>(a.batch * a.beams * j.s.chunks), kThreads, smem,
                    stream, j.s);
  if (st == cudaSuccess)
    st = launch_pdl(beam_join_kernel, static_cast<unsigned>(a.batch), kThreads, join_smem, stream, j);
  return st;
}

}  // namespace

size_t beam_select_bytes(const uocr_beam_select_args& a) {
  return static_cast<size_t>(a.batch * a.beams) * chunks_of(a) * (sizeof(float2) + a.select * sizeof(uint64_t));
}

cudaError_t launch_beam_select(const uocr_beam_select_args& a, cudaStream_t stream) {
  Join j{};
  Select& s = j.s;
  s.logits = a.logits, s.scores = a.scores, s.finished = a.finished;
  s.ld = a.ld_logits;
  s.vocab = static_cast<int>(a.vocab), s.beams = static_cast<int>(a.beams), s.select = static_cast<int>(a.select);
  s.chunks = chunks_of(a);
  const size_t eb = a.dtype == UOCR_DTYPE_BF16 ? 2 : 4;
  s.vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld_logits * eb % 16 == 0;
  const size_t cells = static_cast<size_t>(a.batch * a.beams) * s.chunks;
  s.best = static_cast<uint64_t*>(a.workspace);
  s.sums = reinterpret_cast<float2*>(s.best + cells * a.select);
  j.tokens = a.tokens, j.parents = a.parents, j.new_scores = a.new_scores, j.new_finished = a.new_finished;
  j.eos = a.eos;
  const bool small = chunk_each(a) == 16;
  if (a.dtype == UOCR_DTYPE_BF16)
    return small ? launch<__nv_bfloat16, 16>(a, j, stream) : launch<__nv_bfloat16, kEachMost>(a, j, stream);
  return small ? launch<float, 16>(a, j, stream) : launch<float, kEachMost>(a, j, stream);
}

}  // namespace uocr_b200
