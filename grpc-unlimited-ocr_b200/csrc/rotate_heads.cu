// Query and key heads normalised, rotated and appended to a cache
// (uocr_rotate_heads).
//
// y = x * rsqrt(mean(x^2) + eps) * gain per head, then (a, b) -> (a cos - b sin,
// b cos + a sin) over the pairs of the first rotary_dim dimensions, in fp32,
// rounded once to bf16. One pass: every element is read once and written once,
// so the bound is memory, and for few rows the launch and one round of loads.
#include <algorithm>

#include "beam.h"
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kMaxPairs = 128;  // head_dim 256
constexpr int kMaxThreads = 512;
constexpr int kBatch = 2;              // rows of a step of a resident block
constexpr int kStages = 3;             // its steps under way
constexpr int kHelpers = 64;           // its threads that form turns
constexpr int kStreamThreads = 1024;
constexpr int kThreadsOfSm = 1152;     // with at most 56 registers
constexpr size_t kSmemOfSm = 224 << 10;

__device__ __forceinline__ void load4(const float* p, bool vec, float* v) {
  if (vec) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[i];
  }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, bool vec, float* v) {
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(u.x));
    const float2 b = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(u.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __bfloat162float(p[i]);
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, const float* v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  if (vec) {
    *reinterpret_cast<uint2*>(p) =
        make_uint2(reinterpret_cast<const uint32_t&>(a), reinterpret_cast<const uint32_t&>(b));
  } else {
    p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
  }
}

struct Rotate {
  const void* q;
  const void* k;
  const void* v;
  const float* q_norm;
  const float* k_norm;
  const float* inv_freq;
  const int* positions;
  const int* cache_rows;
  const int* slots;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_cache;
  __nv_bfloat16* v_cache;
  int64_t ldq, ldk, ldv, ldqo, cache_stride, head_stride;
  int64_t caches, capacity;
  int64_t rows;
  int q_heads, kv_heads, dim, rot;
  uint32_t row_bytes;  // of a row's q, k and v in the ring
  float eps, magnitude, inv_dim;
  bool vec_in, vec_out, vec_gain;  // rows, gains allow 4 elements at a time
  bool bulk;                       // rows allow bulk copies
  ErrorWord* err;
};

// A thread takes 8 elements of a head: in the half layout 4 of a half and the 4
// that they pair with, so that a pair never leaves its thread; in the interleaved
// one, and of v, 8 in a row. kLanes threads (a power of two, at least head_dim / 8)
// share a head and its norm's sum. The row's cosines and sines are formed once and
// shared by all heads.

// One of a row's angles in turns, reduced in 64 bits: what is left of a far
// position is exact to 2^-25 of a turn.
__device__ __forceinline__ float2 turn_of(int position, float inv_freq, float magnitude) {
  const double turns = position * (static_cast<double>(inv_freq) * 0.15915494309189533577);
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c * magnitude, s * magnitude);
}

// Where row `row` goes in a cache's head, -1 where it has no place (recorded).
__device__ __forceinline__ int64_t place_of(const Rotate& a, int64_t row, int cache, int slot) {
  if (cache >= 0 && cache < a.caches && slot >= 0 && slot < a.capacity)
    return cache * a.cache_stride + static_cast<int64_t>(slot) * a.dim;
  raise_error(a.err, kDevBadIndex, kSiteCachePlace, static_cast<int>(row),
              cache >= 0 && cache < a.caches ? slot : cache);
  return -1;
}

// What a thread has of a head: where its elements lie, and what becomes of them.
template <int kLanes, bool kInterleaved>
struct Unit {
  int at0, at1, pair0;
  bool is_q, is_v, work, rotated;
  int head;
  __device__ __forceinline__ Unit(const Rotate& a, int h) : head(h) {
    const int unit = threadIdx.x % kLanes, half = a.rot / 2;
    is_q = head < a.q_heads;
    is_v = head >= a.q_heads + a.kv_heads;
    work = head < a.q_heads + 2 * a.kv_heads && unit * 8 < a.dim;
    rotated = !is_v && unit * 4 < half;
    pair0 = unit * 4;
    at0 = unit * 8;
    at1 = unit * 8 + 4;
    if (!kInterleaved && !is_v) {
      at0 = rotated ? pair0 : half + pair0;  // the rest of the head: its two halves
      at1 = rotated ? pair0 + half : half + pair0 + (a.dim - a.rot) / 2;
    }
  }
  // The gains of the thread's elements, 1 without.
  __device__ __forceinline__ void load_gains(const Rotate& a, float* g) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = 1.0f;
    const float* gain = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
    if (gain != nullptr && work) {
      load4(gain + at0, a.vec_gain, g);
      load4(gain + at1, a.vec_gain, g + 4);
    }
  }
  // Its row's elements, without the row or place.
  __device__ __forceinline__ __nv_bfloat16* destination(const Rotate& a) const {
    return is_q   ? a.q_out + head * a.dim
           : is_v ? a.v_cache + (head - a.q_heads - a.kv_heads) * a.head_stride
                  : a.k_cache + (head - a.q_heads) * a.head_stride;
  }
  // All threads of a warp call it. scale: 1 / root of the mean square where the head is normed.
  __device__ __forceinline__ float root(const Rotate& a, const float* x) const {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    if (!work) sum = 0.0f;
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return rsqrtf(fmaf(sum, a.inv_dim, a.eps));
  }
  __device__ __forceinline__ bool normed(const Rotate& a) const {
    return !is_v && (is_q ? a.q_norm : a.k_norm) != nullptr;
  }
  // turn: of the thread's four pairs, 16-byte aligned.
  __device__ __forceinline__ void rotate(float* x, const float2* turn) const {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float4 two = *reinterpret_cast<const float4*>(turn + i);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float c = e == 0 ? two.x : two.z, s = e == 0 ? two.y : two.w;
        float& u = kInterleaved ? x[2 * (i + e)] : x[i + e];
        float& w = kInterleaved ? x[2 * (i + e) + 1] : x[i + e + 4];
        const float u0 = u, w0 = w;
        u = u0 * c - w0 * s;
        w = w0 * c + u0 * s;
      }
    }
  }
};

// A block takes a row: for few rows, and rows at any address.
template <typename T, int kLanes, bool kInterleaved>
__global__ void __launch_bounds__(kMaxThreads) rotate_heads_kernel(Rotate a) {
  __shared__ __align__(16) float2 turn[kMaxPairs];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const int heads = a.q_heads + 2 * a.kv_heads, half = a.rot / 2;
  const int position = a.positions[row];
  for (int p = threadIdx.x; p < half; p += blockDim.x) turn[p] = turn_of(position, a.inv_freq[p], a.magnitude);
  const int64_t place = a.kv_heads == 0 ? -1
                                        : place_of(a, row, a.cache_rows != nullptr ? a.cache_rows[row] : static_cast<int>(row),
                                                   a.slots != nullptr ? a.slots[row] : position);
  __syncthreads();
  const bool any_norm = a.q_norm != nullptr || a.k_norm != nullptr;
  for (int h0 = 0; h0 < heads; h0 += blockDim.x / kLanes) {
    const Unit<kLanes, kInterleaved> u(a, h0 + threadIdx.x / kLanes);
    float x[8];
    if (u.work) {
      const T* src = u.is_q   ? static_cast<const T*>(a.q) + row * a.ldq + u.head * a.dim
                     : u.is_v ? static_cast<const T*>(a.v) + row * a.ldv + (u.head - a.q_heads - a.kv_heads) * a.dim
                              : static_cast<const T*>(a.k) + row * a.ldk + (u.head - a.q_heads) * a.dim;
      load4(src + u.at0, a.vec_in, x);
      load4(src + u.at1, a.vec_in, x + 4);
    }
    if (any_norm) {
      const float inv = u.root(a, x);
      float g[8];
      u.load_gains(a, g);
      if (u.normed(a)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = g[i] * (x[i] * inv);
      }
    }
    if (!u.work || (!u.is_q && place < 0)) continue;
    if (u.rotated) u.rotate(x, turn + u.pair0);
    __nv_bfloat16* dst = u.destination(a) + (u.is_q ? row * a.ldqo : place);
    const bool vec = !u.is_q || a.vec_out;
    store4(dst + u.at0, vec, x);
    store4(dst + u.at1, vec, x + 4);
  }
}

// A resident block goes from kBatch rows to the next, a thread keeping to its head
// and place in it: the rows come by bulk copies into a ring in shared memory, so
// that what is under way does not hang on the registers of waiting threads, and
// all that does not change from row to row is formed once. Warps of their own form
// the rows' turns and places, a batch ahead, and ask for the copies. A block a row
// took 164 us and 300 instructions a thread where this takes 94, 32768 rows of 24
// fp32 heads (92 at the copy rate); batches of 1, 2 and 4 rows 120, 94 and 102.
template <typename T, int kLanes, bool kInterleaved, bool kNorm>
__global__ void __launch_bounds__(kStreamThreads) rotate_stream_kernel(Rotate a, int workers) {
  extern __shared__ __align__(16) unsigned char ring[];  // [kStages][kBatch][row_bytes]
  __shared__ __align__(16) float2 turn[2][kBatch][kMaxPairs];
  __shared__ int64_t places[2][kBatch];
  __shared__ uint64_t full[kStages];
  __shared__ int lost;  // a copy that never came
  const int half = a.rot / 2;
  const int64_t batches = (a.rows + kBatch - 1) / kBatch, step = gridDim.x;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    lost = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int64_t first = blockIdx.x;
  if (static_cast<int>(threadIdx.x) >= workers) {
    const int helper = static_cast<int>(threadIdx.x) - workers, helpers = static_cast<int>(blockDim.x) - workers;
    const uint32_t q_bytes = a.q_heads * a.dim * sizeof(T), kv_bytes = a.kv_heads * a.dim * sizeof(T);
    auto fill = [&](int64_t batch, int stage) {  // by one thread
      if (batch >= batches) return;
      const int64_t row0 = batch * kBatch;
      const int n = static_cast<int>(min(static_cast<int64_t>(kBatch), a.rows - row0));
      mbar_arrive_expect_tx(&full[stage], n * a.row_bytes);
      for (int b = 0; b < n; ++b) {
        unsigned char* to = ring + (stage * kBatch + b) * a.row_bytes;
        if (q_bytes > 0) bulk_g2s(to, static_cast<const T*>(a.q) + (row0 + b) * a.ldq, q_bytes, &full[stage]);
        if (kv_bytes == 0) continue;
        bulk_g2s(to + q_bytes, static_cast<const T*>(a.k) + (row0 + b) * a.ldk, kv_bytes, &full[stage]);
        bulk_g2s(to + q_bytes + kv_bytes, static_cast<const T*>(a.v) + (row0 + b) * a.ldv, kv_bytes, &full[stage]);
      }
    };
    // What a batch's turns and places need is read a batch before they are formed.
    int position[kBatch] = {}, cache = 0, slot = 0;
    auto read = [&](int64_t batch) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (batch * kBatch + b < a.rows) position[b] = a.positions[batch * kBatch + b];
      const int64_t row = batch * kBatch + helper;
      if (helper >= kBatch || row >= a.rows || a.kv_heads == 0) return;
      cache = a.cache_rows != nullptr ? a.cache_rows[row] : static_cast<int>(row);
      slot = a.slots != nullptr ? a.slots[row] : a.positions[row];
    };
    auto form = [&](int64_t batch, int k) {
      if (batch >= batches) return;
      for (int p = helper; p < half; p += helpers) {
        const float freq = a.inv_freq[p];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) turn[k][b][p] = turn_of(position[b], freq, a.magnitude);
      }
      const int64_t row = batch * kBatch + helper;
      if (helper < kBatch && row < a.rows && a.kv_heads > 0) places[k][helper] = place_of(a, row, cache, slot);
    };
    if (helper == 0)
      for (int i = 0; i < kStages; ++i) fill(first + i * step, i);
    read(first);
    form(first, 0);
    read(first + step);
    __syncthreads();
    int stage = 0, phase = 0, k = 0;
    for (int64_t batch = first; batch < batches; batch += step, k ^= 1) {
      form(batch + step, k ^ 1);
      read(batch + 2 * step);
      __syncthreads();  // the stage has been read, the next turns are there
      if (lost != 0) {
        // Nothing more is asked for; what is under way has to land before the block ends.
        if (helper == 0) {
          raise_error(a.err, kDevWaitTimeout, kSiteCachePlace, static_cast<int>(batch), stage);
          for (int i = 1; i < kStages; ++i) {
            const int s = (stage + i) % kStages;
            if (batch + i * step < batches) mbar_wait(&full[s], s > stage ? phase : phase ^ 1);
          }
        }
        return;
      }
      if (helper == 0) fill(batch + kStages * step, stage);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    return;
  }
  const Unit<kLanes, kInterleaved> u(a, threadIdx.x / kLanes);
  float g[8];
  if (kNorm) u.load_gains(a, g);
  const bool normed = u.normed(a), vec = !u.is_q || a.vec_out;
  __nv_bfloat16* const to = u.destination(a);
  const unsigned char* const from = ring + u.head * a.dim * sizeof(T);
  __syncthreads();
  int stage = 0, phase = 0, k = 0;
  for (int64_t batch = first; batch < batches; batch += step, k ^= 1) {
    if (!mbar_wait(&full[stage], phase)) lost = 1;
    float x[kBatch][8];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (!u.work) continue;
      const T* src = reinterpret_cast<const T*>(from + (stage * kBatch + b) * a.row_bytes);
      load4(src + u.at0, true, x[b]);
      load4(src + u.at1, true, x[b] + 4);
    }
    if (kNorm) {
      float inv[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) inv[b] = u.root(a, x[b]);
      if (normed) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[b][i] = g[i] * (x[b][i] * inv[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t row = batch * kBatch + b;
      const int64_t place = u.is_q ? row * a.ldqo : places[k][b];
      if (!u.work || row >= a.rows || place < 0) continue;
      if (u.rotated) u.rotate(x[b], turn[k][b] + u.pair0);
      store4(to + place + u.at0, vec, x[b]);
      store4(to + place + u.at1, vec, x[b] + 4);
    }
    __syncthreads();  // the stage has been read, the next turns are there
    if (lost != 0) return;
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

template <typename T, int kLanes, bool kInterleaved, bool kNorm>
cudaError_t launch_stream(const Rotate& r, int blocks, int workers, size_t smem, cudaStream_t stream) {
  cudaError_t st = allow_max_dynamic_smem_once<rotate_stream_kernel<T, kLanes, kInterleaved, kNorm>>();
  if (st != cudaSuccess) return st;
  return launch_pdl(rotate_stream_kernel<T, kLanes, kInterleaved, kNorm>, static_cast<unsigned>(148 * blocks),
                    workers + kHelpers, smem, stream, r, workers);
}

template <typename T, int kLanes, bool kInterleaved>
cudaError_t launch(const uocr_rotate_heads_args& a, Rotate r, cudaStream_t stream) {
  const int heads = r.q_heads + 2 * r.kv_heads;
  r.row_bytes = static_cast<uint32_t>(heads * r.dim * sizeof(T));
  const size_t smem = static_cast<size_t>(kStages) * kBatch * r.row_bytes;
  // Rows for a step of every resident block, all of them at 16 bytes, whose heads fit side by side. 296, 592 and 1184 rows
  // of 24 fp32 heads take 3.8, 3.9 and 5.7 us that way and 3.0, 4.3 and 6.6 with a block a row.
  const int workers = (heads * kLanes + 31) / 32 * 32;
  if (r.bulk && workers + kHelpers <= kStreamThreads) {
    const int blocks = static_cast<int>(
        std::min<size_t>(kSmemOfSm / (smem + sizeof(float2) * 2 * kBatch * kMaxPairs + 1024), kThreadsOfSm / (workers + kHelpers)));
    if (blocks > 0 && a.rows >= kBatch * 148 * blocks)
      return r.q_norm != nullptr || r.k_norm != nullptr
                 ? launch_stream<T, kLanes, kInterleaved, true>(r, blocks, workers, smem, stream)
                 : launch_stream<T, kLanes, kInterleaved, false>(r, blocks, workers, smem, stream);
  }
  const int passes = (heads * kLanes + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((heads + passes - 1) / passes * kLanes + 31) / 32 * 32;
  return launch_pdl(rotate_heads_kernel<T, kLanes, kInterleaved>, static_cast<unsigned>(a.rows), threads, 0, stream, r);
}

template <typename T, int kLanes>
cudaError_t launch(const uocr_rotate_heads_args& a, const Rotate& r, cudaStream_t stream) {
  return a.interleaved != 0 ? launch<T, kLanes, true>(a, r, stream) : launch<T, kLanes, false>(a, r, stream);
}

template <typename T>
cudaError_t choose(const uocr_rotate_heads_args& a, const Rotate& r, cudaStream_t stream) {
  if (r.dim <= 64) return launch<T, 8>(a, r, stream);
  if (r.dim <= 128) return launch<T, 16>(a, r, stream);
  return launch<T, 32>(a, r, stream);
}

}  // namespace

cudaError_t launch_rotate_heads(const uocr_rotate_heads_args& a, ErrorWord* err, cudaStream_t stream) {
  Rotate r{};
  r.q = a.q, r.k = a.k, r.v = a.v;
  r.q_norm = a.q_norm, r.k_norm = a.k_norm;
  r.inv_freq = a.inv_freq, r.positions = a.positions, r.cache_rows = a.cache_rows, r.slots = a.slots;
  r.q_out = reinterpret_cast<__nv_bfloat16*>(a.q_out);
  r.k_cache = reinterpret_cast<__nv_bfloat16*>(a.k_cache);
  r.v_cache = reinterpret_cast<__nv_bfloat16*>(a.v_cache);
  r.ldq = a.ldq, r.ldk = a.ldk, r.ldv = a.ldv, r.ldqo = a.ldqo;
  r.cache_stride = a.cache_stride, r.head_stride = a.head_stride;
  r.caches = a.caches, r.capacity = a.capacity;
  r.rows = a.rows;
  r.q_heads = static_cast<int>(a.q_heads), r.kv_heads = static_cast<int>(a.kv_heads);
  r.dim = static_cast<int>(a.head_dim), r.rot = static_cast<int>(a.rotary_dim);
  r.eps = a.eps, r.magnitude = a.magnitude;
  const size_t need = a.dtype == UOCR_DTYPE_BF16 ? 8 : 16, eb = need / 4;
  auto fits = [&](const void* p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % need == 0 && static_cast<size_t>(ld) * eb % need == 0;
  };
  r.vec_in = fits(a.q, a.ldq) && fits(a.k, a.ldk) && fits(a.v, a.ldv);
  auto at16 = [&](const void* p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && static_cast<size_t>(ld) * eb % 16 == 0;
  };
  r.bulk = at16(a.q, a.ldq) && at16(a.k, a.ldk) && at16(a.v, a.ldv);
  r.vec_gain = reinterpret_cast<uintptr_t>(a.q_norm) % 16 == 0 && reinterpret_cast<uintptr_t>(a.k_norm) % 16 == 0;
  r.vec_out = reinterpret_cast<uintptr_t>(a.q_out) % 8 == 0 && a.ldqo % 4 == 0;
  r.inv_dim = 1.0f / static_cast<float>(r.dim);
  r.err = err;
  return a.dtype == UOCR_DTYPE_BF16 ? choose<__nv_bfloat16>(a, r, stream) : choose<float>(a, r, stream);
}

}  // namespace uocr_b200
