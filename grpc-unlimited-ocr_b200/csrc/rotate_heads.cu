// Query and key heads normalised, rotated and appended to a cache
// (uocr_rotate_heads).
//
// y = x * rsqrt(mean(x^2) + eps) * gain per head, then (a, b) -> (a cos - b sin,
// b cos + a sin) over the pairs of the first rotary_dim dimensions, in fp32,
// rounded once to bf16. One pass: every element is read once and written once,
// so the bound is memory, and for few rows the launch and one round of loads.
#include "beam.h"
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kMaxPairs = 128;  // head_dim 256
constexpr int kMaxThreads = 512;

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
  int q_heads, kv_heads, dim, rot;
  float eps, magnitude;
  bool vec_in, vec_out;  // rows allow 4 elements at a time
  ErrorWord* err;
};

// A block takes a row. A thread takes 8 elements of a head: in the half layout
// 4 of a half and the 4 that they pair with, so that a pair never leaves its
// thread; in the interleaved one, and of v, 8 in a row. kLanes threads (a power
// of two, at least head_dim / 8) share a head and its norm's sum. The row's
// cosines and sines are formed once and shared by all heads.
template <typename T, int kLanes, bool kInterleaved>
__global__ void __launch_bounds__(kMaxThreads) rotate_heads_kernel(Rotate a) {
  __shared__ float2 turn[kMaxPairs];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const int heads = a.q_heads + 2 * a.kv_heads, half = a.rot / 2;
  const int position = a.positions[row];
  // The angle in turns, reduced in 64 bits: what is left of a far position is
  // exact to 2^-25 of a turn.
  for (int p = threadIdx.x; p < half; p += blockDim.x) {
    const double turns = position * (static_cast<double>(a.inv_freq[p]) * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    turn[p] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  int64_t place = -1;  // of the row in a cache's head
  if (a.kv_heads > 0) {
    const int cache = a.cache_rows != nullptr ? a.cache_rows[row] : static_cast<int>(row);
    const int slot = a.slots != nullptr ? a.slots[row] : position;
    if (cache >= 0 && cache < a.caches && slot >= 0 && slot < a.capacity)
      place = cache * a.cache_stride + static_cast<int64_t>(slot) * a.dim;
    else if (threadIdx.x == 0)
      raise_error(a.err, kDevBadIndex, kSiteCachePlace, static_cast<int>(row),
                  cache >= 0 && cache < a.caches ? slot : cache);
  }
  __syncthreads();
  const int unit = threadIdx.x % kLanes;
  for (int h0 = 0; h0 < heads; h0 += blockDim.x / kLanes) {
    const int head = h0 + threadIdx.x / kLanes;
    const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.kv_heads;
    const bool work = head < heads && unit * 8 < a.dim;
    float x[8];
    int at0 = unit * 8, at1 = unit * 8 + 4;
    const bool rotated = !is_v && unit * 4 < half;
    if (!kInterleaved && !is_v) {
      const int p = unit * 4;
      at0 = rotated ? p : half + p;  // the rest of the head: its two halves
      at1 = rotated ? p + half : half + p + (a.dim - a.rot) / 2;
    }
    float sum = 0.0f;
    if (work) {
      const T* src = is_q ? static_cast<const T*>(a.q) + row * a.ldq + head * a.dim
                     : is_v
                         ? static_cast<const T*>(a.v) + row * a.ldv + (head - a.q_heads - a.kv_heads) * a.dim
                         : static_cast<const T*>(a.k) + row * a.ldk + (head - a.q_heads) * a.dim;
      load4(src + at0, a.vec_in, x);
      load4(src + at1, a.vec_in, x + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    }
    const float* gain = is_q ? a.q_norm : a.k_norm;
    if (a.q_norm != nullptr || a.k_norm != nullptr) {
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
    if (!work) continue;
    if (!is_v && gain != nullptr) {
      const float inv = rsqrtf(sum / static_cast<float>(a.dim) + a.eps);
      float g[8];
      load4(gain + at0, false, g);
      load4(gain + at1, false, g + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = g[i] * (x[i] * inv);
    }
    if (rotated) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = turn[unit * 4 + i];
        float& u = kInterleaved ? x[2 * i] : x[i];
        float& w = kInterleaved ? x[2 * i + 1] : x[i + 4];
        const float u0 = u, w0 = w;
        u = u0 * t.x - w0 * t.y;
        w = w0 * t.x + u0 * t.y;
      }
    }
    __nv_bfloat16* dst;
    bool vec = true;
    if (is_q) {
      dst = a.q_out + row * a.ldqo + head * a.dim;
      vec = a.vec_out;
    } else {
      if (place < 0) continue;
      dst = is_v ? a.v_cache + place + (head - a.q_heads - a.kv_heads) * a.head_stride
                 : a.k_cache + place + (head - a.q_heads) * a.head_stride;
    }
    store4(dst + at0, vec, x);
    store4(dst + at1, vec, x + 4);
  }
}

template <typename T, int kLanes>
cudaError_t launch(const uocr_rotate_heads_args& a, const Rotate& r, cudaStream_t stream) {
  const int heads = r.q_heads + 2 * r.kv_heads;
  const int passes = (heads * kLanes + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((heads + passes - 1) / passes * kLanes + 31) / 32 * 32;
  const unsigned grid = static_cast<unsigned>(a.rows);
  return a.interleaved != 0 ? launch_pdl(rotate_heads_kernel<T, kLanes, true>, grid, threads, 0, stream, r)
                            : launch_pdl(rotate_heads_kernel<T, kLanes, false>, grid, threads, 0, stream, r);
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
  r.q_heads = static_cast<int>(a.q_heads), r.kv_heads = static_cast<int>(a.kv_heads);
  r.dim = static_cast<int>(a.head_dim), r.rot = static_cast<int>(a.rotary_dim);
  r.eps = a.eps, r.magnitude = a.magnitude;
  const size_t need = a.dtype == UOCR_DTYPE_BF16 ? 8 : 16, eb = need / 4;
  auto fits = [&](const void* p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % need == 0 && static_cast<size_t>(ld) * eb % need == 0;
  };
  r.vec_in = fits(a.q, a.ldq) && fits(a.k, a.ldk) && fits(a.v, a.ldv);
  r.vec_out = reinterpret_cast<uintptr_t>(a.q_out) % 8 == 0 && a.ldqo % 4 == 0;
  r.err = err;
  return a.dtype == UOCR_DTYPE_BF16 ? choose<__nv_bfloat16>(a, r, stream) : choose<float>(a, r, stream);
}

}  // namespace uocr_b200
