// Activations to int8 with one scale per token (include/uocr_int8.h).
//
// s = max|x| * fl(1 / 127), q = clamp(rint(x / s), +-127) with an IEEE division,
// so the bits do not depend on the variant below. (quantize_rows_kernel in
// weights.cu divides the maximum by 127: its s may differ in the last bit.)
// One pass: a thread keeps its part of the row in registers between the
// maximum and the rounding.
#include <cfloat>

#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8;   // elements a thread takes at a time
constexpr int kKeep = 8;    // chunks of a row a thread keeps

// Elements c .. c + 7 of a row; `vec`: the row is 16-byte aligned and holds all eight.
__device__ __forceinline__ void load8(const float* row, int64_t c, int64_t cols, bool vec, float (&v)[kChunk]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) v[i] = c + i < cols ? row[c + i] : 0.0f;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* row, int64_t c, int64_t cols, bool vec,
                                      float (&v)[kChunk]) {
  if (vec) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of its fp32 value
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) v[i] = c + i < cols ? __bfloat162float(row[c + i]) : 0.0f;
}

// max over |v|, kept as bits: for non-negative floats the order of the bits is
// the order of the values, and infinities and NaNs come out on top.
__device__ __forceinline__ uint32_t peak8(const float (&v)[kChunk], uint32_t peak) {
#pragma unroll
  for (int i = 0; i < kChunk; ++i) peak = max(peak, __float_as_uint(v[i]) & 0x7fffffffu);
  return peak;
}

__device__ __forceinline__ void store8(const float (&v)[kChunk], float scale, bool finite, int8_t* row, int64_t c,
                                       int64_t cols) {
  uint32_t w[2] = {0u, 0u};
  if (finite) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float r = fminf(fmaxf(rintf(v[i] / scale), -127.0f), 127.0f);
      w[i / 4] |= (static_cast<uint32_t>(static_cast<int>(r)) & 0xffu) << (8 * (i % 4));
    }
  }
  if (c + kChunk <= cols) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (c + i < cols) row[c + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

// kPerRow threads (32: a warp, or the whole block) take a row; the part of a
// row beyond kPerRow * kKeep chunks is read a second time.
template <typename T, int kPerRow>
__global__ void __launch_bounds__(kThreads) quantize_tokens_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                                   int64_t ldx, bool aligned, int8_t* __restrict__ q,
                                                                   int64_t ldq, float* __restrict__ scales) {
  __shared__ uint32_t part[kThreads / 32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kPerRow) + threadIdx.x / kPerRow;
  if (row >= rows) return;  // whole warps; with kPerRow == kThreads never
  const int t = threadIdx.x % kPerRow;
  const T* src = x + row * ldx;
  int8_t* dst = q + row * ldq;
  float keep[kKeep][kChunk];
  uint32_t peak = 0u;
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int64_t c = static_cast<int64_t>(t + u * kPerRow) * kChunk;
    if (c < cols) load8(src, c, cols, aligned && c + kChunk <= cols, keep[u]);
  }
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int64_t c = static_cast<int64_t>(t + u * kPerRow) * kChunk;
    if (c < cols) peak = peak8(keep[u], peak);
  }
  for (int64_t c = static_cast<int64_t>(t + kKeep * kPerRow) * kChunk; c < cols; c += kPerRow * kChunk) {
    float v[kChunk];
    load8(src, c, cols, aligned && c + kChunk <= cols, v);
    peak = peak8(v, peak);
  }
  peak = __reduce_max_sync(0xffffffffu, peak);
  if (kPerRow > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPerRow / 32; ++w) peak = max(peak, part[w]);
  }
  const bool finite = peak < 0x7f800000u;
  const float scale = !finite       ? __uint_as_float(0x7fc00000u)
                      : peak == 0u  ? 1.0f
                                    : fmaxf(__uint_as_float(peak) * (1.0f / 127.0f), FLT_MIN);
  if (t == 0) scales[row] = scale;
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int64_t c = static_cast<int64_t>(t + u * kPerRow) * kChunk;
    if (c < cols) store8(keep[u], scale, finite, dst, c, cols);
  }
  for (int64_t c = static_cast<int64_t>(t + kKeep * kPerRow) * kChunk; c < cols; c += kPerRow * kChunk) {
    float v[kChunk];
    load8(src, c, cols, aligned && c + kChunk <= cols, v);
    store8(v, scale, finite, dst, c, cols);
  }
}

template <typename T>
cudaError_t launch(const T* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                   cudaStream_t stream) {
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * sizeof(T)) % 16 == 0;
  // A warp per row where a warp can keep the row; wider rows take a block.
  if (cols <= 32 * kKeep * kChunk) {
    const int64_t blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
    quantize_tokens_kernel<T, 32><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(x, rows, cols, ldx, aligned,
                                                                                          q, ldq, scales);
  } else {
    quantize_tokens_kernel<T, kThreads><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(x, rows, cols, ldx,
                                                                                              aligned, q, ldq, scales);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_tokens(const void* x, bool bf16, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                                   int64_t ldq, float* scales, cudaStream_t stream) {
  if (rows == 0) return cudaSuccess;
  return bf16 ? launch(static_cast<const __nv_bfloat16*>(x), rows, cols, ldx, q, ldq, scales, stream)
              : launch(static_cast<const float*>(x), rows, cols, ldx, q, ldq, scales, stream);
}

}  // namespace uocr_b200
