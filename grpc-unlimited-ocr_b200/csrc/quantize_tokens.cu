// Activations to int8 with one scale per token (include/uocr_int8.h).
//
// s = max|x| * fl(1 / 127), q = rint(x / s) with the quotient as an IEEE
// division rounds it, whatever the variant below. (quantize_rows_kernel in
// weights.cu divides the maximum by 127: its s may differ in the last bit. The
// product is what elementwise tensor code makes of a division by a constant, so
// that a caller who quantises that way has the same bits.)
// |x| / s is at most 127 (1 + 2^-22), so nothing is clamped. One pass: a thread
// keeps its part of the row in registers between the maximum and the rounding.
//
// Bound by bytes in fp32 (32768 x 2048: 49 us, the card's copy rate) and by
// latency in bf16, whose rows take as long with half the bytes (54 us; 4096 x
// 2048 6.9, 1.8 times its floor): a block's loads are out at once and nothing of
// the next row is, so that its warps mostly wait for them (39 % of DRAM, 52 % of
// the issue slots, the ALUs 45 %).
#include <cfloat>

#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8;   // elements a thread takes at a time

// Elements c .. c + 7 of a row; `vec`: the row is 16-byte aligned and holds all eight.
__device__ __forceinline__ void load8(const float* row, int c, int cols, bool vec, float (&v)[kChunk]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) v[i] = c + i < cols ? row[c + i] : 0.0f;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* row, int c, int cols, bool vec, float (&v)[kChunk]) {
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

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

struct RowScale {
  float scale;
  uint64_t inv2, minus2;  // 1 / scale and -scale, twice
  bool finite, tiny;
};

// rint(v / scale) of eight elements to bytes. The quotient by Markstein's
// method: with y = RN(1 / s), q <- RN(q + RN(v - q s) y) from q = RN(v y) is
// within an ulp of v / s after one step and RN(v / s) after two, in packed
// products (an IEEE division and a conversion for each element made the kernel
// three times slower). Adding 1.5 * 2^23 rounds to an integer, the low byte of
// the sum. Rows below 2^-90, where a remainder could underflow, are divided.
__device__ __forceinline__ void store8(const float (&v)[kChunk], const RowScale& s, int8_t* row, int c, int cols) {
  constexpr float kRound = 12582912.0f;
  const uint64_t zero2 = 0, round2 = pair(kRound, kRound), one2 = pair(1.0f, 1.0f);
  uint32_t r[kChunk];
  if (s.tiny) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) r[i] = __float_as_uint(v[i] / s.scale + kRound);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; i += 2) {
      const uint64_t x = pair(v[i], v[i + 1]);
      uint64_t q = fma2(x, s.inv2, zero2);
      q = fma2(fma2(q, s.minus2, x), s.inv2, q);
      q = fma2(fma2(q, s.minus2, x), s.inv2, q);
      const uint64_t b = fma2(q, one2, round2);
      r[i] = static_cast<uint32_t>(b);
      r[i + 1] = static_cast<uint32_t>(b >> 32);
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = s.finite ? __byte_perm(__byte_perm(r[4 * h], r[4 * h + 1], 0x0040),
                                  __byte_perm(r[4 * h + 2], r[4 * h + 3], 0x0040), 0x5410)
                    : 0u;
  if (c + kChunk <= cols) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (c + i < cols) row[c + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

// kPerRow threads (a warp, several, or the whole block) take a row and keep
// kKeep chunks of it each; what is beyond is read a second time. kAligned: x's rows
// start at 16-byte boundaries.
template <typename T, int kPerRow, int kKeep, bool kAligned>
__global__ void __launch_bounds__(kThreads) quantize_tokens_kernel(const T* x, int64_t rows, int cols,
                                                                   int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                                   float* __restrict__ scales) {
  __shared__ uint32_t part[kThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kPerRow) + threadIdx.x / kPerRow;
  if (kPerRow <= 32 && row >= rows) return;
  if (row >= rows) cols = 0;  // goes along to the barrier
  const int c0 = static_cast<int>(threadIdx.x % kPerRow) * kChunk;
  constexpr int kStride = kPerRow * kChunk;
  const T* src = x + row * ldx;
  int8_t* dst = q + row * ldq;
  float keep[kKeep][kChunk];
  uint32_t peak = 0u;
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int c = c0 + u * kStride;
    if (c < cols) load8(src, c, cols, kAligned && c + kChunk <= cols, keep[u]);
  }
#pragma unroll
  for (int u = 0; u < kKeep; ++u)
    if (c0 + u * kStride < cols) peak = peak8(keep[u], peak);
  for (int c = c0 + kKeep * kStride; c < cols; c += kStride) {
    float v[kChunk];
    load8(src, c, cols, kAligned && c + kChunk <= cols, v);
    peak = peak8(v, peak);
  }
  peak = __reduce_max_sync(0xffffffffu, peak);
  if (kPerRow > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPerRow / 32; ++w) peak = max(peak, part[threadIdx.x / kPerRow * (kPerRow / 32) + w]);
    if (row >= rows) return;
  }
  RowScale s;
  s.finite = peak < 0x7f800000u;
  s.scale = !s.finite    ? __uint_as_float(0x7fc00000u)
            : peak == 0u ? 1.0f
                         : fmaxf(__uint_as_float(peak) * (1.0f / 127.0f), FLT_MIN);
  s.tiny = s.scale < 0x1p-90f;
  s.inv2 = pair(1.0f / s.scale, 1.0f / s.scale);
  s.minus2 = pair(-s.scale, -s.scale);
  if (c0 == 0) scales[row] = s.scale;
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int c = c0 + u * kStride;
    if (c < cols) store8(keep[u], s, dst, c, cols);
  }
  for (int c = c0 + kKeep * kStride; c < cols; c += kStride) {
    float v[kChunk];
    load8(src, c, cols, kAligned && c + kChunk <= cols, v);
    store8(v, s, dst, c, cols);
  }
}

template <int kPerRow, int kKeep, bool kAligned, typename T>
cudaError_t launch(const T* x, int64_t rows, int cols, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                   cudaStream_t stream) {
  constexpr int kRows = kThreads / kPerRow;
  return launch_pdl(quantize_tokens_kernel<T, kPerRow, kKeep, kAligned>,
                    static_cast<unsigned>((rows + kRows - 1) / kRows), kThreads, 0, stream, x, rows, cols, ldx, q, ldq,
                    scales);
}

template <bool kAligned, typename T>
cudaError_t choose(const T* x, int64_t rows, int cols, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                   cudaStream_t stream) {
  // Two chunks a thread: enough in flight, and few idle threads. Measured in us:
  // 4096 x 2048 bf16 12.3 by a warp a row, 7.5 by 128 threads (since then 6.9), 8.1 by
  // 256 of one chunk (3.85 at the card's copy rate); 24576 x 1024 bf16 27 by a warp, 23 by
  // 64 threads; 32768 x 2048 fp32 49.5 by 128 threads (the copy rate: 51). Few
  // rows are a matter of latency: 1 x 2048 1.6 by 256 threads, 5.5 by a warp.
  if (cols <= 512) return launch<32, 2, kAligned>(x, rows, cols, ldx, q, ldq, scales, stream);
  if (cols <= 2048 && rows <= 592) return launch<256, 1, kAligned>(x, rows, cols, ldx, q, ldq, scales, stream);
  if (cols <= 1024) return launch<64, 2, kAligned>(x, rows, cols, ldx, q, ldq, scales, stream);
  if (cols <= 2048) return launch<128, 2, kAligned>(x, rows, cols, ldx, q, ldq, scales, stream);
  return launch<256, 4, kAligned>(x, rows, cols, ldx, q, ldq, scales, stream);
}

template <typename T>
cudaError_t choose(const void* xv, int64_t rows, int cols, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                   cudaStream_t stream) {
  const T* x = static_cast<const T*>(xv);
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * sizeof(T)) % 16 == 0
             ? choose<true>(x, rows, cols, ldx, q, ldq, scales, stream)
             : choose<false>(x, rows, cols, ldx, q, ldq, scales, stream);
}

}  // namespace

cudaError_t launch_quantize_tokens(const void* x, bool bf16, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                                   int64_t ldq, float* scales, cudaStream_t stream) {
  if (rows == 0) return cudaSuccess;
  const int n = static_cast<int>(cols);
  return bf16 ? choose<__nv_bfloat16>(x, rows, n, ldx, q, ldq, scales, stream)
              : choose<float>(x, rows, n, ldx, q, ldq, scales, stream);
}

}  // namespace uocr_b200
