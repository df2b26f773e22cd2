// Host interface of the 8-bit integer operators: the token quantiser
// (quantize_tokens.cu) and the products (w8a8_gemm.cu, w8a8_rows.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "moe_common.cuh"

namespace uocr_b200 {

// Launches a kernel that may start before the previous grid of the stream ends:
// every thread of it calls pdl_wait before it reads or writes global memory (a
// block that ended without would let the grid after it overtake the one before).
// Its inputs may still be being written when it starts: it reads them by plain
// loads, which stay behind that wait, and not as data that is read-only for the
// kernel's whole life (the non-coherent loads of __ldg and of const __restrict__
// pointers, which need not).
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                       Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

// q, scales = int8 rows of x [rows, cols] (fp32 or bf16, pitch ldx) with one
// scale per row; q rows at pitch ldq, 16-byte aligned.
cudaError_t launch_quantize_tokens(const void* x, bool bf16, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                                   int64_t ldq, float* scales, cudaStream_t stream);

// y[r, c] = (sum_k x[row(r), k] w[g, c, k]) x_scales[row(r)] w_scales[g, c]
// (+ bias[c]) (+ residual[r, c]) for the rows r of group g; with w_up
// silu(that with w) * (that with w_up), without bias and residual.
struct W8a8 {
  const int8_t* x;
  const float* x_scales;
  const int* row_index;  // null: row(r) = r
  int64_t x_rows;
  const int* starts;     // [groups] first row of each group; null: one group of all rows
  const int* counts;     // [groups] rows of each group; null: starts has groups + 1 entries
  int64_t rows, groups, n, k;
  const int8_t* w;
  const float* w_scales;
  const int8_t* w_up;
  const float* w_up_scales;
  const float* bias;
  const void* residual;
  void* y;
  int64_t ldx, ldw, ldr, ldy;
  bool y_bf16;
  int8_t* workspace;     // with row_index: w8a8_gather_bytes, 16-byte aligned
  ErrorWord* err;
};
// Device memory a grouped product with row_index needs for its duration: the rows it names, copied together.
size_t w8a8_gather_bytes(int64_t rows, int64_t groups, int64_t k);
cudaError_t launch_w8a8(const W8a8& p, cudaStream_t stream);
// Sets the product kernels up on the current device (otherwise their first
// launch does); for callers whose first launch may be inside a stream capture.
cudaError_t prepare_w8a8();
// The kernel for few rows (w8a8_rows.cu); launch_w8a8 chooses.
cudaError_t launch_w8a8_rows(const W8a8& p, cudaStream_t stream);

// Values of y's type (and the residual's) as the epilogues take them.
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// silu(g) * u = g / (1 + exp(-g)) * u. The quotient to 2 ulp (__fdividef): an
// IEEE division branches, which keeps a thread's outputs from overlapping.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

}  // namespace uocr_b200
