// C ABI of the 8-bit integer operators (include/uocr_int8.h): argument checks
// and launches. Host code only; the kernels are in quantize_tokens.cu,
// w8a8_gemm.cu and w8a8_rows.cu.
#include <cuda_runtime.h>

#include <string>

#include "../../include/uocr_int8.h"
#include "moe_kernels.h"
#include "w8a8.h"

using namespace uocr_b200;

namespace {

constexpr int64_t kMaxRows = 1 << 30;  // row coordinates, tiles' overhang included, are 32-bit

int bad(const char* op, const char* what) {
  return set_last_error(UOCR_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

int done(const char* op, cudaError_t st) {
  if (st == cudaSuccess) return UOCR_OK;
  return set_last_error(st == cudaErrorMemoryAllocation ? UOCR_ERR_OUT_OF_MEMORY : UOCR_ERR_CUDA,
                        std::string(op) + ": " + cudaGetErrorString(st));
}

bool int8_rows_ok(const int8_t* base, int64_t ld) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld % 16 == 0;
}

// What the two products check alike. rows, groups and the pointers that may
// be null are the caller's.
int check_product(const char* op, const int8_t* x, const float* x_scales, const int8_t* w, const float* w_scales,
                  const void* y, int64_t rows, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int64_t ldy,
                  int32_t y_dtype, int32_t reserved) {
  if (rows < 0 || n < 0 || k <= 0 || rows > kMaxRows || n > kMaxRows) return bad(op, "bad shape");
  if (k > UOCR_W8A8_MAX_K) return set_last_error(UOCR_ERR_UNSUPPORTED, std::string(op) + ": k above 131071");
  if (y_dtype != UOCR_DTYPE_F32 && y_dtype != UOCR_DTYPE_BF16) return bad(op, "y must be f32 or bf16");
  if (reserved != 0) return bad(op, "reserved must be 0");
  if (rows == 0 || n == 0) return UOCR_OK;
  if (x_scales == nullptr || w_scales == nullptr || y == nullptr || x == nullptr || w == nullptr)
    return bad(op, "null pointer");
  if (ldx < k || ldw < k || ldy < n) return bad(op, "a pitch is smaller than its row");
  if (!int8_rows_ok(x, ldx) || !int8_rows_ok(w, ldw))
    return bad(op, "int8 rows must start at 16-byte boundaries (base pointers, and pitches a multiple of 16)");
  if (reinterpret_cast<uintptr_t>(y) % (y_dtype == UOCR_DTYPE_F32 ? 4 : 2) != 0) return bad(op, "y is misaligned");
  return UOCR_OK;
}

}  // namespace

extern "C" {

int uocr_quantize_tokens(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                         int64_t ldq, float* scales, void* stream) {
  const char* op = "quantize_tokens";
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxRows) return bad(op, "bad shape");
  if (dtype != UOCR_DTYPE_F32 && dtype != UOCR_DTYPE_BF16) return bad(op, "x must be f32 or bf16");
  if (rows == 0) return UOCR_OK;
  if (scales == nullptr || (cols > 0 && (x == nullptr || q == nullptr))) return bad(op, "null pointer");
  if (ldx < cols || ldq < cols) return bad(op, "a pitch is smaller than its row");
  if (!int8_rows_ok(q, ldq))
    return bad(op, "int8 rows must start at 16-byte boundaries (base pointer, and pitch a multiple of 16)");
  if (reinterpret_cast<uintptr_t>(x) % (dtype == UOCR_DTYPE_F32 ? 4 : 2) != 0) return bad(op, "x is misaligned");
  return done(op, launch_quantize_tokens(x, dtype == UOCR_DTYPE_BF16, rows, cols, ldx, q, ldq, scales,
                                         static_cast<cudaStream_t>(stream)));
}

int uocr_linear_w8a8(const uocr_linear_w8a8_args* a, void* stream) {
  const char* op = "linear_w8a8";
  if (a == nullptr) return bad(op, "null arguments");
  const int rc = check_product(op, a->x, a->x_scales, a->w, a->w_scales, a->y, a->m, a->n, a->k, a->ldx, a->ldw,
                               a->ldy, a->y_dtype, a->reserved);
  if (rc != UOCR_OK || a->m == 0 || a->n == 0) return rc;
  if (a->residual != nullptr) {
    if (a->ldr < a->n) return bad(op, "a pitch is smaller than its row");
    if (a->residual == a->y && a->ldr != a->ldy) return bad(op, "an in-place residual has y's pitch");
    if (reinterpret_cast<uintptr_t>(a->residual) % (a->y_dtype == UOCR_DTYPE_F32 ? 4 : 2) != 0)
      return bad(op, "residual is misaligned");
  }
  W8a8 p{};
  p.x = a->x;
  p.x_scales = a->x_scales;
  p.x_rows = a->m;
  p.rows = a->m;
  p.groups = 1;
  p.n = a->n;
  p.k = a->k;
  p.w = a->w;
  p.w_scales = a->w_scales;
  p.bias = a->bias;
  p.residual = a->residual;
  p.y = a->y;
  p.ldx = a->ldx;
  p.ldw = a->ldw;
  p.ldr = a->ldr;
  p.ldy = a->ldy;
  p.y_bf16 = a->y_dtype == UOCR_DTYPE_BF16;
  const cudaError_t st = ops_error_word(&p.err);
  return done(op, st != cudaSuccess ? st : launch_w8a8(p, static_cast<cudaStream_t>(stream)));
}

int uocr_grouped_w8a8_workspace(const uocr_grouped_w8a8_args* a, int64_t* bytes) {
  const char* op = "grouped_w8a8_workspace";
  if (a == nullptr || bytes == nullptr) return bad(op, "null arguments");
  if (a->rows < 0 || a->k <= 0 || a->rows > kMaxRows || a->k > UOCR_W8A8_MAX_K) return bad(op, "bad shape");
  *bytes = a->row_index == nullptr ? 0 : static_cast<int64_t>(w8a8_gather_bytes(a->rows, a->groups, a->k));
  return UOCR_OK;
}

int uocr_grouped_linear_w8a8(const uocr_grouped_w8a8_args* a, void* stream) {
  const char* op = "grouped_linear_w8a8";
  if (a == nullptr) return bad(op, "null arguments");
  if (a->groups < 0) return bad(op, "bad shape");
  if (a->groups > UOCR_W8A8_MAX_GROUPS)
    return set_last_error(UOCR_ERR_UNSUPPORTED, std::string(op) + ": more than 512 groups");
  const int rc = check_product(op, a->x, a->x_scales, a->w, a->w_scales, a->y, a->rows, a->n, a->k, a->ldx, a->ldw,
                               a->ldy, a->y_dtype, a->reserved);
  if (rc != UOCR_OK || a->rows == 0 || a->n == 0 || a->groups == 0) return rc;
  if (a->offsets == nullptr) return bad(op, "null pointer");
  if (a->groups * a->n > kMaxRows)
    return set_last_error(UOCR_ERR_UNSUPPORTED, std::string(op) + ": groups * n above 2^30");
  if (a->x_rows <= 0 || a->x_rows > kMaxRows) return bad(op, "bad shape");
  if (a->row_index == nullptr && a->x_rows != a->rows) return bad(op, "without row_index x has one row per output row");
  if (a->w_up != nullptr && (a->w_up_scales == nullptr || reinterpret_cast<uintptr_t>(a->w_up) % 16 != 0))
    return bad(op, "w_up needs its scales and a 16-byte aligned base");
  W8a8 p{};
  p.x = a->x;
  p.x_scales = a->x_scales;
  p.row_index = a->row_index;
  p.x_rows = a->x_rows;
  p.starts = a->offsets;
  p.rows = a->rows;
  p.groups = a->groups;
  p.n = a->n;
  p.k = a->k;
  p.w = a->w;
  p.w_scales = a->w_scales;
  p.w_up = a->w_up;
  p.w_up_scales = a->w_up_scales;
  p.y = a->y;
  p.ldx = a->ldx;
  p.ldw = a->ldw;
  p.ldy = a->ldy;
  p.y_bf16 = a->y_dtype == UOCR_DTYPE_BF16;
  p.workspace = static_cast<int8_t*>(a->workspace);
  const size_t need = a->row_index == nullptr ? 0 : w8a8_gather_bytes(a->rows, a->groups, a->k);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < static_cast<int64_t>(need) ||
                   reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0))
    return bad(op, "the workspace is missing, too small or not 16-byte aligned (uocr_grouped_w8a8_workspace)");
  const cudaError_t st = ops_error_word(&p.err);
  return done(op, st != cudaSuccess ? st : launch_w8a8(p, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
