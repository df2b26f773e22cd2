/* uocr_int8.h — C ABI of the 8-bit integer operators on B200 (W8A8).
 *
 * Matrix products of int8 activations (one fp32 scale per token) with int8
 * weights (one fp32 scale per output channel, the UOCR_WEIGHT_INT8 layout of
 * uocr_moe.h and what uocr_quantize_q8 writes with group = cols), and the
 * quantiser that makes the activations. The products sum in int32, which is
 * exact, so their results do not depend on the kernel or on any order; each
 * output is float(sum) * x_scale * w_scale, then the epilogue, in fp32, rounded
 * once to the output's type.
 *
 * Conventions are uocr_moe.h's: plain device pointers, a cudaStream_t passed as
 * void*, status codes with uocr_last_error(), nothing synchronises the stream
 * and nothing is allocated. Rows are row-major with a pitch ("ld") counted in
 * elements. An int8 row starts at a 16-byte boundary: base pointers 16-byte
 * aligned and int8 pitches a multiple of 16. Its width is free: the bytes from
 * the width up to the next multiple of 16 may be read, and are not used.
 */
#ifndef UOCR_INT8_H
#define UOCR_INT8_H

#include <stdint.h>

#include "uocr_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Row width and group count limits of the products: |q| <= 128, so a sum of
 * UOCR_W8A8_MAX_K products stays below 2^31. */
#define UOCR_W8A8_MAX_K 131071
#define UOCR_W8A8_MAX_GROUPS 512

/* q[r, c] = clamp(rint(x[r, c] / s), -127, 127) with s = scales[r] =
 * max_c |x[r, c]| * fl(1 / 127), the rule of uocr_quantize_q8 (src/model/cuda/
 * device_weight.cpp:11-26) with one group per row, but for the last bit of s
 * (a product here, a quotient there); x is fp32 or bf16 (dtype) and may be a
 * column range of wider rows (ldx >= cols). s is 1 for a row of zeros and at
 * least FLT_MIN otherwise. A row that holds a NaN or an infinity
 * gets s = NaN and q = 0, so every product of that row is NaN. */
int uocr_quantize_tokens(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                         int64_t ldq, float* scales, void* stream);

typedef struct uocr_linear_w8a8_args {
  const int8_t* x;         /* [m, k], pitch ldx */
  const float* x_scales;   /* [m] */
  const int8_t* w;         /* [n, k], pitch ldw */
  const float* w_scales;   /* [n] */
  const float* bias;       /* [n] or NULL */
  const void* residual;    /* [m, n] of y's type, pitch ldr, or NULL; may be y itself with ldr == ldy */
  void* y;                 /* [m, n], pitch ldy */
  int64_t m, n, k;
  int64_t ldx, ldw, ldr, ldy;
  int32_t y_dtype;         /* UOCR_DTYPE_F32 or UOCR_DTYPE_BF16 */
  int32_t reserved;        /* 0 */
} uocr_linear_w8a8_args;

/* y = x w^T * x_scales[m] * w_scales[n] (+ bias) (+ residual): the reference's
 * linear (src/backend/cuda/ops.h:14-17) on quantised operands, for one token
 * up to many. */
int uocr_linear_w8a8(const uocr_linear_w8a8_args* args, void* stream);

typedef struct uocr_grouped_w8a8_args {
  const int8_t* x;          /* [x_rows, k], pitch ldx */
  const float* x_scales;    /* [x_rows] */
  const int32_t* row_index; /* [rows]: output row r reads x's row row_index[r]; NULL: row r (x_rows == rows) */
  const int32_t* offsets;   /* [groups + 1], device: group g owns the output rows offsets[g] .. offsets[g + 1] - 1 */
  const int8_t* w;          /* [groups, n, k], row pitch ldw */
  const float* w_scales;    /* [groups, n] */
  const int8_t* w_up;       /* [groups, n, k], row pitch ldw, or NULL */
  const float* w_up_scales; /* [groups, n], with w_up */
  void* y;                  /* [rows, n], pitch ldy */
  int64_t rows, x_rows, groups, n, k;
  int64_t ldx, ldw, ldy;
  int32_t y_dtype;          /* UOCR_DTYPE_F32 or UOCR_DTYPE_BF16 */
  int32_t reserved;         /* 0 */
  void* workspace;          /* device memory for the call's duration, 16-byte aligned; NULL when none is needed */
  int64_t workspace_bytes;  /* at least what uocr_grouped_w8a8_workspace says */
} uocr_grouped_w8a8_args;

/* Bytes of workspace the call below needs with these sizes (row_index given,
 * many rows: the rows it names, copied together; else 0). Only the sizes and
 * whether row_index is NULL are looked at. */
int uocr_grouped_w8a8_workspace(const uocr_grouped_w8a8_args* args, int64_t* bytes);

/* Each group of rows with its own matrix: y[r] = x[row_index[r]] w[g]^T, scaled
 * as above; with w_up the gated form silu(x w[g]^T) * (x w_up[g]^T)
 * (src/model/feed_forward.cpp:50-64). Groups are an expert's tokens in expert
 * order, as ragged as they come, empty ones included; the group sizes stay on
 * the device. Rows outside offsets[0] .. offsets[groups] are left as they are.
 * An offset outside [0, rows], a group that ends before it starts, or a row
 * index outside [0, x_rows) is recorded in the device's error word
 * (uocr_ops_check): such a group is skipped, such a row is computed as zero. */
int uocr_grouped_linear_w8a8(const uocr_grouped_w8a8_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* UOCR_INT8_H */
