// What the kernels of prefix_attention.cu and prefix_attention_tc.cu share: the
// call's view on the device, its partial results and the search for the rows a
// block works on.
#pragma once

#include <cuda_bf16.h>

#include "beam.h"
#include "ptx.cuh"

namespace uocr_b200 {

constexpr float kLog2e = 1.4426950408889634f;

// Partial results: for every (row, head) and slot a maximum and a sum in the
// log2 domain, and the unnormalised output. Slots 0 .. prefix_slots - 1 are the
// prefix's parts, the others the own keys'.
struct Attention {
  const __nv_bfloat16* q;
  const __nv_bfloat16* prefix_k;
  const __nv_bfloat16* prefix_v;
  const int* prefix_lens;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const int* lens;
  const int* ancestry;
  const int* row_offsets;
  __nv_bfloat16* out;
  float* lse;
  int64_t ldq, ldo, ld_ancestry;
  int64_t prefix_stride, prefix_head_stride, cache_stride, head_stride;
  int rows, sequences, prefixes, caches, heads, kv_heads, group;  // group: query heads per key/value head
  int per;                                                        // sequences per prefix
  int prefix_capacity, capacity;
  int prefix_slots, slots;
  bool split;  // tensor-core kernel: a block's two tiles are the same rows, for every other 128 keys
  unsigned tc_units;  // and the most units it can have
  float scale_log2;
  float* part_o;     // [rows, heads, slots, dim]
  float2* part_ml;   // [rows, heads, slots]
  ErrorWord* err;
};

// Rows [first, first + n) of sequence b; none where the offsets are not in order.
__device__ __forceinline__ int rows_of(const Attention& a, int b, int* first) {
  if (a.row_offsets == nullptr) {
    *first = b;
    return 1;
  }
  const int r0 = a.row_offsets[b], r1 = a.row_offsets[b + 1];
  *first = r0;
  if (r0 < 0 || r1 < r0 || r1 > a.rows) {
    raise_error(a.err, kDevBadIndex, kSiteRowOffsets, b, r0);
    return 0;
  }
  return r1 - r0;
}
// The same of the sequences behind prefix p.
__device__ __forceinline__ int prefix_rows_of(const Attention& a, int p, int* first) {
  if (a.row_offsets == nullptr) {
    *first = p * a.per;
    return a.per;
  }
  const int r0 = a.row_offsets[p * a.per], r1 = a.row_offsets[(p + 1) * a.per];
  *first = r0;
  if (r0 < 0 || r1 < r0 || r1 > a.rows) {
    raise_error(a.err, kDevBadIndex, kSiteRowOffsets, p * a.per, r0);
    return 0;
  }
  return r1 - r0;
}

// a + b, or the most that an unsigned holds. Rows that offsets out of order name many times over would otherwise make
// sums of units that have gone past it; where a sum is above what there can be, no units are worked on.
__device__ __forceinline__ unsigned add_saturated(unsigned a, unsigned b) {
  const unsigned s = a + b;
  return s < a ? ~0u : s;
}

__device__ __forceinline__ int prefix_len_of(const Attention& a, int p) {
  const int n = a.prefix_lens[p];
  if (n < 0 || n > a.prefix_capacity) raise_error(a.err, kDevBadIndex, kSiteLength, -1 - p, n);
  return min(max(n, 0), a.prefix_capacity);
}
__device__ __forceinline__ int len_of(const Attention& a, int b) {
  const int n = a.lens[b];
  if (n < 0 || n > a.capacity) raise_error(a.err, kDevBadIndex, kSiteLength, b, n);
  return min(max(n, 0), a.capacity);
}

// 2^x to 2 ulp; 2^-inf = 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(h);
}

// Rows (a row and a query head each) of a tile of the tensor-core kernel; a block takes two.
constexpr int kAttentionTcRows = 128;
// The prefixes' parts of many rows by tcgen05 (prefix_attention_tc.cu): `blocks`
// resident blocks; at least three slots, six and an even number to split; a scale that is a normal number above 0.
cudaError_t launch_attention_tc(const Attention& a, int dim, unsigned blocks, cudaStream_t stream);

}  // namespace uocr_b200
