// Host interface of the operators for sequences that share a page
// (include/uocr_beam.h): the rotation of heads with the cache append, attention
// behind shared prefixes, the selection of beams and the reordering of their
// states. The launchers take arguments that the C ABI has checked.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "moe_common.cuh"
#include "../../include/uocr_beam.h"

namespace uocr_b200 {

cudaError_t launch_rotate_heads(const uocr_rotate_heads_args& a, ErrorWord* err, cudaStream_t stream);

size_t prefix_attention_bytes(const uocr_prefix_attention_args& a);
cudaError_t launch_prefix_attention(const uocr_prefix_attention_args& a, ErrorWord* err, cudaStream_t stream);

size_t beam_select_bytes(const uocr_beam_select_args& a);
cudaError_t launch_beam_select(const uocr_beam_select_args& a, cudaStream_t stream);

cudaError_t launch_reorder_states(const uocr_reorder_states_args& a, ErrorWord* err, cudaStream_t stream);

}  // namespace uocr_b200
