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

// Whether the call's units of work are few enough to be counted.
bool prefix_attention_counts(const uocr_prefix_attention_args& a);
size_t prefix_attention_bytes(const uocr_prefix_attention_args& a);
cudaError_t launch_prefix_attention(const uocr_prefix_attention_args& a, ErrorWord* err, cudaStream_t stream);

size_t beam_select_bytes(const uocr_beam_select_args& a);
cudaError_t launch_beam_select(const uocr_beam_select_args& a, cudaStream_t stream);

cudaError_t launch_reorder_states(const uocr_reorder_states_args& a, ErrorWord* err, cudaStream_t stream);

// What a beam search keeps on the device between its steps (beam_search.cu).
struct BeamState {
  int beams, steps, vocab, hidden;
  int eos;
  int* table;        // [2, beams, steps]: the caches that a beam's keys lie in, then its tokens
  int* step;         // [1] tokens chosen so far
  int* prefix_len;   // [1]
  int* positions;    // [beams] of the tokens that a step consumes
  int* slots;        // [beams] their places in the beams' caches
  int* lens;         // [beams] keys of a beam, the new one among them
  int* tokens;       // [beams] the current tokens
  int* parents;      // [beams]
  int* finished;     // [beams]
  int* new_finished;
  float* scores;     // [beams]
  float* new_scores;
};
cudaError_t launch_beam_init(const BeamState& s, int prefix_len, cudaStream_t stream);
// x [beams, hidden] = the tokens' embedding rows; positions, slots and lens of the step.
cudaError_t launch_beam_embed(const BeamState& s, const __nv_bfloat16* embed, float* x, cudaStream_t stream);
// The selected beams become the current ones; their tokens are recorded.
cudaError_t launch_beam_record(const BeamState& s, cudaStream_t stream);
cudaError_t launch_beam_finish(const BeamState& s, int* tokens, float* scores, int* lengths, cudaStream_t stream);

}  // namespace uocr_b200
