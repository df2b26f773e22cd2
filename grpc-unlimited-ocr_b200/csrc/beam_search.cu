// The small kernels between the operators of a beam search on the page decoder
// (uocr_decoder_beam_search): what a step needs stays on the device.
#include "beam.h"

namespace uocr_b200 {
namespace {

__global__ void beam_init_kernel(BeamState s, int prefix_len) {
  const int cells = s.beams * s.steps;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < cells; i += gridDim.x * blockDim.x) {
    s.table[i] = i / s.steps;  // a beam's keys are its own until it is reordered
    s.table[cells + i] = 0;
  }
  if (blockIdx.x != 0) return;
  for (int b = threadIdx.x; b < s.beams; b += blockDim.x) {
    s.scores[b] = 0.0f;
    s.finished[b] = 0;
  }
  if (threadIdx.x == 0) {
    *s.step = 0;
    *s.prefix_len = prefix_len;
  }
}

__global__ void beam_embed_kernel(BeamState s, const __nv_bfloat16* embed, float* x) {
  const int b = blockIdx.x, step = *s.step;
  const __nv_bfloat16* row = embed + static_cast<int64_t>(min(max(s.tokens[b], 0), s.vocab - 1)) * s.hidden;
  for (int i = threadIdx.x; i < s.hidden; i += blockDim.x)
    x[static_cast<int64_t>(b) * s.hidden + i] = __bfloat162float(row[i]);
  if (threadIdx.x == 0) {
    s.positions[b] = *s.prefix_len + step - 1;
    s.slots[b] = step - 1;
    s.lens[b] = step;
  }
}

__global__ void beam_record_kernel(BeamState s) {
  const int b = threadIdx.x, step = *s.step;
  if (b < s.beams && step < s.steps) {
    s.table[(s.beams + b) * s.steps + step] = s.tokens[b];
    s.scores[b] = s.new_scores[b];
    s.finished[b] = s.new_finished[b];
  }
  __syncthreads();
  if (b == 0) *s.step = step + 1;
}

__global__ void beam_finish_kernel(BeamState s, int* tokens, float* scores, int* lengths) {
  const int b = blockIdx.x;
  __shared__ int first;
  if (threadIdx.x == 0) first = s.steps - 1;
  __syncthreads();
  for (int t = threadIdx.x; t < s.steps; t += blockDim.x) {
    const int token = s.table[(s.beams + b) * s.steps + t];
    tokens[b * s.steps + t] = token;
    if (token == s.eos) atomicMin(&first, t);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    scores[b] = s.scores[b];
    if (lengths != nullptr) lengths[b] = first + 1;
  }
}

}  // namespace

cudaError_t launch_beam_init(const BeamState& s, int prefix_len, cudaStream_t stream) {
  beam_init_kernel<<<32, 256, 0, stream>>>(s, prefix_len);
  return cudaGetLastError();
}
cudaError_t launch_beam_embed(const BeamState& s, const __nv_bfloat16* embed, float* x, cudaStream_t stream) {
  beam_embed_kernel<<<s.beams, 256, 0, stream>>>(s, embed, x);
  return cudaGetLastError();
}
cudaError_t launch_beam_record(const BeamState& s, cudaStream_t stream) {
  beam_record_kernel<<<1, kDecodeMaxRows, 0, stream>>>(s);
  return cudaGetLastError();
}
cudaError_t launch_beam_finish(const BeamState& s, int* tokens, float* scores, int* lengths, cudaStream_t stream) {
  beam_finish_kernel<<<s.beams, 256, 0, stream>>>(s, tokens, scores, lengths);
  return cudaGetLastError();
}

}  // namespace uocr_b200
