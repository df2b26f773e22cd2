// States of a group's beams brought into a new order in place
// (uocr_reorder_states): state[r] = state[parent[r]] for all r at once.
//
// A thread holds one column (up to 16 bytes at one place of a segment) of all
// the rows that another row is to become, then writes the rows that change: no
// second buffer, every source read once, every changed row written once, and
// no order of the rows matters, cycles among them included. Bound: memory: 24 layers
// of 32 rows of 0.5 MB take 62.9 us, 5.6 TB/s of reads and writes.
#include "beam.h"
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kThreads = 128;

struct Reorder {
  char* state;
  const int* parents;
  const int* counts;
  int64_t layer_stride, row_stride, segment_stride;
  int64_t units, unit_bytes;
  int64_t columns;  // of a segment
  int groups, beams, segments;
  ErrorWord* err;
};

template <typename Word, int kBeams>
__global__ void __launch_bounds__(kThreads) reorder_states_kernel(Reorder a, unsigned blocks_each) {
  __shared__ unsigned children[kBeams];  // bit r: row r becomes a copy of this one
  __shared__ int64_t held[kBeams];       // bytes of a segment
  pdl_wait();
  pdl_launch_dependents();
  // Blocks of a (layer, group, segment) follow one another.
  unsigned b = blockIdx.x;
  const unsigned part = b % blocks_each;
  b /= blocks_each;
  const int segment = b % a.segments;
  b /= a.segments;
  const int group = b % a.groups;
  const int64_t layer = b / a.groups;
  if (threadIdx.x < kBeams) children[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x < a.beams) {
    const int row = group * a.beams + threadIdx.x;
    const int parent = a.parents[row];
    const bool first = part == 0 && segment == 0 && layer == 0;
    if (parent < 0 || parent >= a.beams) {
      if (first) raise_error(a.err, kDevBadIndex, kSiteParent, row, parent);
    } else if (parent != static_cast<int>(threadIdx.x)) {
      atomicOr(&children[parent], 1u << threadIdx.x);
    }
    int64_t n = a.units;
    if (a.counts != nullptr) {
      const int c = a.counts[row];
      if ((c < 0 || c > a.units) && first) raise_error(a.err, kDevBadIndex, kSiteCount, row, c);
      n = min(static_cast<int64_t>(max(c, 0)), a.units);
    }
    held[threadIdx.x] = n * a.unit_bytes;
  }
  __syncthreads();
  const int64_t column = static_cast<int64_t>(part) * kThreads + threadIdx.x;
  const int64_t at = column * sizeof(Word);
  char* base = a.state + layer * a.layer_stride + static_cast<int64_t>(group) * a.beams * a.row_stride +
               segment * a.segment_stride + at;
  Word v[kBeams];
#pragma unroll
  for (int p = 0; p < kBeams; ++p)
    if (p < a.beams && children[p] != 0 && at < held[p]) v[p] = *reinterpret_cast<const Word*>(base + p * a.row_stride);
#pragma unroll
  for (int p = 0; p < kBeams; ++p) {
    if (p >= a.beams || at >= held[p]) continue;
    for (unsigned m = children[p]; m != 0; m &= m - 1)
      *reinterpret_cast<Word*>(base + (__ffs(m) - 1) * a.row_stride) = v[p];
  }
}

template <typename Word, int kBeams>
cudaError_t launch(const Reorder& r, int64_t layers, cudaStream_t stream) {
  const int64_t each = (r.columns + kThreads - 1) / kThreads;
  return launch_pdl(reorder_states_kernel<Word, kBeams>,
                    static_cast<unsigned>(each * r.segments * r.groups * layers), kThreads, 0, stream, r,
                    static_cast<unsigned>(each));
}

template <typename Word>
cudaError_t choose(Reorder r, int64_t layers, cudaStream_t stream) {
  r.columns = r.units * r.unit_bytes / static_cast<int64_t>(sizeof(Word));
  if (r.beams <= 4) return launch<Word, 4>(r, layers, stream);
  if (r.beams <= 8) return launch<Word, 8>(r, layers, stream);
  if (r.beams <= 16) return launch<Word, 16>(r, layers, stream);
  return launch<Word, 32>(r, layers, stream);
}

}  // namespace

cudaError_t launch_reorder_states(const uocr_reorder_states_args& a, ErrorWord* err, cudaStream_t stream) {
  Reorder r{};
  r.state = static_cast<char*>(a.state);
  r.parents = a.parents, r.counts = a.counts;
  r.layer_stride = a.layer_stride, r.row_stride = a.row_stride, r.segment_stride = a.segment_stride;
  r.units = a.units, r.unit_bytes = a.unit_bytes;
  r.groups = static_cast<int>(a.groups), r.beams = static_cast<int>(a.beams), r.segments = static_cast<int>(a.segments);
  r.err = err;
  // The widest word that every unit and address is a multiple of.
  const uint64_t all = reinterpret_cast<uintptr_t>(a.state) | static_cast<uint64_t>(a.unit_bytes) |
                       static_cast<uint64_t>(a.layers > 1 ? a.layer_stride : 0) | static_cast<uint64_t>(a.row_stride) |
                       static_cast<uint64_t>(a.segments > 1 ? a.segment_stride : 0);
  if (all % 16 == 0) return choose<uint4>(r, a.layers, stream);
  if (all % 4 == 0) return choose<uint32_t>(r, a.layers, stream);
  return choose<uint8_t>(r, a.layers, stream);
}

}  // namespace uocr_b200
