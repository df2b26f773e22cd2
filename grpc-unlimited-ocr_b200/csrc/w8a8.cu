// W8A8 products (include/uocr_int8.h): int8 rows times int8 weight rows with
// int32 sums, dense or grouped by expert.
//
// A block computes 64 rows x 64 columns of one group; 64-byte slices of both
// operands pass through shared memory and four products at a time are added
// by dp4a.
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kTile = 64, kThreads = 256, kSlice = 64;

struct Group {
  int first, count;
};

// Group g's rows; a bad extent is recorded and empty.
__device__ __forceinline__ Group group_rows(const W8a8& p, int g) {
  if (p.starts == nullptr) return Group{0, static_cast<int>(p.rows)};
  const int s = __ldg(p.starts + g);
  const int64_t c = p.counts != nullptr ? __ldg(p.counts + g) : static_cast<int64_t>(__ldg(p.starts + g + 1)) - s;
  if (s < 0 || c < 0 || s + c > p.rows) {
    raise_error(p.err, kDevBadIndex, kSiteGroupRows, g, s);
    return Group{0, 0};
  }
  return Group{s, static_cast<int>(c)};
}

__device__ __forceinline__ float load_y(const W8a8& p, const void* base, int64_t i) {
  return p.y_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]) : static_cast<const float*>(base)[i];
}

__global__ void __launch_bounds__(kThreads) w8a8_kernel(W8a8 p, int n_tiles) {
  __shared__ __align__(16) int xs[kTile][kSlice / 4 + 1], ws[kTile][kSlice / 4 + 1], us[kTile][kSlice / 4 + 1];
  __shared__ int s_group, s_tile;
  if (threadIdx.x == 0) {
    int t = blockIdx.x / n_tiles, g = 0;
    for (; g < p.groups; ++g) {
      const int tiles = (group_rows(p, g).count + kTile - 1) / kTile;
      if (t < tiles) break;
      t -= tiles;
    }
    s_group = g;
    s_tile = t;
  }
  __syncthreads();
  const int g = s_group;
  if (g >= p.groups) return;
  const Group rows = group_rows(p, g);
  const int r0 = rows.first + s_tile * kTile, nr = min(kTile, rows.count - s_tile * kTile);
  const int64_t c0 = static_cast<int64_t>(blockIdx.x % n_tiles) * kTile;
  const bool gated = p.w_up != nullptr;
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  int acc[4][4] = {}, acu[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kSlice) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * kSlice; i += kThreads) {
      const int r = i / kSlice, c = i % kSlice;
      const bool in_k = k0 + c < p.k;
      int8_t xv = 0, wv = 0, uv = 0;
      if (r < nr && in_k) {
        int64_t src = r0 + r;
        if (p.row_index != nullptr) {
          src = p.row_index[src];
          if (src < 0 || src >= p.x_rows) {
            raise_error(p.err, kDevBadIndex, kSiteRowIndex, r0 + r, static_cast<int>(src));
            src = -1;
          }
        }
        if (src >= 0) xv = p.x[src * p.ldx + k0 + c];
      }
      if (c0 + r < p.n && in_k) {
        wv = p.w[(g * p.n + c0 + r) * p.ldw + k0 + c];
        if (gated) uv = p.w_up[(g * p.n + c0 + r) * p.ldw + k0 + c];
      }
      reinterpret_cast<int8_t*>(xs[r])[c] = xv;
      reinterpret_cast<int8_t*>(ws[r])[c] = wv;
      reinterpret_cast<int8_t*>(us[r])[c] = uv;
    }
    __syncthreads();
    for (int c = 0; c < kSlice / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __dp4a(xs[tr + 16 * i][c], ws[tc + 16 * j][c], acc[i][j]);
          acu[i][j] = __dp4a(xs[tr + 16 * i][c], us[tc + 16 * j][c], acu[i][j]);
        }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = tr + 16 * i;
      const int64_t c = c0 + tc + 16 * j;
      if (r >= nr || c >= p.n) continue;
      const int64_t row = r0 + r;
      int64_t src = p.row_index != nullptr ? p.row_index[row] : row;
      const float sx = src >= 0 && src < p.x_rows ? p.x_scales[src] : 0.0f;
      float v = static_cast<float>(acc[i][j]) * sx * p.w_scales[g * p.n + c];
      if (gated) v = swiglu(v, static_cast<float>(acu[i][j]) * sx * p.w_up_scales[g * p.n + c]);
      if (p.bias != nullptr) v += p.bias[c];
      if (p.residual != nullptr) v += load_y(p, p.residual, row * p.ldr + c);
      if (p.y_bf16)
        static_cast<__nv_bfloat16*>(p.y)[row * p.ldy + c] = __float2bfloat16_rn(v);
      else
        static_cast<float*>(p.y)[row * p.ldy + c] = v;
    }
}

}  // namespace

cudaError_t launch_w8a8(const W8a8& p, cudaStream_t stream) {
  if (p.rows == 0 || p.n == 0) return cudaSuccess;
  const int64_t n_tiles = (p.n + kTile - 1) / kTile;
  const int64_t m_tiles = p.starts == nullptr ? (p.rows + kTile - 1) / kTile
                                              : p.rows / kTile + (p.groups < p.rows ? p.groups : p.rows);
  w8a8_kernel<<<static_cast<unsigned>(n_tiles * m_tiles), kThreads, 0, stream>>>(p, static_cast<int>(n_tiles));
  return cudaGetLastError();
}

}  // namespace uocr_b200
