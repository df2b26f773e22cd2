// W8A8 products of a few rows (include/uocr_int8.h): the weights of a group are
// streamed once for every kTiles * 8 of its rows (grouped and gated products: 8).
//
// A warp takes 16 weight rows of one group (gate and up rows when gated) and
// all of K or a part of it, with mma.sync m16n8k32 on signed bytes: A = 16
// weight rows, B = 8 tokens. The order of K does not matter to an integer sum,
// so a lane loads 16 consecutive bytes of a weight row and of a token row and
// feeds them to two MMAs as they are. The int32 partials of the kSplit warps
// that share rows meet in shared memory, where the scales and the epilogue
// follow.
//
// Bound by the weights' bytes where they are many, else by the latency of one
// pass: start, offsets, row indices, loads, one exchange, store. K is split
// over as many warps (up to 8) as the device holds beside each other (choose).
#include "ptx.cuh"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRows = 16;    // weight rows of a warp
constexpr int kStep = 64;    // bytes of K a warp takes at a time

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once: past L1.
__device__ __forceinline__ uint4 load_weights(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The first `bytes` of 16, the others zero.
__device__ __forceinline__ uint4 keep_bytes(uint4 v, int64_t bytes) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t left = bytes - 4 * i;
    if (left < 4) w[i] = left > 0 ? w[i] & ((1u << (8 * left)) - 1u) : 0u;
  }
  return v;
}

// kTiles: tiles of 8 tokens a warp takes at a time. kSplit: warps that share
// 16 weight rows. T: y's type. blocks: (groups that have rows) x n_blocks.
// The bounds on registers cost up to 76 bytes of spills (kSplit 4, and 8 when
// gated) for a block more on each SM. In us as it is / with one block fewer,
// spilling nothing: 1 row by 16384 x 2048 8.2 / 10.2, by 102400 x 2048 36.8 / 39.8;
// 6 rows of 64 gated groups of 1024 x 2048 7.9 / 9.8, 18 rows 15.2 / 18.2; but
// 1 row by 12000 x 2048 7.4 / 5.5, 24 rows of 12 such groups 13.2 / 11.8.
template <bool kGated, int kTiles, int kSplit, typename T>
__global__ void __launch_bounds__(kThreads, kSplit == 8 ? (kGated ? 3 : 2) : 4)
    w8a8_rows_kernel(const W8a8 p, int n_blocks) {
  constexpr int kMats = kGated ? 2 : 1;
  constexpr int kDeep = (kSplit == 8 && kTiles < 4 ? 4 : 2) / kMats;  // steps in flight (as many as registers hold)
  __shared__ int part[kWarps][kMats * kTiles][32][4];
  __shared__ int s_first, s_count, s_group, s_has[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, tq = lane & 3;
  const int sub = warp / kSplit, split = warp % kSplit;
  pdl_wait();
  pdl_launch_dependents();

  // A block's group is the one its place among the groups that have rows names.
  const int place = blockIdx.x / n_blocks;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x % n_blocks) * (kWarps / kSplit) + sub) * kRows;
  int64_t g = 0;
  int first = 0, count = static_cast<int>(p.rows);
  if (p.starts != nullptr) {
    if (threadIdx.x == 0) s_group = -1;
    int before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += kThreads) {
      const int mine = g0 + threadIdx.x;
      int f = 0;
      int64_t c = 0;
      if (mine < p.groups) {
        f = p.starts[mine];
        c = p.counts != nullptr ? p.counts[mine] : static_cast<int64_t>(p.starts[mine + 1]) - f;
        if (f < 0 || c < 0 || f + c > p.rows) {
          if (blockIdx.x == 0) raise_error(p.err, kDevBadIndex, kSiteGroupRows, mine, f);
          c = 0;
        }
      }
      const unsigned has = __ballot_sync(0xffffffffu, c > 0);
      if (lane == 0) s_has[warp] = __popc(has);
      __syncthreads();
      int nth = before + __popc(has & ((1u << lane) - 1u));
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        nth += w < warp ? s_has[w] : 0;
        before += s_has[w];
      }
      if (c > 0 && nth == place) {
        s_group = mine;
        s_first = f;
        s_count = static_cast<int>(c);
      }
      __syncthreads();
    }
    g = s_group;
    if (g < 0) return;
    first = s_first;
    count = s_count;
  }

  const bool lo_ok = n0 + gr < p.n, hi_ok = n0 + gr + 8 < p.n;
  const int8_t* w_lo[kMats];
#pragma unroll
  for (int m = 0; m < kMats; ++m) w_lo[m] = (m == 0 ? p.w : p.w_up) + (g * p.n + n0 + gr) * p.ldw + tq * 16;
  const int64_t to_hi = 8 * p.ldw;
  const int steps = static_cast<int>((p.k + kStep - 1) / kStep);
  const int share = (steps + kSplit - 1) / kSplit;  // consecutive steps of this warp
  const int s0 = split * share, s1 = min(steps, s0 + share);
  const uint4 zero = make_uint4(0, 0, 0, 0);

  for (int r0 = 0; r0 < count; r0 += kTiles * 8) {
    uint4 a[kMats][2][kDeep];
    auto load_a = [&](int s) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int64_t kb = static_cast<int64_t>(s + u) * kStep;
        const bool in = s + u < s1 && kb + tq * 16 < p.k;
#pragma unroll
        for (int m = 0; m < kMats; ++m) {
          a[m][0][u] = in && lo_ok ? load_weights(w_lo[m] + kb) : zero;
          a[m][1][u] = in && hi_ok ? load_weights(w_lo[m] + to_hi + kb) : zero;
        }
      }
    };
    load_a(s0);  // before the row indices are waited for
    const int8_t* xr[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int r = r0 + 8 * i + gr;
      int64_t src = -1;
      if (r < count) {
        src = first + r;
        if (p.row_index != nullptr) {
          src = p.row_index[src];
          if (src >= p.x_rows) src = -1;  // reported below
        }
      }
      xr[i] = src < 0 ? nullptr : p.x + src * p.ldx + tq * 16;
    }
    // Output e: channel n0 + e % 16 of token e / 16; in an MMA's result, thread
    // 4 (channel % 8) + token % 8 / 2 holds it at [channel / 8][token % 2].
    // Where a thread has one output, its operands are loaded before the sums are there.
    constexpr int kOuts = (kRows * 8 * kTiles + kSplit * 32 - 1) / (kSplit * 32);
    struct Operands {
      bool in;
      float x, w, up, bias, residual;
    };
    auto operands = [&](int it) {
      Operands o{};
      const int e = (it * kSplit + split) * 32 + lane, tok = e / kRows;
      const int64_t c = n0 + e % kRows;
      o.in = tok < 8 * kTiles && r0 + tok < count && c < p.n;
      if (!o.in) return o;
      const int64_t row = static_cast<int64_t>(first) + r0 + tok;
      const int64_t src = p.row_index != nullptr ? p.row_index[row] : row;
      const bool has = src >= 0 && src < p.x_rows;
      if (!has) raise_error(p.err, kDevBadIndex, kSiteRowIndex, static_cast<int>(row), static_cast<int>(src));
      o.x = has ? p.x_scales[src] : 0.0f;
      o.w = p.w_scales[g * p.n + c];
      if (kGated) {
        o.up = p.w_up_scales[g * p.n + c];
      } else {
        if (p.bias != nullptr) o.bias = p.bias[c];
        if (p.residual != nullptr) o.residual = to_f32(static_cast<const T*>(p.residual)[row * p.ldr + c]);
      }
      return o;
    };
    Operands ahead{};
    if (kOuts == 1) ahead = operands(0);
    int acc[kMats][kTiles][4] = {};
    for (int s = s0; s < s1; s += kDeep) {
      uint4 b[kTiles][kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int64_t kb = static_cast<int64_t>(s + u) * kStep, left = p.k - kb - tq * 16;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          b[i][u] = s + u < s1 && left > 0 && xr[i] != nullptr ? *reinterpret_cast<const uint4*>(xr[i] + kb) : zero;
          if (left < 16) b[i][u] = keep_bytes(b[i][u], left);
        }
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u)
#pragma unroll
        for (int m = 0; m < kMats; ++m)
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            mma_s8(acc[m][i], a[m][0][u].x, a[m][1][u].x, a[m][0][u].y, a[m][1][u].y, b[i][u].x, b[i][u].y);
            mma_s8(acc[m][i], a[m][0][u].z, a[m][1][u].z, a[m][0][u].w, a[m][1][u].w, b[i][u].z, b[i][u].w);
          }
      if (s + kDeep < s1) load_a(s + kDeep);
    }
    // The warps of these rows meet: the partials are there, and those of the tokens before have been read.
    auto meet = [&] {
      if (kSplit == 1)
        __syncwarp();
      else
        named_bar_sync(1 + sub, kSplit * 32);
    };
    if (r0 > 0) meet();
#pragma unroll
    for (int m = 0; m < kMats; ++m)
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        *reinterpret_cast<int4*>(part[warp][m * kTiles + i][lane]) =
            make_int4(acc[m][i][0], acc[m][i][1], acc[m][i][2], acc[m][i][3]);
    meet();
#pragma unroll
    for (int it = 0; it < kOuts; ++it) {
      const Operands o = kOuts == 1 ? ahead : operands(it);
      if (!o.in) continue;
      const int e = (it * kSplit + split) * 32 + lane, ch = e % kRows, tok = e / kRows;
      const int tl = tok / 8, owner = (ch & 7) * 4 + (tok & 7) / 2, reg = (ch >> 3) * 2 + (tok & 1);
      int sum = 0, sum_up = 0;
#pragma unroll
      for (int w = 0; w < kSplit; ++w) {
        sum += part[sub * kSplit + w][tl][owner][reg];
        if (kGated) sum_up += part[sub * kSplit + w][kTiles + tl][owner][reg];
      }
      float v = __fmul_rn(static_cast<float>(sum) * o.x, o.w);  // not fused with a sum: the bits of w8a8_gemm.cu
      if (kGated)
        v = silu_mul(v, static_cast<float>(sum_up) * o.x * o.up);
      else
        v = v + o.bias + o.residual;
      put(static_cast<T*>(p.y) + (static_cast<int64_t>(first) + r0 + tok) * p.ldy + n0 + ch, v);
    }
  }
}

template <bool kGated, int kTiles, int kSplit, typename T>
cudaError_t launch(const W8a8& p, int64_t places, cudaStream_t stream) {
  constexpr int kBlockRows = kWarps / kSplit * kRows;
  const int64_t n_blocks = (p.n + kBlockRows - 1) / kBlockRows;
  return launch_pdl(w8a8_rows_kernel<kGated, kTiles, kSplit, T>, static_cast<unsigned>(places * n_blocks), kThreads, 0,
                    stream, p, static_cast<int>(n_blocks));
}

template <bool kGated, typename T>
cudaError_t choose(const W8a8& p, cudaStream_t stream) {
  // Groups that can have rows, and the warps that take all of K.
  const int64_t places = p.starts == nullptr ? 1 : p.groups < p.rows ? p.groups : p.rows;
  const int64_t warps = places * ((p.n + kRows - 1) / kRows);
  // Groups mostly have a row or two each; a dense product's rows are taken in one
  // pass (16 by 2048 x 2048 4.3 us, in passes of 8 5.0; by 8192 x 2048 8.3 and
  // 10.9; 24 by 2048 x 1024 3.9, in passes of 16 5.6).
  if constexpr (!kGated) {
    if (p.rows > 16 && p.starts == nullptr) return launch<kGated, 4, 8, T>(p, places, stream);
    if (p.rows > 8 && p.starts == nullptr) return launch<kGated, 2, 8, T>(p, places, stream);
  }
  // Measured in us by 8, 4 and 2 warps for 16 rows' K: 1 row by 2048 x 2048 2.9,
  // 4.9, 7.0; 8192 x 2048 5.7, 5.9, 8.4; 12000 x 2048 8.3, 7.7, 9.7; 16384 x 2048
  // 10.7, 8.3, 10.5; 20000 x 2048 12.2, 12.5, 11.4; 102400 x 2048 46, 38, 36; 96
  // rows of 64 groups of 2048 x 1024 58, 28, 23. Gated (twice the loads a warp)
  // of 64 groups of 2 x 1024 x 2048: 6 rows 7.7, 9.8, 14.0; 18 rows 17.4, 15.1,
  // 18.5; 24 rows 20.0, 19.5, 21.1; 30 rows 23.4, 22.9, 22.2.
  if (warps <= 512) return launch<kGated, 1, 8, T>(p, places, stream);
  if (warps <= (kGated ? 1536 : 1024)) return launch<kGated, 1, 4, T>(p, places, stream);
  return launch<kGated, 1, 2, T>(p, places, stream);
}

}  // namespace

cudaError_t launch_w8a8_rows(const W8a8& p, cudaStream_t stream) {
  if (p.w_up != nullptr) return p.y_bf16 ? choose<true, __nv_bfloat16>(p, stream) : choose<true, float>(p, stream);
  return p.y_bf16 ? choose<false, __nv_bfloat16>(p, stream) : choose<false, float>(p, stream);
}

}  // namespace uocr_b200
