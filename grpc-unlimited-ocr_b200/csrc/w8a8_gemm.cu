// W8A8 products on the tensor cores (include/uocr_int8.h): tcgen05.mma of
// signed 8-bit operands with int32 accumulators in TMEM, dense or grouped.
//
// The weights are the M operand and the tokens the N operand: a pair of SMs
// (cta_group::2) multiplies 256 output channels (128 in each SM) by up to 256
// tokens, N being the tile's own token count rounded up to 32. A ragged group
// so wastes at most 31 tokens' work, where a token tile of 256 rows would
// waste half of it, and a handful of tokens costs a narrow MMA. The gated form
// multiplies gate and up rows of the same channels by up to 128 tokens into
// two accumulators, so that a thread has both values of a channel.
//
// One persistent pair of blocks per two SMs, warp-specialised:
//   warp 0     producer: each CTA's 128 weight rows (one box; two when gated)
//              and its half of the token rows (boxes of 16 rows, a lane each,
//              or gather4 of four indexed rows a lane) per 128-byte slice of K;
//   warp 1     allocates TMEM; in the leader one lane issues the MMAs;
//   warps 4-11 epilogue: lane = channel, register = token, so the channel's
//              scale stays in a register and a token's row is stored 32
//              channels at a time, without staging.
#include <mutex>

#include "tc.cuh"
#include "tc_gemm.h"
#include "w8a8.h"

namespace uocr_b200 {
namespace {

constexpr int kMaxGroups = 512;
constexpr int kBM = 128;               // channels per CTA
constexpr int kBK = 128;               // bytes of K per stage (one swizzle atom)
constexpr int kMaxN = 256;             // tokens per tile (128 when gated)
constexpr int kRowBytes = kBK;
constexpr int kThreads = 384;
constexpr int kEpilogueWarps = 8;
constexpr int kTmemCols = 512;
constexpr int kBoxRows = 16;
constexpr int kBand = 8;               // token tiles of a band (decode_tile)

template <bool kGated>
struct Shape {
  static constexpr int kTokens = kGated ? kMaxN / 2 : kMaxN;
  static constexpr int kABytes = (kGated ? 2 : 1) * kBM * kRowBytes;
  static constexpr int kStageBytes = kABytes + kTokens / 2 * kRowBytes;
  static constexpr int kStages = kGated ? 5 : 6;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
};

struct Args {
  CUtensorMap x, x_wide, x_half, w, up;  // token boxes of 16 rows (gather: 1), 64, and a full tile's half
  W8a8 p;
  int tokens_per_tile;  // at most Shape::kTokens, a multiple of 32
  int c_tiles, k_blocks;
};

struct Shared {
  uint64_t full[6], empty[6];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drain;
  uint32_t tmem;
  int tile_start[kMaxGroups + 1];
  int first[kMaxGroups], count[kMaxGroups];
  alignas(16) float x_scale[2][kMaxN];
};

struct Tile {
  int g, row0, rows, c0;
};

__device__ __forceinline__ int round32(int v) { return (v + 31) & ~31; }

__device__ __forceinline__ Tile decode_tile(int t, const Shared& sh, int groups, const Args& a) {
  int lo = 0, hi = groups - 1;  // last g with tile_start[g] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sh.tile_start[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int local = t - sh.tile_start[lo], count = sh.count[lo];
  const int r_tiles = (count + a.tokens_per_tile - 1) / a.tokens_per_tile;
  const int per = round32((count + r_tiles - 1) / r_tiles);  // the group's tokens dealt evenly
  // Bands of kBand token tiles, token tile fastest: the pairs at work at a time share both operands in L2.
  const int band = local / (kBand * a.c_tiles), in_band = local - band * kBand * a.c_tiles;
  const int high = min(kBand, r_tiles - band * kBand);
  const int c = in_band / high;
  const int r = (band * kBand + in_band - c * high) * per;
  return Tile{lo, sh.first[lo] + r, min(per, count - r), c * 2 * kBM};
}

// silu(g) * u = g / (1 + exp(-g)) * u. The quotient to 2 ulp (__fdividef): an
// IEEE division branches, and 32 of them in a row keep a thread's 32 tokens
// from overlapping (the gated kernel's time at eight pages: 928 us with it).
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

template <bool kBf16>
__device__ __forceinline__ float load_as_f32(const void* base, int64_t i) {
  return kBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]) : static_cast<const float*>(base)[i];
}
template <bool kBf16>
__device__ __forceinline__ void store_f32(void* base, int64_t i, float v) {
  if (kBf16)
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(base)[i] = v;
}

template <bool kGated, bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    w8a8_gemm_kernel(const __grid_constant__ Args args) {
  using S = Shape<kGated>;
  extern __shared__ unsigned char dyn_raw[];
  __shared__ Shared sh;
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const W8a8& p = args.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int groups = static_cast<int>(p.groups);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], 2 * kEpilogueWarps);
    }
    mbar_init(&sh.drain, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
      const int g = g0 + lane;
      int tiles = 0;
      if (g < groups) {
        int first = 0;
        int64_t count = p.rows;
        if (p.starts != nullptr) {
          first = __ldg(p.starts + g);
          count = p.counts != nullptr ? __ldg(p.counts + g) : static_cast<int64_t>(__ldg(p.starts + g + 1)) - first;
          if (first < 0 || count < 0 || first + count > p.rows) {
            raise_error(p.err, kDevBadIndex, kSiteGroupRows, g, first);
            count = 0;
          }
        }
        sh.first[g] = first;
        sh.count[g] = static_cast<int>(count);
        tiles = static_cast<int>((count + args.tokens_per_tile - 1) / args.tokens_per_tile) * args.c_tiles;
      }
      int incl = tiles;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (g < groups) sh.tile_start[g] = carry + incl - tiles;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) sh.tile_start[groups] = carry;
  }
  if (warp == 1) tmem_alloc_pair(&sh.tmem, kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers exist before either is signalled from the other
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem;
  const int total = sh.tile_start[groups];
  const int step = gridDim.x / 2;

  if (warp == 0) {
    // ---- producer ----
    const bool gather = p.row_index != nullptr;
    // A tile's four gathered rows of this lane; rows past the tile or outside x read row 0 (never stored, or scaled
    // by zero).
    auto indices = [&](const Tile& tl, int (&idx)[4]) {
      const int half = round32(tl.rows) / 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = rank * half + 4 * lane + i;
        const int v = 4 * lane + i < half && j < tl.rows ? __ldg(p.row_index + tl.row0 + j) : 0;
        idx[i] = v < 0 || v >= p.x_rows ? 0 : v;
      }
    };
    int stage = 0;
    uint32_t phase = 0;
    int idx[4] = {0, 0, 0, 0};
    int t = blockIdx.x / 2;
    Tile tl{};
    if (t < total) {
      tl = decode_tile(t, sh, groups, args);
      if (gather) indices(tl, idx);
    }
    bool ok = true;
    while (t < total && ok) {
      // The next tile and its indices are fetched while this one's copies run.
      const int next_t = t + step;
      Tile next{};
      int next_idx[4] = {0, 0, 0, 0};
      if (next_t < total) {
        next = decode_tile(next_t, sh, groups, args);
        if (gather) indices(next, next_idx);
      }
      const int n = round32(tl.rows), half = n / 2;
      const int w_row = tl.g * static_cast<int>(p.n) + tl.c0 + rank * kBM;
      for (int kb = 0; kb < args.k_blocks; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[stage], phase ^ 1));  // the whole warp goes on or stops
        if (!ok) {
          raise_error(p.err, kDevWaitTimeout, 82, t, kb);
          break;
        }
        const uint32_t bar = pair_leader_addr(&sh.full[stage]);
        unsigned char* sa = smem + stage * S::kStageBytes;
        unsigned char* sb = sa + S::kABytes;
        if (lane == 0) {
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[stage], 2 * S::kABytes + n * kRowBytes);
          tma_load_2d_pair(sa, &args.w, kb * kBK, w_row, bar);
          if (kGated) tma_load_2d_pair(sa + kBM * kRowBytes, &args.up, kb * kBK, w_row, bar);
        }
        __syncwarp();
        if (gather) {
          if (4 * lane < half)
            tma_gather4_pair(sb + lane * 4 * kRowBytes, &args.x, kb * kBK, idx[0], idx[1], idx[2], idx[3], bar);
        } else if (half == S::kTokens / 2) {
          if (lane == 0) tma_load_2d_pair(sb, &args.x_half, kb * kBK, tl.row0 + rank * half, bar);
        } else {
          const int wide = half & ~63;  // rows in boxes of 64, the rest in boxes of 16
          if (lane * 64 < wide)
            tma_load_2d_pair(sb + lane * 64 * kRowBytes, &args.x_wide, kb * kBK, tl.row0 + rank * half + lane * 64, bar);
          const int r = wide + (lane - 16) * kBoxRows;
          if (lane >= 16 && r < half)
            tma_load_2d_pair(sb + r * kRowBytes, &args.x, kb * kBK, tl.row0 + rank * half + r, bar);
        }
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      t = next_t;
      tl = next;
#pragma unroll
      for (int i = 0; i < 4; ++i) idx[i] = next_idx[i];
    }
    if (!ok) {  // the copies in flight land before this CTA's shared memory is given up
      const uint64_t until = global_timer_ns() + 5000000ull;
      for (int i = 0; i < (1 << 20) && global_timer_ns() < until; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---- MMA issuer (for both CTAs) ----
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x / 2; t < total && ok; t += step, ++local) {
        const Tile tl = decode_tile(t, sh, groups, args);
        const uint32_t idesc = i8_idesc(2 * kBM, round32(tl.rows));
        const int acc = local & 1;
        if (!mbar_wait(&sh.acc_empty[acc], ((local >> 1) & 1) ^ 1)) {
          raise_error(p.err, kDevWaitTimeout, 83, t, 0);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kMaxN);
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!mbar_wait(&sh.full[stage], phase)) {
            raise_error(p.err, kDevWaitTimeout, 84, t, kb);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_addr(smem + stage * S::kStageBytes);
          const uint64_t ad = sw128_kmajor_desc(sa);
          const uint64_t ud = sw128_kmajor_desc(sa + kBM * kRowBytes);
          const uint64_t bd = sw128_kmajor_desc(sa + S::kABytes);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k) {  // 32 bytes of K per instruction: +2 in the address field
            umma_i8_pair(d, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
            if (kGated) umma_i8_pair(d + kMaxN / 2, ud + 2 * k, bd + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          umma_commit_pair(&sh.empty[stage]);
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) umma_commit_pair(&sh.acc_full[acc]);
      }
      umma_commit_pair(&sh.drain);
      if (!mbar_wait(&sh.drain, 0)) raise_error(p.err, kDevWaitTimeout, 85, 0, 0);
    }
  } else if (warp >= 4) {
    // ---- epilogue: TMEM lane quarter = warp % 4; the two warps of a quarter take every other 32 tokens ----
    const int quarter = warp & 3, odd = (warp - 4) >> 2;
    const int et = threadIdx.x - 128;
    int local = 0;
    bool ok = true;
    for (int t = blockIdx.x / 2; t < total; t += step, ++local) {
      const Tile tl = decode_tile(t, sh, groups, args);
      const int acc = local & 1;
      const int64_t c = tl.c0 + rank * kBM + quarter * 32 + lane;
      const bool c_ok = c < p.n;
      const float ws = c_ok ? __ldg(p.w_scales + tl.g * p.n + c) : 0.0f;
      const float us = kGated && c_ok ? __ldg(p.w_up_scales + tl.g * p.n + c) : 0.0f;
      const float bias = p.bias != nullptr && c_ok ? __ldg(p.bias + c) : 0.0f;
      if (et < tl.rows) {
        float s = 0.0f;
        int64_t r = tl.row0 + et;
        if (p.row_index != nullptr) {
          const int v = __ldg(p.row_index + r);
          if (v < 0 || v >= p.x_rows) {
            raise_error(p.err, kDevBadIndex, kSiteRowIndex, static_cast<int>(r), v);
            r = -1;
          } else {
            r = v;
          }
        }
        if (r >= 0) s = __ldg(p.x_scales + r);
        sh.x_scale[acc][et] = s;
      }
      named_bar_sync(1, kEpilogueWarps * 32);
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], (local >> 1) & 1));
        if (!ok) raise_error(p.err, kDevWaitTimeout, 86, t, 0);
      }
      if (!ok) continue;  // the warps that go on still meet this one at the barrier above
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kMaxN);
      auto release = [&] {  // this warp has read its last columns: the accumulator may be written again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(pair_leader_addr(&sh.acc_empty[acc]));
      };
      if (odd * 32 >= tl.rows) release();
      for (int j0 = odd * 32; j0 < tl.rows; j0 += 64) {
        int a[32], u[32];
        tmem_ld32_async(taddr + j0, a);
        if (kGated) tmem_ld32_async(taddr + kMaxN / 2 + j0, u);
        tmem_ld_wait(a);
        if (kGated) tmem_ld_wait(u);
        if (j0 + 64 >= tl.rows) release();
        const int nr = c_ok ? min(32, tl.rows - j0) : 0;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(&sh.x_scale[acc][j0 + i]);
          const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[i + e] = static_cast<float>(a[i + e]) * s[e] * ws;
            if (kGated) v[i + e] = silu_mul(v[i + e], static_cast<float>(u[i + e]) * s[e] * us);
          }
        }
        const int64_t row = tl.row0 + j0;
        if (!kGated) {
          if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += bias;
          }
          if (p.residual != nullptr) {
            float r[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = i < nr ? load_as_f32<kBf16>(p.residual, (row + i) * p.ldr + c) : 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += r[i];
          }
        }
        char* out = static_cast<char*>(p.y) + (row * p.ldy + c) * (kBf16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < nr) {
            store_f32<kBf16>(out, 0, v[i]);
            out += p.ldy * (kBf16 ? 2 : 4);
          }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // the pair's MMAs are complete: no operand, accumulator or barrier is in use any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  __syncthreads();
  cluster_barrier();
}

// Pairs that run at the same time on the current device (0: the kernel cannot run).
template <bool kGated, bool kBf16>
cudaError_t resident_pairs(int* pairs) {
  static std::mutex mu;
  static int known[kMaxDevices] = {};
  int dev = 0;
  cudaError_t st = cudaGetDevice(&dev);
  if (st != cudaSuccess) return st;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev] == 0) {
    const auto kernel = w8a8_gemm_kernel<kGated, kBf16>;
    st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kGated>::kSmem);
    if (st != cudaSuccess) return st;
    int sms = 0;
    if ((st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return st;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(sms / 2 * 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<kGated>::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if ((st = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg)) != cudaSuccess) return st;
    if (n <= 0) return cudaErrorNotSupported;
    known[dev] = n;
  }
  *pairs = known[dev];
  return cudaSuccess;
}

// Tokens per tile: as many as fit where there are tiles enough for the pairs.
// A narrower MMA costs less, down to 64 tokens, so where the tiles are few
// (one wave or a broken one) the width that ends first is taken.
int choose_tokens(int64_t rows, int64_t groups, int c_tiles, int pairs, int most) {
  if (groups > 1) {
    int bn = most;
    while (bn > 64 && (rows / bn + (groups < rows ? groups : rows) / 2) * c_tiles < pairs) bn /= 2;
    return bn;
  }
  int best = most;
  int64_t best_cost = INT64_MAX;
  for (int bn = most; bn >= 32; bn -= 32) {
    const int64_t r = (rows + bn - 1) / bn;
    const int64_t per = ((rows + r - 1) / r + 31) / 32 * 32;
    const int64_t cost = ((r * c_tiles + pairs - 1) / pairs) * ((per > 64 ? per : 64) + 16);
    if (cost < best_cost) {
      best_cost = cost;
      best = bn;
    }
  }
  return best;
}

template <bool kGated, bool kBf16>
cudaError_t launch(const W8a8& p, cudaStream_t stream) {
  int pairs = 0;
  cudaError_t st = resident_pairs<kGated, kBf16>(&pairs);
  if (st != cudaSuccess) return st;
  Args a{};
  const bool ok = make_int8_tmap(&a.x, p.x, p.x_rows, p.k, p.ldx, p.row_index != nullptr ? 1 : kBoxRows) &&
                  make_int8_tmap(&a.x_wide, p.x, p.x_rows, p.k, p.ldx, 64) &&
                  make_int8_tmap(&a.x_half, p.x, p.x_rows, p.k, p.ldx, Shape<kGated>::kTokens / 2) &&
                  make_int8_tmap(&a.w, p.w, p.groups * p.n, p.k, p.ldw, kBM) &&
                  (!kGated || make_int8_tmap(&a.up, p.w_up, p.groups * p.n, p.k, p.ldw, kBM));
  if (!ok) return cudaErrorInvalidValue;
  a.p = p;
  a.c_tiles = static_cast<int>((p.n + 2 * kBM - 1) / (2 * kBM));
  a.k_blocks = static_cast<int>((p.k + kBK - 1) / kBK);
  a.tokens_per_tile = choose_tokens(p.rows, p.groups, a.c_tiles, pairs, Shape<kGated>::kTokens);
  const int64_t most =
      (p.rows / a.tokens_per_tile + (p.groups < p.rows ? p.groups : p.rows)) * static_cast<int64_t>(a.c_tiles);
  const unsigned blocks = 2u * static_cast<unsigned>(most < pairs ? most : pairs);
  w8a8_gemm_kernel<kGated, kBf16><<<blocks, kThreads, Shape<kGated>::kSmem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_w8a8(const W8a8& p, cudaStream_t stream) {
  if (p.rows == 0 || p.n == 0) return cudaSuccess;
  if (p.w_up != nullptr) return p.y_bf16 ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
  return p.y_bf16 ? launch<false, true>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace uocr_b200
