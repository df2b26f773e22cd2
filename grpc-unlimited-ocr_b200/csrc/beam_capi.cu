// C ABI of the operators for sequences that share a page (include/uocr_beam.h):
// argument checks and launches. Host code only; the kernels are in
// rotate_heads.cu, prefix_attention.cu, beam_select.cu and reorder_states.cu,
// the beam search beside the page decoder in decoder_capi.cu.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "beam.h"
#include "moe_kernels.h"

using namespace uocr_b200;

namespace {

constexpr int64_t kMaxCount = 1 << 30;  // rows, sequences, keys and grids are 32-bit in the kernels
constexpr int64_t kMaxVocab = 1 << 20;

int bad(const char* op, const char* what) {
  return set_last_error(UOCR_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}
int unsupported(const char* op, const char* what) {
  return set_last_error(UOCR_ERR_UNSUPPORTED, std::string(op) + ": " + what);
}
int done(const char* op, cudaError_t st) {
  if (st == cudaSuccess) return UOCR_OK;
  return set_last_error(st == cudaErrorMemoryAllocation ? UOCR_ERR_OUT_OF_MEMORY : UOCR_ERR_CUDA,
                        std::string(op) + ": " + cudaGetErrorString(st));
}

bool in(int64_t v, int64_t lo, int64_t hi) { return v >= lo && v <= hi; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
// Rows of a bf16 cache start at 16 bytes.
bool cache_ok(const void* p, int64_t stride, int64_t head_stride) {
  return aligned(p, 16) && stride % 8 == 0 && head_stride % 8 == 0 && stride >= 0 && head_stride >= 0;
}
// Whether the pieces of `extent` at a dimension's multiples of a stride, of every dimension, lie apart as views of memory
// do: each stride is at least what the dimensions of smaller strides span.
struct Dim {
  int64_t count, stride;
};
bool apart(int64_t extent, std::initializer_list<Dim> list) {
  Dim dims[4];
  size_t n = 0;
  for (const Dim& d : list)
    if (d.count > 1) dims[n++] = d;
  std::sort(dims, dims + n, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  double span = static_cast<double>(extent);  // counts and strides of any size
  for (size_t i = 0; i < n; ++i) {
    if (static_cast<double>(dims[i].stride) < span) return false;
    span += static_cast<double>(dims[i].stride) * static_cast<double>(dims[i].count - 1);
  }
  return true;
}
// a * b * ... stays a sum of bytes that int64_t holds.
bool product_fits(std::initializer_list<int64_t> v) {
  double p = 1.0;
  for (int64_t x : v) p *= static_cast<double>(x);
  return p < 4.0e18;
}

int check_attention_sizes(const char* op, const uocr_prefix_attention_args* a) {
  if (!in(a->rows, 0, kMaxCount) || !in(a->sequences, 0, kMaxCount) || !in(a->prefixes, 1, kMaxCount) ||
      !in(a->heads, 1, 1 << 16) || !in(a->kv_heads, 1, 1 << 16) || !in(a->prefix_capacity, 0, kMaxCount) ||
      !in(a->capacity, 0, kMaxCount) || !in(a->caches, 0, kMaxCount))
    return bad(op, "bad shape");
  if (a->head_dim != 64 && a->head_dim != 128) return unsupported(op, "head_dim must be 64 or 128");
  if (a->heads % a->kv_heads != 0) return bad(op, "heads must be a multiple of kv_heads");
  if (a->sequences % a->prefixes != 0) return bad(op, "sequences must be a multiple of prefixes");
  if (a->row_offsets == nullptr && a->rows != a->sequences)
    return bad(op, "without row_offsets there is one row per sequence");
  if (a->rows * a->heads > kMaxCount) return unsupported(op, "rows * heads above 2^30");
  if (a->reserved != 0) return bad(op, "reserved must be 0");
  if (!prefix_attention_counts(*a)) return unsupported(op, "rows * heads * keys too large");
  return UOCR_OK;
}

int check_select_sizes(const char* op, const uocr_beam_select_args* a) {
  if (!in(a->batch, 0, kMaxCount) || !in(a->vocab, 1, kMaxCount)) return bad(op, "bad shape");
  if (!in(a->beams, 1, UOCR_BEAM_MAX) || !in(a->select, 1, UOCR_BEAM_MAX))
    return bad(op, "beams and select must be 1 .. 32");
  if (a->vocab > kMaxVocab) return unsupported(op, "vocab above 2^20");
  // grid: at most ceil(vocab / 4096) blocks a row
  if (a->batch * a->beams * ((a->vocab + 4095) / 4096) > kMaxCount) return unsupported(op, "batch too large");
  return UOCR_OK;
}

}  // namespace

extern "C" {

int uocr_rope_frequencies(int64_t rotary_dim, double theta, int32_t scaling, double factor, int64_t original,
                          float* inv_freq, float* magnitude) {
  const char* op = "rope_frequencies";
  if (!in(rotary_dim, 2, 1 << 16) || rotary_dim % 2 != 0) return bad(op, "rotary_dim must be even and positive");
  if (!(theta > 1.0) || !std::isfinite(theta)) return bad(op, "theta must be above 1");
  if (!in(scaling, UOCR_ROPE_PLAIN, UOCR_ROPE_YARN)) return bad(op, "unknown scaling");
  if (!(factor >= 1.0) || !std::isfinite(factor)) return bad(op, "factor must be at least 1");
  if (inv_freq == nullptr) return bad(op, "null pointer");
  if (scaling == UOCR_ROPE_YARN && original <= 0) return bad(op, "yarn needs the original positions");
  if (scaling == UOCR_ROPE_NTK && rotary_dim < 4) return bad(op, "ntk needs two pairs");
  const double d = static_cast<double>(rotary_dim), two_pi = 6.28318530717958647692;
  if (scaling == UOCR_ROPE_NTK) theta *= std::pow(factor, d / (d - 2.0));
  // The pair that makes `turns` turns within the original positions.
  auto pair_of = [&](double turns) {
    return d * std::log(static_cast<double>(original) / (turns * two_pi)) / (2.0 * std::log(theta));
  };
  double low = 0.0, high = 0.0;
  if (scaling == UOCR_ROPE_YARN) {
    low = std::max(std::floor(pair_of(32.0)), 0.0);
    high = std::min(std::ceil(pair_of(1.0)), d - 1.0);
    if (high <= low) high = low + 0.001;
  }
  for (int64_t i = 0; i < rotary_dim / 2; ++i) {
    double f = 1.0 / std::pow(theta, 2.0 * static_cast<double>(i) / d);
    if (scaling == UOCR_ROPE_LINEAR) f /= factor;
    if (scaling == UOCR_ROPE_YARN) {
      const double ramp = std::min(std::max((static_cast<double>(i) - low) / (high - low), 0.0), 1.0);
      f = f * (1.0 - ramp) + f / factor * ramp;
    }
    inv_freq[i] = static_cast<float>(f);
  }
  if (magnitude != nullptr)
    *magnitude = scaling == UOCR_ROPE_YARN ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
  return UOCR_OK;
}

int uocr_rotate_heads(const uocr_rotate_heads_args* a, void* stream) {
  const char* op = "rotate_heads";
  if (a == nullptr) return bad(op, "null arguments");
  if (!in(a->rows, 0, kMaxCount) || !in(a->q_heads, 0, 1 << 16) || !in(a->kv_heads, 0, 1 << 16))
    return bad(op, "bad shape");
  if (!in(a->head_dim, 8, 256) || a->head_dim % 8 != 0)
    return unsupported(op, "head_dim must be a multiple of 8 up to 256");
  if (!in(a->rotary_dim, 0, a->head_dim) || a->rotary_dim % 8 != 0)
    return unsupported(op, "rotary_dim must be a multiple of 8 up to head_dim");
  if (a->dtype != UOCR_DTYPE_F32 && a->dtype != UOCR_DTYPE_BF16) return bad(op, "q, k and v must be f32 or bf16");
  if (a->interleaved != 0 && a->interleaved != 1) return bad(op, "interleaved must be 0 or 1");
  if (a->rows == 0 || a->q_heads + a->kv_heads == 0) return UOCR_OK;
  if (a->positions == nullptr || (a->rotary_dim > 0 && a->inv_freq == nullptr)) return bad(op, "null pointer");
  const size_t eb = a->dtype == UOCR_DTYPE_F32 ? 4 : 2;
  if (a->q_heads > 0) {
    if (a->q == nullptr || a->q_out == nullptr) return bad(op, "null pointer");
    if (a->ldq < a->q_heads * a->head_dim || a->ldqo < a->q_heads * a->head_dim)
      return bad(op, "a pitch is smaller than its row");
    if (!aligned(a->q, eb) || !aligned(a->q_out, 2)) return bad(op, "q or q_out is misaligned");
    if (a->q == a->q_out && (a->dtype != UOCR_DTYPE_BF16 || a->ldq != a->ldqo))
      return bad(op, "q_out in q's place is bf16 with q's pitch");
  }
  if (a->kv_heads > 0) {
    if (a->k == nullptr || a->v == nullptr || a->k_cache == nullptr || a->v_cache == nullptr)
      return bad(op, "null pointer");
    if (a->ldk < a->kv_heads * a->head_dim || a->ldv < a->kv_heads * a->head_dim)
      return bad(op, "a pitch is smaller than its row");
    if (!aligned(a->k, eb) || !aligned(a->v, eb)) return bad(op, "k or v is misaligned");
    if (!in(a->caches, 1, kMaxCount) || !in(a->capacity, 1, kMaxCount)) return bad(op, "bad shape");
    if (!cache_ok(a->k_cache, a->cache_stride, a->head_stride) || !cache_ok(a->v_cache, a->cache_stride, a->head_stride))
      return bad(op, "the caches' bases and strides must be multiples of 16 bytes");
    if (!apart(a->capacity * a->head_dim, {{a->kv_heads, a->head_stride}, {a->caches, a->cache_stride}}))
      return bad(op, "the caches or their heads overlap");
  }
  ErrorWord* err = nullptr;
  const cudaError_t st = ops_error_word(&err);
  return done(op, st != cudaSuccess ? st : launch_rotate_heads(*a, err, static_cast<cudaStream_t>(stream)));
}

int uocr_prefix_attention_workspace(const uocr_prefix_attention_args* a, int64_t* bytes) {
  const char* op = "prefix_attention_workspace";
  if (a == nullptr || bytes == nullptr) return bad(op, "null arguments");
  const int rc = check_attention_sizes(op, a);
  if (rc != UOCR_OK) return rc;
  *bytes = a->rows == 0 || a->sequences == 0 ? 0 : static_cast<int64_t>(prefix_attention_bytes(*a));
  return UOCR_OK;
}

int uocr_prefix_attention(const uocr_prefix_attention_args* a, void* stream) {
  const char* op = "prefix_attention";
  if (a == nullptr) return bad(op, "null arguments");
  const int rc = check_attention_sizes(op, a);
  if (rc != UOCR_OK || a->rows == 0 || a->sequences == 0) return rc;
  if (a->q == nullptr || a->out == nullptr || a->prefix_lens == nullptr || a->lens == nullptr)
    return bad(op, "null pointer");
  if (a->ldq < a->heads * a->head_dim || a->ldo < a->heads * a->head_dim)
    return bad(op, "a pitch is smaller than its row");
  if (!aligned(a->q, 16) || a->ldq % 8 != 0) return bad(op, "q's base and pitch must be multiples of 16 bytes");
  if (!aligned(a->out, 16) || a->ldo % 8 != 0) return bad(op, "out's base and pitch must be multiples of 16 bytes");
  if (!std::isfinite(a->scale)) return bad(op, "scale must be finite");
  if (a->prefix_capacity > 0) {
    if (a->prefix_k == nullptr || a->prefix_v == nullptr) return bad(op, "null pointer");
    if (!cache_ok(a->prefix_k, a->prefix_stride, a->prefix_head_stride) ||
        !cache_ok(a->prefix_v, a->prefix_stride, a->prefix_head_stride))
      return bad(op, "the prefixes' bases and strides must be multiples of 16 bytes");
  }
  if (a->capacity > 0) {
    if (a->k == nullptr || a->v == nullptr || a->caches == 0) return bad(op, "null pointer");
    if (!cache_ok(a->k, a->cache_stride, a->head_stride) || !cache_ok(a->v, a->cache_stride, a->head_stride))
      return bad(op, "the caches' bases and strides must be multiples of 16 bytes");
    if (a->ancestry == nullptr && a->caches != a->sequences)
      return bad(op, "without ancestry there is one cache per sequence");
    if (a->ancestry != nullptr && a->ld_ancestry < a->capacity) return bad(op, "a pitch is smaller than its row");
  }
  const int64_t need = static_cast<int64_t>(prefix_attention_bytes(*a));  // 0 without prefixes' keys
  if (need > 0 && (a->workspace == nullptr || !aligned(a->workspace, 16) || a->workspace_bytes < need))
    return bad(op, "the workspace is missing, too small or not 16-byte aligned (uocr_prefix_attention_workspace)");
  ErrorWord* err = nullptr;
  const cudaError_t st = ops_error_word(&err);
  return done(op, st != cudaSuccess ? st : launch_prefix_attention(*a, err, static_cast<cudaStream_t>(stream)));
}

int uocr_beam_select_workspace(const uocr_beam_select_args* a, int64_t* bytes) {
  const char* op = "beam_select_workspace";
  if (a == nullptr || bytes == nullptr) return bad(op, "null arguments");
  const int rc = check_select_sizes(op, a);
  if (rc != UOCR_OK) return rc;
  *bytes = static_cast<int64_t>(beam_select_bytes(*a));
  return UOCR_OK;
}

int uocr_beam_select(const uocr_beam_select_args* a, void* stream) {
  const char* op = "beam_select";
  if (a == nullptr) return bad(op, "null arguments");
  const int rc = check_select_sizes(op, a);
  if (rc != UOCR_OK) return rc;
  if (a->dtype != UOCR_DTYPE_F32 && a->dtype != UOCR_DTYPE_BF16) return bad(op, "logits must be f32 or bf16");
  if (a->eos < -1 || a->eos >= a->vocab) return bad(op, "eos must be a token or -1");
  if (a->batch == 0) return UOCR_OK;
  if (a->logits == nullptr || a->scores == nullptr || a->tokens == nullptr || a->parents == nullptr ||
      a->new_scores == nullptr)
    return bad(op, "null pointer");
  if (a->ld_logits < a->vocab) return bad(op, "a pitch is smaller than its row");
  if (!aligned(a->logits, a->dtype == UOCR_DTYPE_F32 ? 4 : 2)) return bad(op, "logits are misaligned");
  if (a->new_scores == a->scores || (a->new_finished != nullptr && a->new_finished == a->finished))
    return bad(op, "the new scores and flags may not take the place of the old ones");
  if (a->workspace == nullptr || !aligned(a->workspace, 16) ||
      a->workspace_bytes < static_cast<int64_t>(beam_select_bytes(*a)))
    return bad(op, "the workspace is missing, too small or not 16-byte aligned (uocr_beam_select_workspace)");
  return done(op, launch_beam_select(*a, static_cast<cudaStream_t>(stream)));
}

int uocr_reorder_states(const uocr_reorder_states_args* a, void* stream) {
  const char* op = "reorder_states";
  if (a == nullptr) return bad(op, "null arguments");
  if (!in(a->layers, 0, kMaxCount) || !in(a->groups, 0, kMaxCount) || !in(a->segments, 0, kMaxCount) ||
      !in(a->units, 0, kMaxCount) || !in(a->unit_bytes, 1, kMaxCount))
    return bad(op, "bad shape");
  if (!in(a->beams, 1, UOCR_BEAM_MAX)) return bad(op, "beams must be 1 .. 32");
  if (a->layers == 0 || a->groups == 0 || a->segments == 0 || a->units == 0) return UOCR_OK;
  if (a->state == nullptr || a->parents == nullptr) return bad(op, "null pointer");
  if (a->groups * a->beams > kMaxCount) return unsupported(op, "too many rows");
  const int64_t segment = a->units * a->unit_bytes;
  if ((a->beams * a->groups > 1 && a->row_stride < segment) || (a->segments > 1 && a->segment_stride < segment) ||
      (a->layers > 1 && a->layer_stride < segment))
    return bad(op, "a stride is smaller than a segment");
  // One block for every 128 columns of at least a byte.
  if (!product_fits({a->layers, a->groups, a->segments, segment}) ||
      a->layers * a->groups * a->segments > kMaxCount / ((segment + 127) / 128))
    return unsupported(op, "too large");
  if (!apart(segment, {{a->layers, a->layer_stride}, {a->groups * a->beams, a->row_stride}, {a->segments, a->segment_stride}}))
    return bad(op, "layers, rows or segments overlap");
  ErrorWord* err = nullptr;
  const cudaError_t st = ops_error_word(&err);
  return done(op, st != cudaSuccess ? st : launch_reorder_states(*a, err, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
