/* uocr_beam.h — C ABI of the operators for sequences that share a page.
 *
 * Several continuations of one prefix (the beams of a search, or different
 * prompts on one page) need, around the products of uocr_moe.h: queries and
 * keys normalised, rotated and appended to caches; attention over the shared
 * prefix, read once for all of them, and over each one's own keys; the
 * selection of the next beams over beams and vocabulary; and the beams' states
 * brought into their new order. uocr_decoder_beam_search runs them on the page
 * decoder of uocr_decoder.h.
 *
 * Conventions are uocr_moe.h's: plain device pointers, a cudaStream_t passed as
 * void*, status codes with uocr_last_error(), nothing synchronises the stream
 * and nothing is allocated. Pitches and strides are counted in elements unless
 * a field says bytes. Lengths, offsets, slots and parents stay on the device;
 * a bad one is recorded in the device's error word (uocr_ops_check), and nothing
 * outside the arrays is read or written.
 */
#ifndef UOCR_BEAM_H
#define UOCR_BEAM_H

#include <stdint.h>

#include "uocr_decoder.h"
#include "uocr_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotation of heads ---- */

/* How a rotary table is stretched for long contexts. */
typedef enum uocr_rope_scaling {
  UOCR_ROPE_PLAIN = 0,
  UOCR_ROPE_LINEAR = 1, /* every frequency divided by factor */
  UOCR_ROPE_NTK = 2,    /* theta * factor^(d / (d - 2)): the lowest frequency divided by factor, the highest kept */
  UOCR_ROPE_YARN = 3    /* by the turns a pair makes within `original` positions: above 32 kept, below 1 divided,
                         * between the two a linear ramp over the pairs; magnitude 0.1 ln(factor) + 1 */
} uocr_rope_scaling;

/* Host: inv_freq [rotary_dim / 2] (host memory) = float(theta^(-2 i / rotary_dim)),
 * stretched; *magnitude (may be NULL) = what cos and sin are multiplied by.
 * factor >= 1; original > 0 matters to UOCR_ROPE_YARN alone. */
int uocr_rope_frequencies(int64_t rotary_dim, double theta, int32_t scaling, double factor, int64_t original,
                          float* inv_freq, float* magnitude);

typedef struct uocr_rotate_heads_args {
  const void* q;             /* [rows, q_heads, head_dim], pitch ldq */
  const void* k;             /* [rows, kv_heads, head_dim], pitch ldk; NULL with kv_heads 0 */
  const void* v;             /* [rows, kv_heads, head_dim], pitch ldv */
  const float* q_norm;       /* [head_dim] RMSNorm gain of a query head, or NULL: no norm */
  const float* k_norm;       /* [head_dim] of a key head, or NULL */
  const float* inv_freq;     /* [rotary_dim / 2] */
  const int32_t* positions;  /* [rows] */
  const int32_t* cache_rows; /* [rows]: row r goes into cache cache_rows[r]; NULL: cache r */
  const int32_t* slots;      /* [rows]: at this place of the cache; NULL: positions[r] */
  uint16_t* q_out;           /* bf16 [rows, q_heads, head_dim], pitch ldqo; may be q itself (bf16, ldqo == ldq) */
  uint16_t* k_cache;         /* bf16 [caches, kv_heads, capacity, head_dim] with the two strides below */
  uint16_t* v_cache;         /* the same */
  int64_t rows, q_heads, kv_heads, head_dim, rotary_dim;
  int64_t ldq, ldk, ldv, ldqo;
  int64_t caches, capacity;
  int64_t cache_stride, head_stride; /* elements between caches, between a cache's heads */
  float eps;                 /* of the norms */
  float magnitude;           /* cos and sin are multiplied by it (1 for plain tables) */
  int32_t dtype;             /* of q, k, v: UOCR_DTYPE_F32 or UOCR_DTYPE_BF16 */
  int32_t interleaved;       /* 0: pairs (i, i + rotary_dim / 2), the page decoder's layout; 1: pairs (2 i, 2 i + 1) */
} uocr_rotate_heads_args;

/* Every query and key head of every row: x * rsqrt(mean(x^2) + eps) * gain where
 * a gain is given, then over the first rotary_dim dimensions (a, b) ->
 * (a cos - b sin, b cos + a sin) at the angle positions[r] * inv_freq[i] — formed
 * in 64 bits, so that far positions keep their angle — rounded to bf16: q into
 * q_out, k and v (v only rounded) into the caches at [cache_rows[r], :, slots[r]].
 * head_dim is a multiple of 8 up to 256, rotary_dim one of 8 up to head_dim (0:
 * no rotation). The caches' bases and strides are multiples of 16 bytes, and caches
 * and heads lie apart. A row
 * whose cache or slot does not exist is not appended (recorded); of two rows
 * with the same place, either may stay. */
int uocr_rotate_heads(const uocr_rotate_heads_args* args, void* stream);

/* ---- attention behind shared prefixes ---- */

typedef struct uocr_prefix_attention_args {
  const uint16_t* q;            /* bf16 [rows, heads, head_dim], pitch ldq */
  const uint16_t* prefix_k;     /* bf16 [prefixes, kv_heads, prefix_capacity, head_dim], two strides below */
  const uint16_t* prefix_v;
  const int32_t* prefix_lens;   /* [prefixes]: keys of each prefix, 0 .. prefix_capacity */
  const uint16_t* k;            /* bf16 [caches, kv_heads, capacity, head_dim], two strides below */
  const uint16_t* v;
  const int32_t* lens;          /* [sequences]: own keys of each sequence, 0 .. capacity, its rows' own among them */
  const int32_t* ancestry;      /* [sequences, capacity], pitch ld_ancestry: own key t of sequence b lies in cache
                                 * ancestry[b, t], at t; NULL: in cache b (caches == sequences) */
  const int32_t* row_offsets;   /* [sequences + 1]: sequence b has the rows row_offsets[b] .. row_offsets[b + 1] - 1;
                                 * NULL: row b (rows == sequences) */
  uint16_t* out;                /* bf16 [rows, heads, head_dim], pitch ldo */
  float* lse;                   /* [rows, heads]: log of the sum of a row's exponentials; or NULL */
  int64_t rows, sequences, prefixes, caches;
  int64_t heads, kv_heads, head_dim;
  int64_t prefix_capacity, capacity;
  int64_t ldq, ldo, ld_ancestry;
  int64_t prefix_stride, prefix_head_stride;
  int64_t cache_stride, head_stride;
  float scale;                  /* of the scores */
  int32_t reserved;             /* 0 */
  void* workspace;              /* device memory for the call's duration, 16-byte aligned */
  int64_t workspace_bytes;      /* at least what uocr_prefix_attention_workspace says */
} uocr_prefix_attention_args;

/* Bytes of workspace the call below needs with these sizes (pointers are not
 * looked at, but for row_offsets being NULL or not; nor are scale, pitches and strides). */
int uocr_prefix_attention_workspace(const uocr_prefix_attention_args* args, int64_t* bytes);

/* out = softmax(scale * q k^T) v. Sequence b stands behind prefix
 * b / (sequences / prefixes) and sees all its keys; row j of the sequence's n
 * rows also sees its own keys t < lens[b] - (n - 1 - j): its last row all of
 * them, the ones before it one less each, as the new tokens of a sequence do.
 * Query head h reads key/value head h / (heads / kv_heads). A prefix is read
 * once for all its sequences. A row that sees no key is 0, its lse -inf. What
 * lies in a cache behind a length is not read into a result, NaN included.
 * Scores, sums and the products' accumulators are fp32; the weights of the
 * values are rounded to bf16 (the tensor cores' operand), one below 2^-126 of a
 * row's greatest so far counts as 0. head_dim is 64 or 128.
 * Rows outside row_offsets[0] .. row_offsets[sequences] are left as they are.
 * A length out of range is recorded and taken as the nearest that is in range;
 * a sequence whose row offsets are not in order is recorded, its rows
 * unspecified (where such offsets name rows many times over, all rows); a bad
 * ancestor is recorded, and the sequence's own cache (cache 0 where it has none)
 * read in its place. */
int uocr_prefix_attention(const uocr_prefix_attention_args* args, void* stream);

/* ---- selection of beams ---- */

#define UOCR_BEAM_MAX 32 /* beams of a group, and candidates selected for it */

typedef struct uocr_beam_select_args {
  const void* logits;       /* [batch * beams, vocab], pitch ld_logits */
  const float* scores;      /* [batch, beams]: each beam's log-probability so far; -inf: the beam does not exist */
  const int32_t* finished;  /* [batch, beams]: not 0: the beam has ended; NULL: none has */
  int32_t* tokens;          /* [batch, select] */
  int32_t* parents;         /* [batch, select]: the beam (0 .. beams - 1) a candidate continues */
  float* new_scores;        /* [batch, select]; may not be scores itself */
  int32_t* new_finished;    /* [batch, select], or NULL; may not be finished itself */
  int64_t batch, beams, select, vocab;
  int64_t ld_logits;
  int32_t dtype;            /* of logits: UOCR_DTYPE_F32 or UOCR_DTYPE_BF16 */
  int32_t eos;              /* the token that ends a beam; -1: none */
  void* workspace;          /* device memory for the call's duration, 16-byte aligned */
  int64_t workspace_bytes;  /* at least what uocr_beam_select_workspace says */
} uocr_beam_select_args;

int uocr_beam_select_workspace(const uocr_beam_select_args* args, int64_t* bytes);

/* Of each batch entry's candidates (b, t) with the score scores[b] +
 * log_softmax(logits[b])[t] the `select` best, best first, equal ones by the
 * lower beam, within a beam by the higher logit (a score far from 0 cannot tell
 * close ones apart), then the lower token. A finished beam has one candidate: its eos
 * again (token 0 with eos -1), its score unchanged. A candidate whose score is
 * NaN or -inf, or rounds to -inf, is none (a NaN logit, as -inf; a row that holds
 * +inf has none). Finite logits of any size, masks of the type's lowest value
 * among them, are logits like others.
 * Where candidates run out: token max(eos, 0), parent 0, score -inf, finished.
 * new_finished: the parent was finished, or the token is eos. The scores'
 * comparison is made in 64 bits on sums of fp32 exponentials. */
int uocr_beam_select(const uocr_beam_select_args* args, void* stream);

/* ---- reordering of states ---- */

typedef struct uocr_reorder_states_args {
  void* state;             /* [layers, groups * beams, segments, units of unit_bytes], the units of a segment
                            * contiguous; byte strides below */
  const int32_t* parents;  /* [groups, beams]: 0 .. beams - 1 */
  const int32_t* counts;   /* [groups * beams]: units in use of each row before the call, or NULL: all */
  int64_t layers, groups, beams, segments, units, unit_bytes;
  int64_t layer_stride, row_stride, segment_stride; /* bytes */
} uocr_reorder_states_args;

/* state[:, g * beams + b] = state[:, g * beams + parents[g, b]], in place, for
 * all beams at once: counts[parent] units of every segment; what follows them in
 * the row stays. A beam that is its own parent is not touched. beams is at most
 * UOCR_BEAM_MAX. A bad parent is recorded and leaves its row as it is; a count
 * out of range is recorded and taken as the nearest that is in range. Layers, rows
 * and segments lie apart, in any order. */
int uocr_reorder_states(const uocr_reorder_states_args* args, void* stream);

/* ---- beam search on the page decoder ---- */

typedef struct uocr_beam_search_args {
  int64_t beams;            /* 1 .. 16, at most the decoder's max_prefill */
  int64_t steps;            /* tokens of each beam */
  int32_t eos;              /* the token that ends a beam, or -1 */
  int32_t reserved;         /* 0 */
  int32_t* tokens;          /* [beams, steps]: the beams' tokens, best beam first; behind a beam's end its eos */
  float* scores;            /* [beams]: their log-probabilities */
  int32_t* lengths;         /* [beams]: tokens up to and with the first eos, or NULL */
  void* workspace;          /* device memory for the call's duration, 256-byte aligned: the beams' caches */
  int64_t workspace_bytes;  /* at least what uocr_decoder_beam_workspace says */
} uocr_beam_search_args;

int uocr_decoder_beam_workspace(const uocr_decoder* dec, int64_t beams, int64_t steps, int64_t* bytes);

/* `steps` tokens for `beams` beams behind the decoder's sequence (a prefill, and
 * the decode steps after it): the first tokens come from the logits that the
 * sequence ended with, each later step runs all beams as one batch over the
 * sequence's cache, shared, and their own. The sequence itself stays as it is: a
 * decode or another search may follow. A captured search may be replayed as long
 * as the sequence is the one it was captured with. The sequence and the steps have
 * to fit max_positions. Decoders with int8 weights expand them to bf16 in every step, as
 * their prefill does; with UOCR_DECODER_INT8_ACTIVATIONS the projections and the
 * head run on int8 activations. */
int uocr_decoder_beam_search(uocr_decoder* dec, const uocr_beam_search_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* UOCR_BEAM_H */
