/*
 * uttt_decode.h -- C ABI of libuttt_amd.so's operators for decoding in 4 bits (slow and fast weights, ring caches) and
 * for beam search.
 *
 * The conventions are those of uttt_amd.h: device pointers, int64 sizes and strides in elements unless said otherwise, a
 * HIP stream; nothing allocates, frees or synchronises, so every call can be recorded into a HIP graph; 0 or an error
 * code comes back, uttt_last_error() describes it.  Values that lie on the device (positions, parents, counts)
 * cannot be refused by the host: each entry says what out-of-range ones do.
 *
 * Four bits: 32 neighbours along the contracted axis (along a head's elements in caches) are a group.  Its scale is
 * s = bf16(a * (1/6 in fp32)) with a the largest magnitude, 0 where that is below 2^-126, NaN where a value is not
 * finite.  The code of x is the one of {0, .5, 1, 1.5, 2, 3, 4, 6} nearest to |x| / s (the quotient in fp32; of two
 * as near the one whose index is even; 0 where s is), with bit 3 set for a negative value other than 0.
 *
 * Weights (n, k), k the contracted axis, zero-padded to whole blocks of 16 rows and 128 columns, the blocks of 16 rows one
 * after the other: a block is 1024 bytes of codes, then 16 x 4 bf16 scales (row by row).  Piece 16 h + r of 16 bytes holds,
 * for g = 0..3, in 4 bytes the codes of row r, columns 32 g + 8 h .. + 7, the first in the lowest bits.
 *
 * Caches: a request and kv head has ceil(sinks / 32) + ceil(window / 32) blocks of 32 slots, 36 head_dim bytes each.  The token
 * at position p lies in slot p for p < sinks, else in slot 32 ceil(sinks / 32) + (p - sinks) mod window.  A block is the codes of
 * its keys (16 head_dim bytes), of its values, the keys' scales (2 head_dim bytes) and the values'.  Codes come
 * in words of 8 (4 bytes): word w of lane l = 16 h + r lies at byte 1024 (w / 4) + 16 l + 4 (w mod 4).  Keys: word
 * t head_dim / 32 + g is slot 16 t + r, elements 32 g + 8 h .. + 7.  Values: word w is element 16 w + r of the slots 4 h .. 4 h + 3
 * and 16 + 4 h .. 16 + 4 h + 3.  Scales: group by group, the slots in that order, h = 0..3.
 */
#ifndef UTTT_DECODE_H
#define UTTT_DECODE_H

#include "uttt_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of the structures and entry points of this header (uttt_decode_abi_version() returns it). */
#define UTTT_DECODE_ABI_VERSION 1
int uttt_decode_abi_version(void);

/* ---------------------------------------------------------------------------
 * 1. out = x W^T (+ residual) with W in 4 bits, for the rows of a decode step: the slow projections and the LM head
 *    (engine/inference.py:222-279).  x_eps > 0: the rows of x are RMS-normalised first (the norm's weight belongs into W's
 *    columns before they are quantised).  Products are formed from x's own values (fp32 ones whole), sums in fp32;
 *    the result is rounded once.  out may be the residual, and lies apart from x.  x of any alignment and row stride >= k.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t m, n, k; /* m <= 2^20, n <= 2^24, k <= 2^20 */
  int32_t act_dtype;
  float x_eps;
  const void* x; int64_t x_row_stride;
  const void* w; /* 16-byte aligned */
  const void* residual; int64_t residual_row_stride; /* NULL: none */
  void* out; int64_t out_row_stride;
  void* workspace; size_t workspace_bytes; /* rewritten by each call; NULL where none is needed */
} uttt_linear4_args;

size_t uttt_linear4_workspace(int64_t m, int64_t k, int32_t act_dtype);
int uttt_linear4(const uttt_linear4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 2. uttt_swiglu_readout of a frozen state in 4 bits (model/uttt_layer.py:211-247): per batch row, with x' = x or, with
 *    x_norm_weight, RMSNorm(x) times that weight,  out = x' + LN((SiLU(x' W_gate) * (x' W_up)) W_down).
 *    w_up and w_gate hold (d_ff, d_model) matrices, w_down (d_model, d_ff): k is the contracted axis.  Strides of the
 *    batch in bytes, 0: one matrix for all.  The workspace is rewritten by each call.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t batch, tokens, d_model, d_ff; /* multiples of 64, d_model <= 4096 */
  int32_t act_dtype;
  float eps;
  const void* x; int64_t x_stride_b, x_stride_t; /* 16-byte aligned rows */
  const void* w_up; const void* w_gate; const void* w_down;
  int64_t w_up_stride, w_gate_stride, w_down_stride;
  const float* ln_weight; const float* ln_bias;
  const void* x_norm_weight; float x_norm_eps; /* NULL: x as it is; else x's dtype */
  void* out; int64_t out_stride_b, out_stride_t;
  void* workspace; size_t workspace_bytes;
} uttt_readout4_args;

size_t uttt_readout4_workspace(int64_t batch, int64_t tokens, int64_t d_model, int64_t d_ff);
int uttt_readout4(const uttt_readout4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 3. Attention of a few new tokens per request over its cache in 4 bits: uttt_swa_tree's trees, positions and masks
 *    (uttt_serve.h), the cache as above and never written.  Scores and sums are formed in fp32 from the values that
 *    the codes stand for.  One node per request is a decode step, whose token uttt_kv_commit4 then takes in.
 *    A request with a negative position, a position past the tables, or a node whose parent is neither -1 nor an
 *    earlier node gets NaN outputs and no key or value is written.  Values that a query does not see may be anything;
 *    a key whose score is -inf has no weight.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t n_req, n_heads, n_kv_heads, nodes, head_dim; /* head_dim 64 or 128; nodes in 1..64 */
  int64_t window, sinks;                               /* each <= 2^28 */
  int32_t act_dtype;
  float scale;
  const int64_t* positions;  /* device, (N,) */
  const int32_t* parents;    /* device, (N, nodes); NULL: each node's parent is the one before it */
  const int32_t* counts;     /* device, (N,) or NULL */
  const float* cos_table; const float* sin_table; int64_t table_len; /* NULL: inputs pre-rotated */
  const void* q; int64_t q_stride_n, q_stride_t, q_stride_h;
  const void* k_new; int64_t k_stride_n, k_stride_t, k_stride_h;
  const void* v_new; int64_t v_stride_n, v_stride_t, v_stride_h;
  const void* cache; int64_t cache_stride_n; /* bytes; (Hkv, blocks, 36 head_dim) inside; 0: one cache for all */
  void* out; int64_t o_stride_n, o_stride_t, o_stride_h;
  void* k_nodes; void* v_nodes; int64_t nodes_stride_n; /* (nodes, Hkv, hd) inside; both or neither; not k_new / v_new */
  void* workspace; size_t workspace_bytes; /* rewritten by every call: calls sharing it must be ordered */
} uttt_swa_tree4_args;

size_t uttt_swa_tree4_workspace(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes, int64_t head_dim,
                                int64_t window, int64_t sinks);
int uttt_swa_tree4(const uttt_swa_tree4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 4. Accepted tokens into the caches, all layers in one launch: node nodes[n][a], for a < counts[n], becomes the token
 *    at position positions[n] + a.  Without `nodes` it is node a, without counts all of the path's.  advance:
 *    positions[n] += counts[n] afterwards.  counts are taken into [0, path]; a node id outside [0, n_nodes)
 *    leaves its slot as it was; a request with a negative position is left as it was.  Where a path is
 *    longer than the window, the last token of a slot stays.  Slots that no token takes keep what they hold.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t layers, n_req, n_kv_heads, n_nodes, path, head_dim; /* head_dim 64 or 128 */
  int64_t window, sinks;
  int32_t act_dtype, advance;
  const void* k_nodes; const void* v_nodes;
  int64_t nodes_stride_l, nodes_stride_n, nodes_stride_t, nodes_stride_h; /* 16-byte aligned rows of head_dim */
  const int32_t* nodes; int64_t path_stride; /* device, (N, path) or NULL */
  const int32_t* counts;                     /* device, (N,) or NULL */
  void* cache; int64_t cache_stride_l, cache_stride_n; /* bytes */
  int64_t* positions;                        /* device, (N,) */
} uttt_kv_commit4_args;

int uttt_kv_commit4(const uttt_kv_commit4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 5. The values that caches hold, as (layers, N, Hkv, sinks + window, hd) in act_dtype (contiguous): row p of the first `sinks`
 *    rows is slot p, row sinks + r is ring slot r, as uttt_serve.h lays a ring out.  Slots that hold no token give
 *    whatever their bits stand for.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t layers, n_req, n_kv_heads, head_dim, window, sinks;
  int32_t act_dtype;
  const void* cache; int64_t cache_stride_l, cache_stride_n; /* bytes */
  void* k; void* v;
} uttt_kv_values4_args;

int uttt_kv_values4(const uttt_kv_values4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 6. uttt_kv_fork for caches in 4 bits: request n takes the cache and the position of request sources[n], as they were
 *    before the call.  sources[n] == n, or outside [0, N), leaves request n as it was.  At most 128 requests.
 *    With positions NULL whole caches are copied and no position.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t layers, n_req, n_kv_heads, head_dim, window, sinks;
  const int32_t* sources; /* device, (N,) */
  void* cache; int64_t cache_stride_l, cache_stride_n; /* bytes */
  int64_t* positions; /* device, (N,) or NULL */
} uttt_kv_fork4_args;

int uttt_kv_fork4(const uttt_kv_fork4_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 7. Beam search's choice: per group of `beams` rows, over beams b and the ids v that are below active_limit, not banned
 *    and above -inf, the `beams` best of  score_b + x_bv - log sum_v exp(x_bv)  (sum over those ids), of equal ones the
 *    lower beam's, then the lower id.  Scores are compared in 64 bits; a sum of exponentials is an fp32 one, off by some 2^-23
 *    (at most 2^-15) of itself, so that values of two beams that are closer than that may change places.  A beam with
 *    ended_in != 0 offers one continuation instead, `pad` at its own score; one whose score or whose largest logit is not
 *    finite, or with NaN among those ids, offers none.  Results, the best first: the token, the row it goes on from (uttt_kv_fork's
 *    sources), its score, and whether the beam has ended (its row had, or the token is eos; eos < 0: no id ends one).
 *    Where a group offers fewer than `beams`, the rest are `pad` at -inf from their own rows, ended.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t rows, vocab, beams; /* rows a multiple of beams; beams <= 32; vocab <= 2^20 */
  int32_t dtype;              /* UTTT_DTYPE_BF16 or UTTT_DTYPE_F32 logits */
  int32_t n_banned;           /* <= 8 */
  int32_t banned[8];
  int64_t active_limit; /* < 0 or >= vocab: no limit */
  int64_t eos, pad;
  const void* logits; int64_t row_stride; /* >= vocab */
  const float* scores;      /* (rows,) */
  const int32_t* ended_in;  /* (rows,) or NULL: none has ended */
  int64_t* tokens;          /* (rows,) */
  int32_t* sources;         /* (rows,) */
  float* out_scores;        /* (rows,); may be scores */
  int32_t* ended_out;       /* (rows,) or NULL; may be ended_in */
  void* workspace; size_t workspace_bytes; /* rewritten by every call */
} uttt_beam_select_args;

size_t uttt_beam_select_workspace(int64_t rows, int64_t vocab, int64_t beams);
int uttt_beam_select(const uttt_beam_select_args* args, uttt_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* UTTT_DECODE_H */
