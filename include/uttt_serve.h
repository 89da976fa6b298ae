/*
 * uttt_serve.h -- C ABI of the serving operators of libuttt_amd.so: sampling with per-request settings,
 * sliding-window attention with sinks (prompts, single tokens, trees of drafted tokens over ring caches),
 * and copies between caches.
 *
 * The conventions are those of uttt_amd.h: device pointers, int64 sizes and strides in elements, a HIP
 * stream; nothing allocates, frees or synchronises, so every call can be recorded into a HIP graph; 0 or an
 * error code comes back, uttt_last_error() describes it.  Values that lie on the device (positions,
 * parents, counts, settings) cannot be refused by the host: each entry says what out-of-range ones do.
 *
 * Cache layout of a request and kv head: sinks + window slots of head_dim elements.  The token at position
 * p lies in slot p for p < sinks, else in slot sinks + (p - sinks) mod window.  A query at position p sees the
 * token at position j <= p iff p - j < window or j < sinks.
 */
#ifndef UTTT_SERVE_H
#define UTTT_SERVE_H

#include "uttt_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of the structures and entry points of this header (uttt_serve_abi_version() returns it). */
#define UTTT_SERVE_ABI_VERSION 1
int uttt_serve_abi_version(void);

/* ---------------------------------------------------------------------------
 * 1. Sampling: the branches of uTTTModel.sample_next_token (model/uttt_model.py:1203-1235) above
 *    temperature 0, with top-k and min-p beside top-p, the random numbers given.  Per row, over the ids below
 *    active_limit that are not banned, in the order (logit descending, id ascending), with
 *    w_i = exp((x_i - max x) / temperature):
 *      top_k  keeps the first top_k ids                      (<= 0: all),
 *      min_p  keeps those with w_i >= min_p                  (<= 0 or NaN: all; above 1 as 1),
 *      top_p  keeps those whose mass ahead, among the kept ones, is <= top_p of their mass
 *             (>= 1 or NaN: all; below 0 as 0).
 *    out is the first id, in id order, at which the kept mass up to and including it exceeds
 *    uniform * total (uniforms are taken into [0, 1), NaN as 0); logprob is log(w_out / total).
 *    A temperature that is not above 1e-5 takes the argmax (uttt_greedy_select's rules), logprob 0; so does,
 *    with logprob NaN, a row whose largest logit is not finite (NaN, +inf, or nothing allowed above -inf).
 *    Sums are formed in fixed point (weights from 64-bit arithmetic, each to a whole step of 2^-42 of the largest),
 *    so equal inputs give equal bits whatever the order, the alignment and the other rows.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t rows, vocab; /* vocab <= 2^20 */
  int32_t dtype;       /* UTTT_DTYPE_BF16 or UTTT_DTYPE_F32 logits */
  int32_t n_banned;    /* <= 8 */
  int32_t banned[8];
  int64_t active_limit; /* < 0 or >= vocab: no limit */
  const void* logits; int64_t row_stride; /* >= vocab, or 0: one row for all */
  const float* uniforms;    /* (rows,) */
  const float* temperature; /* (rows,) */
  const int32_t* top_k;     /* (rows,) or NULL: off */
  const float* top_p;       /* (rows,) or NULL: off */
  const float* min_p;       /* (rows,) or NULL: off */
  int64_t* out;             /* (rows,) */
  float* logprob;           /* (rows,) or NULL */
  int64_t* advance;         /* optional (rows,): each entry is incremented by one */
} uttt_sample_args;

int uttt_sample_select(const uttt_sample_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 2. uttt_swa_prefill whose first `sinks` keys stay visible: query i (key index p = q_offset + i) sees key
 *    j <= p iff p - j < window or j < sinks.  sinks 0 is uttt_swa_prefill.  A continued prompt passes its
 *    cache's sink keys first, then the recent ones, then its own.  As in uttt_swa_prefill, values that only some
 *    queries of a tile see (a 64-key tile, the queries of a workgroup) must be finite: their weight of 0 meets them
 *    for the others.  Keys that no query of the call sees may hold anything.
 * ------------------------------------------------------------------------- */
size_t uttt_swa_prefill_sinks_workspace(int64_t batch, int64_t n_heads, int64_t q_len, int64_t kv_len,
                                        int64_t head_dim, int64_t window, int64_t sinks);
int uttt_swa_prefill_sinks(const uttt_swa_prefill_args* args, int64_t sinks, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 3. Attention of a few new tokens per request over its ring cache: a tree of drafted tokens (verification),
 *    or one token (a decode step, write_ring).  Request n has positions[n] tokens in its cache; its
 *    node i has depth 0 without a parent (-1), else its parent's depth + 1, and position
 *    positions[n] + depth.  A node sees the cached tokens and its ancestors and itself, by the rule above.
 *    With tables, q and k_new are rotated at their node's position; the nodes' keys (rotated) and values
 *    go to k_nodes / v_nodes (for uttt_kv_commit), or with write_ring (nodes == 1) into the ring.
 *    counts (optional): only the first counts[n] nodes of request n exist, rows behind them are neither read
 *    nor written.  A request with a negative position, a position past the tables, or a node whose parent is
 *    neither -1 nor an earlier node gets NaN outputs and no key or value is written.
 *    One head's slots of one request, taken as fp32, stay below 2 GB: (window + sinks) head_dim < 2^29.  Requests
 *    may share a ring (stride 0) where none is written.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t n_req, n_heads, n_kv_heads, nodes, head_dim; /* head_dim 64 or 128; nodes in 1..64 */
  int64_t window, sinks;
  int32_t act_dtype;
  int32_t write_ring;
  float scale;
  const int64_t* positions;  /* device, (N,) */
  const int32_t* parents;    /* device, (N, nodes); NULL: each node's parent is the one before it */
  const int32_t* counts;     /* device, (N,) or NULL */
  const float* cos_table; const float* sin_table; int64_t table_len; /* NULL: inputs pre-rotated */
  const void* q; int64_t q_stride_n, q_stride_t, q_stride_h;
  const void* k_new; int64_t k_stride_n, k_stride_t, k_stride_h;
  const void* v_new; int64_t v_stride_n, v_stride_t, v_stride_h;
  void* k_ring; void* v_ring; int64_t ring_stride_n; /* (N, Hkv, sinks + window, hd) */
  void* out; int64_t o_stride_n, o_stride_t, o_stride_h;
  void* k_nodes; void* v_nodes; /* (N, nodes, Hkv, hd) contiguous; NULL with write_ring */
  void* workspace; size_t workspace_bytes; /* rewritten by every call: calls sharing it must be ordered */
} uttt_swa_tree_args;

size_t uttt_swa_tree_workspace(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes, int64_t head_dim,
                               int64_t slots, int32_t act_dtype);
int uttt_swa_tree(const uttt_swa_tree_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 4. The accepted nodes of each request into its rings, all layers in one launch: node nodes[n][a], for
 *    a < counts[n], becomes the token at position positions[n] + a.  advance: positions[n] += counts[n]
 *    afterwards.  counts are taken into [0, path]; a node id outside [0, n_nodes) leaves its slot
 *    as it was; a request with a negative position is left as it was.  Where a path is longer than
 *    the window, the last token of a slot stays.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t layers, n_req, n_kv_heads, n_nodes, path, head_dim; /* path: length of a row of `nodes` */
  int64_t window, sinks;
  int32_t act_dtype, advance;
  const void* k_nodes; const void* v_nodes; int64_t nodes_stride_l, nodes_stride_n; /* (n_nodes, Hkv, hd) inside */
  const int32_t* nodes; int64_t path_stride; /* device, (N, path) */
  const int32_t* counts;                     /* device, (N,) */
  void* k_ring; void* v_ring; int64_t ring_stride_l, ring_stride_n; /* (Hkv, sinks + window, hd) inside */
  int64_t* positions;                        /* device, (N,) */
} uttt_kv_commit_args;

int uttt_kv_commit(const uttt_kv_commit_args* args, uttt_stream_t stream);

/* ---------------------------------------------------------------------------
 * 5. Requests' caches copied over others', all layers in one launch: request n takes the used slots
 *    and the position of request sources[n], as they were before the call (any map: forks, reorderings,
 *    cycles).  sources[n] == n, or outside [0, N), leaves request n as it was.  At most 128 requests.
 * ------------------------------------------------------------------------- */
typedef struct {
  int64_t layers, n_req, n_kv_heads, slots, head_dim;
  int32_t act_dtype;
  const int32_t* sources; /* device, (N,) */
  void* k_ring; void* v_ring; int64_t ring_stride_l, ring_stride_n;
  int64_t* positions;     /* device, (N,) */
} uttt_kv_fork_args;

int uttt_kv_fork(const uttt_kv_fork_args* args, uttt_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* UTTT_SERVE_H */
