/*
 * sfa_window.h - C ABI of the attention node of windowed models over the paged
 * cache of sfa.h (libsfa.so): the append that norms the heads of Q and K and
 * rotates them by one position or several axes, and the attention of a sliding
 * window with a few first tokens that stay visible (sinks), for single tokens
 * and for prompt chunks.
 *
 * The reference's layer has neither head norms nor a window in its attention
 * (its KV window bounds residency only, src/kv/kv_store.h:1-22); the calls
 * stand beside sfa_rope_kv_append, sfa_attn_decode and sfa_attn_prefill for
 * models that do.  Layouts, page tables, page ids, GQA and status codes are
 * those of sfa.h.  Every call is ordered on the given stream, allocates
 * nothing, keeps no state and never throws; pointers are device pointers of
 * the device that is current.
 *
 * Arithmetic: norms, angles, scores, softmax statistics and outputs are held
 * in 32 bits or more (angles are reduced in 64).  Unlike sfa_attn_decode and
 * sfa_attn_prefill the attentions here round neither Q nor a probability to 16
 * bits: over an F16 or Q8_0 cache a 32-bit factor goes through the matrix
 * cores as two f16 halves, so that outputs are those of 32-bit arithmetic on
 * the values that the cache holds (relative error of some 1e-6).  Over an F32
 * cache K and V beyond 2^90 may overflow on the way.
 *
 * NaN and infinities: what a token may not see has no part in its row.  Of
 * what it sees, a NaN in K makes the head's outputs NaN, one in V those of its
 * element (Q8_0: of the block with such a scale); an infinity may do the same.
 */
#ifndef SFA_WINDOW_H
#define SFA_WINDOW_H

#include "sfa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Which elements of a head form a pair (ggml's ids of the rope modes). */
#define SFA_ROPE_NORMAL 0 /* (x[2i], x[2i+1])            */
#define SFA_ROPE_NEOX   2 /* (x[i], x[i + n_rot/2])      */

/* How the n_rot/2 pairs are dealt to the axes of a position. */
#define SFA_AXES_BLOCKS      0 /* sections[0] pairs to axis 0, the next sections[1] to axis 1, ... */
#define SFA_AXES_INTERLEAVED 1 /* pair i to axis i % n_axis; where that axis (1 or higher) has its
                                  sections[] pairs already, to axis 0                              */

/* A rotation: pair i turns by the angle p * freq_base^(-2i/n_rot), p the
 * token's position on the pair's axis. */
typedef struct sfa_rope_desc {
    int32_t n_rot;       /* leading elements of a head that rotate, a multiple of 8 up to head_dim;
                            the others pass through                                               */
    int32_t pairing;     /* SFA_ROPE_NORMAL or SFA_ROPE_NEOX                                       */
    float   freq_base;   /* > 0, finite                                                            */
    int32_t n_axis;      /* 1 to 4 (time, height, width, ...)                                      */
    int32_t sections[4]; /* pairs of each axis, adding up to n_rot/2 (n_axis 1: not read)          */
    int32_t layout;      /* SFA_AXES_BLOCKS or SFA_AXES_INTERLEAVED (n_axis 1: not read)           */
} sfa_rope_desc;

/* Validates a rotation for heads of head_dim elements (host only). */
SFA_API int sfa_rope_desc_check(const sfa_rope_desc *rope, int32_t head_dim);

/* Head norms, rotation and KV append in one pass.  Per token and head:
 *   y = x * 1/sqrt(mean(x^2) + eps) * norm      (Q with q_norm, K with k_norm [head_dim])
 *   y rotated by `rope`
 * Q goes to q_out, K and V (V as it is) into the cache as sfa_kv_append
 * converts.  q_norm and k_norm may each be NULL: those heads are only rotated.
 *   q, k, v : row of token t at q + t * q_stride, ... (strides in floats), each
 *             [n_heads][head_dim] f32 within a token, so the stacked rows of a
 *             Q/K/V product are taken as they are.  q may be NULL (K and V only).
 *   q_out   : [n_tok][n_head][head_dim] f32, contiguous; may be q where
 *             q_stride is n_head * head_dim, and must not overlap the inputs
 *             otherwise
 *   seq, pos, page_table, max_pages : as sfa_kv_append; pos names the cache position
 *   rope_pos: [n_axis][n_tok] int32, the positions that rotate (any sign), or
 *             NULL for `pos` on every axis
 * A token with seq < 0 or pos < 0 is skipped (its q_out row is not written); one
 * whose page is not there has its Q written only.  Where two tokens name the
 * same position, what that row then holds is not defined.
 * q, q_out, k and v 16-byte aligned, strides multiples of 4 that hold a
 * token's heads (one token: any); else SFA_ERR_UNSUPPORTED, or
 * SFA_ERR_INVALID_ARGUMENT for a stride that is too small. */
SFA_API int sfa_norm_rope_kv_append(const sfa_kv_desc *kv, const sfa_rope_desc *rope, const float *q,
                                    int64_t q_stride, float *q_out, const float *k, int64_t k_stride,
                                    const float *v, int64_t v_stride, const float *q_norm,
                                    const float *k_norm, float eps, const int32_t *seq,
                                    const int32_t *pos, const int32_t *rope_pos, int32_t n_tok,
                                    const int32_t *page_table, int32_t max_pages, void *stream);

/* Workspace bytes of sfa_attn_decode_window; 0 for an invalid shape. */
SFA_API size_t sfa_decode_window_workspace_bytes(const sfa_kv_desc *kv, int32_t B, int32_t max_seq_len,
                                                 int32_t window, int32_t n_sink);

/* Decode attention of one token per sequence, at position t = seq_len[b] - 1,
 * over the positions p <= t with p < n_sink or p > t - window (each once).
 * window >= 1 (INT32_MAX for none), n_sink >= 0.  q, out, page_table, seq_len,
 * max_pages and scale as sfa_attn_decode.  max_seq_len: host bound on
 * seq_len[b], which sizes the split and the workspace; a longer sequence is
 * attended in full, by longer splits.  A sequence with seq_len <= 0, or none of
 * whose pages is there, gets zeros; positions past the table or on a page that
 * is not there are not attended, and pages outside the window and the sinks are
 * not read, so their entries may be -1.
 * q and out 16-byte aligned and the workspace 256-byte aligned, B and n_head_kv
 * at most 65535, 64 positions of a tensor in at most 1 GiB (else
 * SFA_ERR_UNSUPPORTED).  scale > 0, and scale * log2(e) finite.  Calls that overlap in time need a workspace each; its
 * contents before a call do not matter. */
SFA_API int sfa_attn_decode_window(const sfa_kv_desc *kv, const float *q, float *out,
                                   const int32_t *page_table, int32_t max_pages,
                                   const int32_t *seq_len, int32_t window, int32_t n_sink, int32_t B,
                                   int32_t max_seq_len, float scale, void *workspace, size_t ws_bytes,
                                   void *stream);

/* Workspace bytes of sfa_attn_prefill_window; 0 where it needs none, and for
 * an invalid shape. */
SFA_API size_t sfa_prefill_window_workspace_bytes(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T,
                                                  int32_t window, int32_t n_sink);

/* Workspace bytes that every sfa_attn_prefill_window of at most max_T tokens
 * over this cache fits in, whatever its position, window and sinks; 0 where none
 * needs any, and for an invalid shape. */
SFA_API size_t sfa_prefill_window_workspace_bound(const sfa_kv_desc *kv, int32_t max_T);

/* Chunk attention of ONE sequence: T query tokens at positions q_pos0 ..
 * q_pos0 + T - 1, whose K/V are appended; the token at position t attends the
 * positions p <= t with p < n_sink or p > t - window.  q, out, page_table,
 * max_pages, scale as sfa_attn_prefill; q_pos0 + T must not pass INT32_MAX.
 * Positions past the table or on a page that is not there are not attended; a
 * token that so attends nothing gets zeros.  page_size must be a multiple of 64
 * and T * n_head / n_head_kv at most 65535 * 128 (SFA_ERR_UNSUPPORTED
 * otherwise); alignment, scale and workspace as sfa_attn_decode_window. */
SFA_API int sfa_attn_prefill_window(const sfa_kv_desc *kv, const float *q, float *out,
                                    const int32_t *page_table, int32_t max_pages, int32_t q_pos0,
                                    int32_t T, int32_t window, int32_t n_sink, float scale,
                                    void *workspace, size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SFA_WINDOW_H */
