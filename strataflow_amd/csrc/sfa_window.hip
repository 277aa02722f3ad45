// sfa_window.hip - attention of a sliding window with sinks over the paged
// cache (sfa_attn_decode_window, sfa_attn_prefill_window; include/sfa_window.h).
//
// The token at position t attends the positions p <= t with p < n_sink or
// p > t - window:  out = sum_p softmax_p(scale q.k_p) v_p.  Argument checks
// and workspace layout; the kernels are in sfa_window_decode.hip and
// sfa_window_prefill.hip.
#include "sfa_window_dev.h"

namespace sfa {

static bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static int window_args(const sfa_kv_desc *kv, const float *q, float *out, const int32_t *page_table,
                       int32_t max_pages, int32_t window, int32_t n_sink, float scale, WindowParams *p) {
    if (max_pages <= 0 || window <= 0 || n_sink < 0) return SFA_ERR_INVALID_ARGUMENT;
    if (!(scale > 0.0f) || !__builtin_isfinite(scale)) return SFA_ERR_INVALID_ARGUMENT;
    if (q == nullptr || out == nullptr || page_table == nullptr) return SFA_ERR_INVALID_ARGUMENT;
    if (!aligned(q, 16) || !aligned(out, 16)) return SFA_ERR_UNSUPPORTED;
    *p = WindowParams{};
    p->q = q;
    p->out = out;
    p->k_pages = static_cast<const uint8_t *>(kv->k_pages);
    p->v_pages = static_cast<const uint8_t *>(kv->v_pages);
    p->k_cold = static_cast<const uint8_t *>(kv->k_cold);
    p->v_cold = static_cast<const uint8_t *>(kv->v_cold);
    p->row_bytes = row_bytes_of(kv->kv_type, kv->head_dim);
    p->page_bytes = (int64_t)p->row_bytes * kv->n_head_kv * kv->page_size;
    p->n_pages = kv->n_pages;
    p->n_cold = kv->n_cold_pages;
    p->page_size = kv->page_size;
    p->page_shift = (kv->page_size & (kv->page_size - 1)) == 0 ? __builtin_ctz((unsigned)kv->page_size) : -1;
    p->max_pages = max_pages;
    p->n_head = kv->n_head;
    p->n_head_kv = kv->n_head_kv;
    p->page_table = page_table;
    p->window = window;
    p->n_sink = n_sink;
    p->scale_log2 = scale * 1.44269504088896340736f;
    if (!__builtin_isfinite(p->scale_log2)) return SFA_ERR_INVALID_ARGUMENT;
    // a tile's offsets are 32-bit, with room for those under its first row
    if ((int64_t)p->row_bytes * kv->n_head_kv * 64 > (1 << 30)) return SFA_ERR_UNSUPPORTED;
    return SFA_OK;
}

// Split records of `rows` rows in a workspace: the outputs, then the statistics.
static size_t records_bytes(int64_t rows, int n_split, int head_dim) {
    return n_split == 1 ? 256 : (size_t)rows * n_split * (head_dim + 2) * sizeof(float);
}
static void set_records(WindowParams *p, void *workspace, int64_t rows, int n_split, int head_dim) {
    p->n_split = n_split;
    p->rec_o = static_cast<float *>(workspace);
    p->rec_ml = reinterpret_cast<float2 *>(p->rec_o + rows * n_split * head_dim);
}

}  // namespace sfa

extern "C" {

SFA_API size_t sfa_decode_window_workspace_bytes(const sfa_kv_desc *kv, int32_t B, int32_t max_seq_len,
                                                 int32_t window, int32_t n_sink) {
    if (sfa_kv_desc_check(kv) != SFA_OK || B <= 0 || max_seq_len <= 0 || window <= 0 || n_sink < 0) return 0;
    return sfa::records_bytes((int64_t)B * kv->n_head, sfa::window_decode_splits(kv, B, max_seq_len, window, n_sink),
                              kv->head_dim);
}

SFA_API int sfa_attn_decode_window(const sfa_kv_desc *kv, const float *q, float *out,
                                   const int32_t *page_table, int32_t max_pages,
                                   const int32_t *seq_len, int32_t window, int32_t n_sink, int32_t B,
                                   int32_t max_seq_len, float scale, void *workspace, size_t ws_bytes,
                                   void *stream) {
    try {
        int rc = sfa_kv_desc_check(kv);
        if (rc != SFA_OK) return rc;
        if (B < 0 || max_seq_len <= 0) return SFA_ERR_INVALID_ARGUMENT;
        if (B == 0) return SFA_OK;
        sfa::WindowParams p;
        rc = sfa::window_args(kv, q, out, page_table, max_pages, window, n_sink, scale, &p);
        if (rc != SFA_OK) return rc;
        if (seq_len == nullptr || workspace == nullptr) return SFA_ERR_INVALID_ARGUMENT;
        if (!sfa::aligned(workspace, 256)) return SFA_ERR_UNSUPPORTED;
        if (ws_bytes < sfa_decode_window_workspace_bytes(kv, B, max_seq_len, window, n_sink))
            return SFA_ERR_INVALID_ARGUMENT;
        p.seq_len = seq_len;
        p.n_tok = B;
        sfa::set_records(&p, workspace, (int64_t)B * kv->n_head,
                         sfa::window_decode_splits(kv, B, max_seq_len, window, n_sink), kv->head_dim);
        return sfa::window_decode_launch(p, kv, B, static_cast<hipStream_t>(stream));
    } catch (...) {
        return SFA_ERR_RUNTIME;
    }
}

SFA_API size_t sfa_prefill_window_workspace_bytes(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T,
                                                  int32_t window, int32_t n_sink) {
    if (sfa_kv_desc_check(kv) != SFA_OK || q_pos0 < 0 || T <= 0 || (int64_t)q_pos0 + T > INT32_MAX || window <= 0 || n_sink < 0)
        return 0;
    const int n = sfa::window_prefill_splits(kv, q_pos0, T, window, n_sink);
    return n == 1 ? 0 : sfa::records_bytes((int64_t)T * kv->n_head, n, kv->head_dim);
}

SFA_API size_t sfa_prefill_window_workspace_bound(const sfa_kv_desc *kv, int32_t max_T) {
    if (sfa_kv_desc_check(kv) != SFA_OK || max_T <= 0) return 0;
    return sfa::records_bytes(sfa::window_prefill_most_records(kv, max_T), 2, kv->head_dim) / 2;
}

SFA_API int sfa_attn_prefill_window(const sfa_kv_desc *kv, const float *q, float *out,
                                    const int32_t *page_table, int32_t max_pages, int32_t q_pos0,
                                    int32_t T, int32_t window, int32_t n_sink, float scale,
                                    void *workspace, size_t ws_bytes, void *stream) {
    try {
        int rc = sfa_kv_desc_check(kv);
        if (rc != SFA_OK) return rc;
        if (T < 0 || q_pos0 < 0 || (int64_t)q_pos0 + T > INT32_MAX) return SFA_ERR_INVALID_ARGUMENT;
        if (T == 0) return SFA_OK;
        sfa::WindowParams p;
        rc = sfa::window_args(kv, q, out, page_table, max_pages, window, n_sink, scale, &p);
        if (rc != SFA_OK) return rc;
        if (kv->page_size % 64 != 0) return SFA_ERR_UNSUPPORTED;
        const size_t need = sfa_prefill_window_workspace_bytes(kv, q_pos0, T, window, n_sink);
        if (need != 0 && workspace == nullptr) return SFA_ERR_INVALID_ARGUMENT;
        if (need != 0 && !sfa::aligned(workspace, 256)) return SFA_ERR_UNSUPPORTED;
        if (ws_bytes < need) return SFA_ERR_INVALID_ARGUMENT;
        p.q_pos0 = q_pos0;
        p.n_tok = T;
        sfa::set_records(&p, workspace, (int64_t)T * kv->n_head,
                         sfa::window_prefill_splits(kv, q_pos0, T, window, n_sink), kv->head_dim);
        return sfa::window_prefill_launch(p, kv, static_cast<hipStream_t>(stream));
    } catch (...) {
        return SFA_ERR_RUNTIME;
    }
}

}  // extern "C"
