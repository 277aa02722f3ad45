// sfa_window.hip - attention of a sliding window with sinks over the paged
// cache (sfa_attn_decode_window, sfa_attn_prefill_window; include/sfa_window.h).
//
// The token at position t attends the positions p <= t with p < n_sink or
// p > t - window:  out = sum_p softmax_p(scale q.k_p) v_p, one pass with the
// running maximum and sum of the softmax.
#include <exception>

#include "sfa_window_dev.h"

namespace sfa {

int window_decode_splits(const sfa_kv_desc *kv, int32_t B, int32_t max_seq_len, int32_t window, int32_t n_sink);
int window_decode_launch(const WindowParams &p, const sfa_kv_desc *kv, int32_t B, hipStream_t s);

// What one token attends: [0, ns) and [lo, hi].
struct Span {
    int ns, lo, hi;
    __device__ inline int count() const { return ns + (hi >= lo ? hi - lo + 1 : 0); }
    __device__ inline int at(int j) const { return j < ns ? j : lo + j - ns; }
};
__device__ inline Span span_of(const WindowParams &p, int pos) {
    const int64_t cap = (int64_t)p.max_pages * p.page_size;
    Span s;
    s.lo = pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
    s.hi = pos < cap ? pos : (int)(cap - 1);
    s.ns = min(min(p.n_sink, s.lo), s.hi + 1);
    return s;
}

// Element e of a row, any cache type.
template <int KVT>
__device__ inline float row_value(const uint8_t *row, int e) {
    if constexpr (KVT == SFA_KV_F32) return reinterpret_cast<const float *>(row)[e];
    if constexpr (KVT == SFA_KV_F16) return (float)reinterpret_cast<const _Float16 *>(row)[e];
    const uint8_t *b = row + e / kQK * kQ8Bytes;
    return (float)*reinterpret_cast<const _Float16 *>(b) * (float)reinterpret_cast<const int8_t *>(b + 2)[e % kQK];
}

// One workgroup per (token, kv head): a lane takes a position's scores of all G
// heads, then a lane takes dims of the outputs; four waves share the span.
template <int KVT, int HD, int G>
__global__ __launch_bounds__(256) void window_simple_kernel(WindowParams p) {
    __shared__ float qs[G][HD];
    __shared__ float ps[4][G][kWave];
    __shared__ float om[4][G], ol[4][G], oo[4][G][HD];
    constexpr int D = HD > kWave ? HD / kWave : 1;
    const int t = blockIdx.x, kvh = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < G * HD; i += 256)
        qs[i / HD][i % HD] = p.q[((int64_t)t * p.n_head + kvh * G) * HD + i] * p.scale_log2;
    __syncthreads();
    const Span sp = span_of(p, p.q_pos0 + t);
    const int n = sp.count();
    const int32_t *table = p.page_table;
    float m[G], l[G], o[G][D];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int d = 0; d < D; ++d) o[g][d] = 0.0f;
    }
    for (int j0 = wave * kWave; j0 < n; j0 += 4 * kWave) {
        const int j = j0 + lane;
        const uint8_t *kr = nullptr, *vr = nullptr;
        if (j < n) {
            const int x = sp.at(j);
            const int lp = x / p.page_size;
            const int64_t off = ((int64_t)(x - lp * p.page_size) * p.n_head_kv + kvh) * p.row_bytes;
            const uint8_t *kb = page_base(table[lp], p.k_pages, p.n_pages, p.k_cold, p.n_cold, p.page_bytes);
            const uint8_t *vb = page_base(table[lp], p.v_pages, p.n_pages, p.v_cold, p.n_cold, p.page_bytes);
            if (kb != nullptr && vb != nullptr) kr = kb + off, vr = vb + off;
        }
        float s[G];
#pragma unroll
        for (int g = 0; g < G; ++g) s[g] = kr != nullptr ? 0.0f : -INFINITY;
        if (kr != nullptr)
            for (int e = 0; e < HD; ++e) {
                const float x = row_value<KVT>(kr, e);
#pragma unroll
                for (int g = 0; g < G; ++g) s[g] = fmaf(x, qs[g][e], s[g]);
            }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float mn = fmaxf(m[g], wave_max(s[g]));
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float w = exp2f(s[g] - base), f = exp2f(m[g] - base);
            m[g] = mn;
            l[g] = l[g] * f + wave_sum(w);
#pragma unroll
            for (int d = 0; d < D; ++d) o[g][d] *= f;
            ps[wave][g][lane] = w;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint64_t mine = reinterpret_cast<uint64_t>(vr);
        for (int i = 0; i < kWave; ++i) {
            const uint32_t u0 = __builtin_amdgcn_readlane((int)(uint32_t)mine, i);
            const uint32_t u1 = __builtin_amdgcn_readlane((int)(mine >> 32), i);
            const uint8_t *row = reinterpret_cast<const uint8_t *>((uint64_t)u1 << 32 | u0);
            if (row == nullptr) continue;
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int e = lane + d * kWave;
                if (e >= HD) continue;
                const float x = row_value<KVT>(row, e);
#pragma unroll
                for (int g = 0; g < G; ++g) o[g][d] = fmaf(ps[wave][g][i], x, o[g][d]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        om[wave][g] = m[g];
        ol[wave][g] = l[g];
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (lane + d * kWave < HD) oo[wave][g][lane + d * kWave] = o[g][d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * HD; i += 256) {
        const int g = i / HD, e = i % HD;
        float mm = fmaxf(fmaxf(om[0][g], om[1][g]), fmaxf(om[2][g], om[3][g]));
        if (mm == -INFINITY) mm = 0.0f;
        float L = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2f(om[w][g] - mm);
            L = fmaf(ol[w][g], f, L);
            acc = fmaf(oo[w][g][e], f, acc);
        }
        p.out[((int64_t)t * p.n_head + kvh * G) * HD + i] = L == 0.0f ? 0.0f : acc / L;
    }
}

template <int KVT, int HD>
static void launch_g(const WindowParams &p, int n_rows, hipStream_t s) {
    const dim3 grid((unsigned)n_rows, (unsigned)p.n_head_kv), block(256);
    switch (p.n_head / p.n_head_kv) {
    case 1: hipLaunchKernelGGL((window_simple_kernel<KVT, HD, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((window_simple_kernel<KVT, HD, 2>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((window_simple_kernel<KVT, HD, 4>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((window_simple_kernel<KVT, HD, 8>), grid, block, 0, s, p); break;
    }
}

template <int KVT>
static int launch_hd(const WindowParams &p, int head_dim, int n_rows, hipStream_t s) {
    if (head_dim == 128) launch_g<KVT, 128>(p, n_rows, s);
    else if (head_dim == 64) launch_g<KVT, 64>(p, n_rows, s);
    else if constexpr (KVT != SFA_KV_Q8_0) launch_g<KVT, 32>(p, n_rows, s);
    else return SFA_ERR_UNSUPPORTED;
    return hipGetLastError() == hipSuccess ? SFA_OK : SFA_ERR_RUNTIME;
}

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
    p->max_pages = max_pages;
    p->n_head = kv->n_head;
    p->n_head_kv = kv->n_head_kv;
    p->page_table = page_table;
    p->window = window;
    p->n_sink = n_sink;
    p->scale_log2 = scale * 1.44269504088896340736f;
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

static int window_launch(const sfa_kv_desc *kv, const WindowParams &p, int n_rows, hipStream_t stream) {
    switch (kv->kv_type) {
    case SFA_KV_F32: return launch_hd<SFA_KV_F32>(p, kv->head_dim, n_rows, stream);
    case SFA_KV_F16: return launch_hd<SFA_KV_F16>(p, kv->head_dim, n_rows, stream);
    case SFA_KV_Q8_0: return launch_hd<SFA_KV_Q8_0>(p, kv->head_dim, n_rows, stream);
    default: return SFA_ERR_UNSUPPORTED;
    }
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
        sfa::set_records(&p, workspace, (int64_t)B * kv->n_head,
                         sfa::window_decode_splits(kv, B, max_seq_len, window, n_sink), kv->head_dim);
        return sfa::window_decode_launch(p, kv, B, static_cast<hipStream_t>(stream));
    } catch (...) {
        return SFA_ERR_RUNTIME;
    }
}

SFA_API size_t sfa_prefill_window_workspace_bytes(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T,
                                                  int32_t window, int32_t n_sink) {
    (void)kv, (void)q_pos0, (void)T, (void)window, (void)n_sink;
    return 0;
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
        return sfa::window_launch(kv, p, T, static_cast<hipStream_t>(stream));
    } catch (...) {
        return SFA_ERR_RUNTIME;
    }
}

}  // extern "C"
