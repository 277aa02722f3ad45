// sfa_norm_rope.hip - per-head RMS norms of Q and K, the rotation by one
// position or several axes, and the KV append in one pass
// (sfa_norm_rope_kv_append, include/sfa_window.h).
//
//   y = x * 1/sqrt(mean(x^2) + eps) * w;  pair (a, b) -> (a c - b s, a s + b c),
//   (c, s) of the angle p * freq_base^(-2i/n_rot), p the position on pair i's axis
//
// Bound by memory: Q is read and written, K and V read (f32), their rows written.
// A lane owns 8 elements of a head, four whole pairs, so that a rotation
// needs no other lane; the sum of squares joins the HD/8 lanes of a head by DPP.
// A token's angles are computed once, in 64 bits, for all its heads.
// Measured (32 / 8 heads of 128): 8192 tokens into an F32 cache 80 us, 5.0 TB/s
// (a large copy: 5.15); 2048 into F16 17.4 us, 5.3 TB/s; one token 4 us, the
// chain of its position, its page and its row.
#include "sfa_append.h"
#include "sfa_window.h"

namespace sfa {

struct NormRopeParams {
    AppendParams a;  // k, v of AppendParams are not read here: rows have strides
    const float *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    float *q_out;
    const float *q_norm, *k_norm;
    float eps;
    const int32_t *rope_pos;  // [n_axis][n_tok] or null
    int n_head;
    int n_rot, neox, n_axis, interleaved;
    int sec[4];
    double exp_step;  // log2(freq_base) * -2 / n_rot
};

// Axis of pair i (see SFA_AXES_* in sfa_window.h).
__device__ inline int axis_of(const NormRopeParams &p, int i) {
    if (p.n_axis == 1) return 0;
    if (p.interleaved) {
        const int a = i % p.n_axis, turn = i / p.n_axis;
        const int have = a == 1 ? p.sec[1] : a == 2 ? p.sec[2] : p.sec[3];
        return a > 0 && turn < have ? a : 0;
    }
    int a = i >= p.sec[0] ? 1 : 0;
    if (i >= p.sec[0] + p.sec[1]) a = 2;
    if (i >= p.sec[0] + p.sec[1] + p.sec[2]) a = 3;
    return a;
}

// Sum over the N = 4, 8 or 16 neighbouring lanes that share a head, the same
// order in every lane.
template <int N>
__device__ inline float head_sum(float x) {
    x += dpp_row<0xB1>(x);
    x += dpp_row<0x4E>(x);
    if constexpr (N >= 8) x += dpp_row<0x141>(x);
    if constexpr (N >= 16) x += dpp_row<0x140>(x);
    return x;
}

template <int KVT, int HD>
__global__ __launch_bounds__(256) void norm_rope_append_kernel(NormRopeParams p) {
    constexpr int L = HD / 8;          // lanes of a head
    constexpr int RPB = 256 / L;       // heads a pass of the workgroup
    __shared__ float2 cs[HD / 2];
    __shared__ __attribute__((aligned(16))) float kq[KVT == SFA_KV_Q8_0 ? RPB : 1][KVT == SFA_KV_Q8_0 ? HD : 4];
    const int tok = blockIdx.x;
    const int tid = threadIdx.x;
    const int ps = p.a.pos[tok];
    const bool valid = ps >= 0 && p.a.seq[tok] >= 0;  // workgroup-uniform
    if (!valid) return;
    const int half = p.n_rot / 2;
    if (tid < half) {
        // the angle in turns, in 64 bits: a far position's angle has all its
        // digits left after whole turns are taken off
        const int rp = p.rope_pos != nullptr ? p.rope_pos[(int64_t)axis_of(p, tid) * p.a.n_tok + tok] : ps;
        const double turns = (double)rp * exp2((double)tid * p.exp_step) * 0.15915494309189533577;
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        cs[tid] = make_float2(c, s);
    }
    __syncthreads();
    const int l = tid % L, slot = tid / L;
    const int n_q = p.q != nullptr ? p.n_head : 0;
    const int n_rows = n_q + 2 * p.a.n_head_kv;
    // this lane's two chunks of four elements in a rotated head
    const bool rot = 8 * l < p.n_rot;
    const int c0 = rot && p.neox ? 4 * l : 8 * l;
    const int c1 = rot && p.neox ? half + 4 * l : 8 * l + 4;
    for (int r = slot + blockIdx.y * RPB; r < n_rows; r += RPB * gridDim.y) {
        const int what = r < n_q ? 0 : r < n_q + p.a.n_head_kv ? 1 : 2;  // Q, K or V
        const int h = what == 0 ? r : (r - n_q) % p.a.n_head_kv;
        const float *src = what == 0   ? p.q + tok * p.q_stride
                           : what == 1 ? p.k + tok * p.k_stride
                                       : p.v + tok * p.v_stride;
        src += h * HD;
        const int e0 = what == 2 ? 8 * l : c0, e1 = what == 2 ? 8 * l + 4 : c1;
        float x[8];
        const floatx4 a = *reinterpret_cast<const floatx4 *>(src + e0);
        const floatx4 b = *reinterpret_cast<const floatx4 *>(src + e1);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
        const float *w = what == 0 ? p.q_norm : what == 1 ? p.k_norm : nullptr;
        if (w != nullptr) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
            const float sc = 1.0f / sqrtf(head_sum<L>(ss) * (1.0f / HD) + p.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = x[j] * sc * w[e0 + j];
                x[4 + j] = x[4 + j] * sc * w[e1 + j];
            }
        }
        if (what != 2 && rot) {
            if (p.neox) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = cs[4 * l + j];
                    rope_rotate(x[j], x[4 + j], t.x, t.y);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = cs[4 * l + j];
                    rope_rotate(x[2 * j], x[2 * j + 1], t.x, t.y);
                }
            }
        }
        if (what == 0) {
            float *dst = p.q_out + ((int64_t)tok * p.n_head + h) * HD;
            *reinterpret_cast<floatx4 *>(dst + e0) = floatx4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<floatx4 *>(dst + e1) = floatx4{x[4], x[5], x[6], x[7]};
            continue;
        }
        uint8_t *dst = row_ptr(p.a, what - 1, tok, h);
        if (dst == nullptr) continue;  // the same for all lanes of the head
        if constexpr (KVT == SFA_KV_F32) {
            float *d = reinterpret_cast<float *>(dst);
            *reinterpret_cast<floatx4 *>(d + e0) = floatx4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<floatx4 *>(d + e1) = floatx4{x[4], x[5], x[6], x[7]};
        } else if constexpr (KVT == SFA_KV_F16) {
            half4 u, v;
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = (_Float16)x[j], v[j] = (_Float16)x[4 + j];
            _Float16 *d = reinterpret_cast<_Float16 *>(dst);
            *reinterpret_cast<half4 *>(d + e0) = u;
            *reinterpret_cast<half4 *>(d + e1) = v;
        } else {
            // back to 8 neighbouring elements a lane: a quantisation block is
            // four lanes' then
            float *row = kq[slot];
            *reinterpret_cast<floatx4 *>(row + e0) = floatx4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<floatx4 *>(row + e1) = floatx4{x[4], x[5], x[6], x[7]};
            __builtin_amdgcn_wave_barrier();
            const floatx4 u = *reinterpret_cast<const floatx4 *>(row + 8 * l);
            const floatx4 v = *reinterpret_cast<const floatx4 *>(row + 8 * l + 4);
            __builtin_amdgcn_wave_barrier();
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(u[j]), fabsf(v[j])));
            amax = fmaxf(amax, dpp_row<0xB1>(amax));
            amax = fmaxf(amax, dpp_row<0x4E>(amax));
            // quantize_row_q8_0: d = amax / 127 stored in f16, q = round(x * (1 / d))
            const float d = amax / 127.0f;
            const float id = d != 0.0f ? 1.0f / d : 0.0f;
            uint16_t *blk = reinterpret_cast<uint16_t *>(dst + l / 4 * kQ8Bytes);
            if (l % 4 == 0) blk[0] = __builtin_bit_cast(uint16_t, (_Float16)d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y0 = j < 2 ? u[2 * j] : v[2 * j - 4], y1 = j < 2 ? u[2 * j + 1] : v[2 * j - 3];
                const int q0 = (int)roundf(y0 * id), q1 = (int)roundf(y1 * id);
                blk[1 + l % 4 * 4 + j] = (uint16_t)((q0 & 0xff) | ((q1 & 0xff) << 8));
            }
        }
    }
}

static int rope_check(const sfa_rope_desc *r, int head_dim) {
    if (r == nullptr || head_dim <= 0) return SFA_ERR_INVALID_ARGUMENT;
    if (r->n_rot <= 0 || r->n_rot > head_dim) return SFA_ERR_INVALID_ARGUMENT;
    if (r->n_rot % 8 != 0) return SFA_ERR_UNSUPPORTED;
    if (r->pairing != SFA_ROPE_NORMAL && r->pairing != SFA_ROPE_NEOX) return SFA_ERR_INVALID_ARGUMENT;
    if (!(r->freq_base > 0.0f) || !__builtin_isfinite(r->freq_base)) return SFA_ERR_INVALID_ARGUMENT;
    if (r->n_axis < 1 || r->n_axis > 4) return SFA_ERR_INVALID_ARGUMENT;
    if (r->n_axis == 1) return SFA_OK;
    if (r->layout != SFA_AXES_BLOCKS && r->layout != SFA_AXES_INTERLEAVED) return SFA_ERR_INVALID_ARGUMENT;
    int64_t sum = 0;
    for (int a = 0; a < r->n_axis; ++a) {
        if (r->sections[a] < 0) return SFA_ERR_INVALID_ARGUMENT;
        sum += r->sections[a];
        // dealt in turn, the axis's last pair must exist
        if (r->layout == SFA_AXES_INTERLEAVED && a > 0 && r->sections[a] > 0 &&
            ((int64_t)r->sections[a] - 1) * r->n_axis + a >= r->n_rot / 2)
            return SFA_ERR_INVALID_ARGUMENT;
    }
    return sum == r->n_rot / 2 ? SFA_OK : SFA_ERR_INVALID_ARGUMENT;
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int KVT>
static int launch_hd(const NormRopeParams &p, hipStream_t s) {
    // up to 512 tokens: a workgroup for every 256 lanes' heads, each with its own
    // table of angles, instead of a loop over them (F16, 32 / 8 heads of 128: 4.5 ->
    // 3.5 us for one token, 5.5 -> 4.6 for 256, 6.4 -> 6.2 for 512; 1024 10.9 -> 11.2)
    const int rows = (p.q != nullptr ? p.n_head : 0) + 2 * p.a.n_head_kv, pass = 2048 / p.a.head_dim;
    const dim3 grid((unsigned)p.a.n_tok, p.a.n_tok <= 512 ? (unsigned)((rows + pass - 1) / pass) : 1u), block(256);
    if (p.a.head_dim == 128) hipLaunchKernelGGL((norm_rope_append_kernel<KVT, 128>), grid, block, 0, s, p);
    else if (p.a.head_dim == 64) hipLaunchKernelGGL((norm_rope_append_kernel<KVT, 64>), grid, block, 0, s, p);
    else if constexpr (KVT != SFA_KV_Q8_0) hipLaunchKernelGGL((norm_rope_append_kernel<KVT, 32>), grid, block, 0, s, p);
    else return SFA_ERR_UNSUPPORTED;
    return hipGetLastError() == hipSuccess ? SFA_OK : SFA_ERR_RUNTIME;
}

static int norm_rope_launch(const sfa_kv_desc *kv, const sfa_rope_desc *rope, const float *q, int64_t q_stride,
                            float *q_out, const float *k, int64_t k_stride, const float *v, int64_t v_stride,
                            const float *q_norm, const float *k_norm, float eps, const int32_t *seq,
                            const int32_t *pos, const int32_t *rope_pos, int32_t n_tok,
                            const int32_t *page_table, int32_t max_pages, hipStream_t stream) {
    if (n_tok < 0 || max_pages <= 0) return SFA_ERR_INVALID_ARGUMENT;
    if (!(eps >= 0.0f) || !__builtin_isfinite(eps)) return SFA_ERR_INVALID_ARGUMENT;
    if (n_tok == 0) return SFA_OK;
    if (k == nullptr || v == nullptr || seq == nullptr || pos == nullptr || page_table == nullptr)
        return SFA_ERR_INVALID_ARGUMENT;
    if ((q == nullptr) != (q_out == nullptr)) return SFA_ERR_INVALID_ARGUMENT;
    const int64_t nq = (int64_t)kv->n_head * kv->head_dim, nk = (int64_t)kv->n_head_kv * kv->head_dim;
    if (n_tok == 1) {
        q_stride = nq;
        k_stride = v_stride = nk;
    }
    if ((q != nullptr && q_stride < nq) || k_stride < nk || v_stride < nk) return SFA_ERR_INVALID_ARGUMENT;
    if (q != nullptr && q == q_out && q_stride != nq) return SFA_ERR_INVALID_ARGUMENT;
    if ((q != nullptr && q_stride % 4 != 0) || k_stride % 4 != 0 || v_stride % 4 != 0) return SFA_ERR_UNSUPPORTED;
    if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v)) return SFA_ERR_UNSUPPORTED;
    NormRopeParams p{};
    p.a.k_pages = static_cast<uint8_t *>(kv->k_pages);
    p.a.v_pages = static_cast<uint8_t *>(kv->v_pages);
    p.a.k_cold = static_cast<uint8_t *>(kv->k_cold);
    p.a.v_cold = static_cast<uint8_t *>(kv->v_cold);
    p.a.row_bytes = row_bytes_of(kv->kv_type, kv->head_dim);
    p.a.page_bytes = (int64_t)p.a.row_bytes * kv->n_head_kv * kv->page_size;
    p.a.n_pages = kv->n_pages;
    p.a.n_cold = kv->n_cold_pages;
    p.a.page_size = kv->page_size;
    p.a.n_head_kv = kv->n_head_kv;
    p.a.head_dim = kv->head_dim;
    p.a.seq = seq;
    p.a.pos = pos;
    p.a.n_tok = n_tok;
    p.a.page_table = page_table;
    p.a.max_pages = max_pages;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_out = q_out;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.eps = eps;
    p.rope_pos = rope_pos;
    p.n_head = kv->n_head;
    p.n_rot = rope->n_rot;
    p.neox = rope->pairing == SFA_ROPE_NEOX;
    p.n_axis = rope->n_axis;
    p.interleaved = rope->layout == SFA_AXES_INTERLEAVED;
    for (int a = 0; a < rope->n_axis; ++a) p.sec[a] = rope->sections[a];
    p.exp_step = -2.0 / rope->n_rot * log2((double)rope->freq_base);
    switch (kv->kv_type) {
    case SFA_KV_F32: return launch_hd<SFA_KV_F32>(p, stream);
    case SFA_KV_F16: return launch_hd<SFA_KV_F16>(p, stream);
    case SFA_KV_Q8_0: return launch_hd<SFA_KV_Q8_0>(p, stream);
    default: return SFA_ERR_UNSUPPORTED;
    }
}

}  // namespace sfa

extern "C" {

SFA_API int sfa_rope_desc_check(const sfa_rope_desc *rope, int32_t head_dim) {
    return sfa::rope_check(rope, head_dim);
}

SFA_API int sfa_norm_rope_kv_append(const sfa_kv_desc *kv, const sfa_rope_desc *rope, const float *q,
                                    int64_t q_stride, float *q_out, const float *k, int64_t k_stride,
                                    const float *v, int64_t v_stride, const float *q_norm,
                                    const float *k_norm, float eps, const int32_t *seq,
                                    const int32_t *pos, const int32_t *rope_pos, int32_t n_tok,
                                    const int32_t *page_table, int32_t max_pages, void *stream) {
    try {
        int rc = sfa_kv_desc_check(kv);
        if (rc != SFA_OK) return rc;
        rc = sfa::rope_check(rope, kv->head_dim);
        if (rc != SFA_OK) return rc;
        return sfa::norm_rope_launch(kv, rope, q, q_stride, q_out, k, k_stride, v, v_stride, q_norm, k_norm, eps,
                                     seq, pos, rope_pos, n_tok, page_table, max_pages,
                                     static_cast<hipStream_t>(stream));
    } catch (...) {
        return SFA_ERR_RUNTIME;
    }
}

}  // extern "C"
