// sfa_window_prefill.hip - a prompt chunk over a sliding window and the sinks,
// a window for every token (sfa_attn_prefill_window, include/sfa_window.h).
//
// Bound by the matrix cores.  A workgroup takes 128 rows of one kv head (its G
// query heads of 128 / G tokens), 32 a wave, and the tiles that any of them
// sees: those of the sinks before the window, then the window's.  K and V tiles
// come into LDS once for the four waves, the next tile under way while one is
// computed.  S^T = K Q^T and O^T = V^T P^T on 32x32 matrix instructions: lane l
// holds the row l % 32 of both products, so scores become operands in place.
//
// Q and P keep 32 bits (see sfa_window_decode.hip): twice the products of
// a kernel that rounds them to 16, on the same tile reads.
//
// Chunks of few rows leave CUs idle: their tiles are split over workgroups,
// whose records window_merge_kernel joins.
#include "sfa_window_dev.h"

namespace sfa {

constexpr int kRows = 128;  // of a workgroup

template <int KVT, int HD>
struct PTile {
    static constexpr int TP = KVT == SFA_KV_F32 ? 32 : 64;           // positions
    static constexpr int ROW = KVT == SFA_KV_F32 ? HD * 4 : HD * 2;  // a row in LDS (Q8_0: its quants as f16)
    static constexpr int RB = KVT == SFA_KV_Q8_0 ? HD / kQK * kQ8Bytes : ROW;
    static constexpr int CPR = ROW / 16;
    static constexpr int BYTES = TP * ROW;
    static constexpr int NI = BYTES / 4096;  // load instructions of a wave, a tensor
    static constexpr int RP = 256 / ROW > 0 ? 256 / ROW : 1;  // rows under all LDS banks
    static constexpr int NG = ROW / 64 > 0 ? ROW / 64 : 1;
};

// Where chunk j of row r lies in its LDS row: K's reads are 16 rows at one
// chunk, V's four rows at 64 neighbouring bytes (F32: two rows at 128).
template <int KVT, int HD>
__device__ inline int pk_slot(int r, int j) {
    using T = PTile<KVT, HD>;
    return j ^ (r / T::RP % (T::CPR < 16 ? T::CPR : 16));
}
template <int KVT, int HD>
__device__ inline int pv_slot(int r, int j) {
    using T = PTile<KVT, HD>;
    if constexpr (KVT == SFA_KV_F32) return j ^ (r / 4 % 2 * (T::CPR >= 16 ? 8 : 0));
    return j ^ (r / T::RP % T::NG * 4);
}

// Runs the N steps of a product loop with the operand reads AHEAD steps before
// their use; left to itself the compiler waits for every operand right before
// it is used.  Vector and scalar arithmetic may move over the fences, reads and
// matrix instructions may not.
template <int N, int AHEAD, typename Read, typename Use>
__device__ inline void pipelined(Read read, Use use) {
    decltype(read(0)) a[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD && i < N; ++i) a[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const auto now = a[i % AHEAD];
        if (i + AHEAD < N) a[i % AHEAD] = read(i + AHEAD);
        __builtin_amdgcn_sched_barrier(0x406);
        use(i, now);
        __builtin_amdgcn_sched_barrier(0x406);
    }
}

template <int KVT, int HD, int G>
__global__ __launch_bounds__(256, 2) void window_prefill_kernel(WindowParams p) {
    using T = PTile<KVT, HD>;
    constexpr int TP = T::TP, PB = TP / 32;  // 32-position blocks of a tile
    constexpr int DB = HD / 32;
    constexpr int KC = HD / 16;              // 16-dim steps of a score (F32: pairs of 4-float chunks are 2 KC)
    constexpr int NB = HD / kQK;
    constexpr bool kQ8 = KVT == SFA_KV_Q8_0, kF32 = KVT == SFA_KV_F32;
    constexpr int BUFS = kQ8 ? 1 : 2;        // Q8_0 tiles wait in registers
    constexpr int SETS = kQ8 ? 3 : 2;        // K, V; Q8_0: K, V's two halves
    __shared__ __attribute__((aligned(256))) uint8_t lds[BUFS][SETS][T::BYTES];
    __shared__ __attribute__((aligned(16))) float k_scale[kQ8 ? NB : 1][kQ8 ? TP : 4];
    __shared__ int v_exp[4];                 // Q8_0: exponent of each 16 positions' largest V scale
    // values that are not finite, held as zeros: Q8_0: the units of a wave whose
    // scale is not; else whether a wave's quarter of the tile has any, and a bit
    // for each value of a chunk
    __shared__ uint64_t v_bad[2][4];
    __shared__ uint8_t v_bits[2][kQ8 ? 4 : TP * T::CPR];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5;
    // Workgroups go round the eight XCDs: with Hkv a multiple of 8 a kv head's
    // tiles stay in one L2.  The last rows, which see the most, come first.
    const int kvh = blockIdx.x, split = blockIdx.y, blk = gridDim.z - 1 - blockIdx.z;

    const int row = blk * kRows + wave * 32 + n;  // token row / G, head row % G of the group
    const bool row_ok = row < p.n_tok * G;
    const int tok = row_ok ? row / G : p.n_tok - 1;
    const int head = kvh * G + row % G;
    const int tpos = p.q_pos0 + tok;
    const bool wave_ok = blk * kRows + wave * 32 < p.n_tok * G;

    // the workgroup's span: sinks before the window [0, ns), then [lo, hi]
    const int tok0 = blk * kRows / G, tok1 = min((blk * kRows + kRows - 1) / G, p.n_tok - 1);
    const int64_t cap = (int64_t)p.max_pages * p.page_size;
    const int first = p.q_pos0 + tok0, last = p.q_pos0 + tok1;
    const int lo = first - p.window + 1 > 0 ? first - p.window + 1 : 0;
    const int hi = last < cap ? last : (int)(cap - 1);
    const int ns = min(min(p.n_sink, lo), hi + 1);
    const int sink_tiles = (ns + TP - 1) / TP;
    const int n_tiles = sink_tiles + (hi >= lo ? hi / TP - lo / TP + 1 : 0);
    // (the divisions run on the vector side: back to scalars, for scalar branches)
    const int t0 = (int)to_scalar((uint32_t)((uint64_t)n_tiles * split / p.n_split));
    const int t1 = (int)to_scalar((uint32_t)((uint64_t)n_tiles * (split + 1) / p.n_split));

    PageWindow pages;
    if (t0 < t1)
        pages.load(p.page_table, p.max_pages, (t0 < sink_tiles ? t0 : lo / TP + t0 - sink_tiles) * TP / p.page_size, lane);

    // Q of this lane's row: dims 16 c + 8 hh + j (F32: 16 c + 4 hh + j and 16 c + 8 + 4 hh + j)
    const float *const qr = p.q + ((int64_t)tok * p.n_head + head) * HD;
    float up = 1.0f;
    half8 qh[kF32 ? 1 : KC], ql[kF32 ? 1 : KC];
    float qf[kF32 ? KC : 1][8];
    {
        float qx[KC][8];
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int d0 = kF32 ? 16 * c + 4 * hh : 16 * c + 8 * hh, d1 = kF32 ? d0 + 8 : d0 + 4;
            const floatx4 u = *reinterpret_cast<const floatx4 *>(qr + d0);
            const floatx4 v = *reinterpret_cast<const floatx4 *>(qr + d1);
#pragma unroll
            for (int j = 0; j < 4; ++j) qx[c][j] = u[j], qx[c][4 + j] = v[j];
        }
        if constexpr (kF32) {
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) qf[c][j] = qx[c][j];
        } else {
            float amax = 0.0f, a, b, down;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[c][j]));
            swap_halves(amax, a, b);
            row_exponent(fmaxf(a, b), down, up);
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 h, l;
                    split_f16(qx[c][j] * down, h, l);
                    qh[c][j] = h;
                    ql[c][j] = l;
                }
        }
    }
    const float f = p.scale_log2 * up;

    const int col_bytes = p.n_head_kv * T::RB;
    // F16 and F32: this wave's quarter of a tile, lane by lane
    int k_off[T::NI], v_off[T::NI];
    if constexpr (!kQ8) {
#pragma unroll
        for (int i = 0; i < T::NI; ++i) {
            const int ch = (T::NI * wave + i) * 64 + lane, r = ch / T::CPR, j = ch % T::CPR;
            k_off[i] = r * col_bytes + 16 * pk_slot<KVT, HD>(r, j);
            v_off[i] = r * col_bytes + 16 * pv_slot<KVT, HD>(r, j);
        }
    }
    // Q8_0: units of one block; with HD 128 a thread has one of K and one of V,
    // with HD 64 the first two waves have K's and the others V's
    constexpr int UN = kQ8 ? NB / 2 : 1;
    const int unit = NB == 4 ? threadIdx.x : threadIdx.x & 127;
    const int u_row = unit / NB, u_blk = unit % NB;
    uint32_t raw[UN][9];

    struct Src {
        int first, from, to;  // position of the tile's row 0, and the rows that any token sees
        bool sink, there;
    };
    auto issue = [&](int t, int buf) {
        Src s;
        s.sink = t < sink_tiles;
        s.first = (s.sink ? t : lo / TP + t - sink_tiles) * TP;
        s.from = max(s.sink ? 0 : lo - s.first, 0);
        s.to = min((s.sink ? ns : hi + 1) - s.first, TP);
        const int lp = (int)to_scalar((uint32_t)s.first / (uint32_t)p.page_size);
        const int32_t id = pages.get(p.page_table, p.max_pages, lp, lane);
        const uint8_t *kb = page_base(id, p.k_pages, p.n_pages, p.k_cold, p.n_cold, p.page_bytes);
        const uint8_t *vb = page_base(id, p.v_pages, p.n_pages, p.v_cold, p.n_cold, p.page_bytes);
        s.there = kb != nullptr && vb != nullptr;
        const int64_t at = (int64_t)(s.first - lp * p.page_size + s.from) * col_bytes + kvh * T::RB;
        const int bytes = s.there ? (s.to - s.from - 1) * col_bytes + T::RB : 0;
        const int back = s.from * col_bytes;
        if constexpr (kQ8) {
            // nine words from the block's first multiple of 4
            const int off = u_row * col_bytes + kQ8Bytes * u_blk - 2 * (u_blk & 1) - back;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const auto r = buffer_of(s.there ? ((UN == 2 ? u == 0 : wave < 2) ? kb : vb) + at : nullptr, bytes);
                const intx4 a = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
                const intx4 b = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 16, 0));
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[u][i] = a[i], raw[u][4 + i] = b[i];
                raw[u][8] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 32, 0);
            }
        } else {
            const auto kr = buffer_of(s.there ? kb + at : nullptr, bytes);
            const auto vr = buffer_of(s.there ? vb + at : nullptr, bytes);
            const uint32_t to = lds_addr(lds[buf][0]) + 1024 * T::NI * wave;
#pragma unroll
            for (int i = 0; i < T::NI; ++i) load_to_lds(kr, to + 1024 * i, k_off[i] - back);
#pragma unroll
            for (int i = 0; i < T::NI; ++i) load_to_lds(vr, to + T::BYTES + 1024 * i, v_off[i] - back);
        }
        return s;
    };
    // Q8_0: a block from registers to LDS: K's quants as f16 and their scale
    // beside them; V's values, under the power of two of the largest scale of
    // the wave's rows, as two f16
    auto stage = [&]() {
        if constexpr (kQ8) {
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const bool is_v = UN == 2 ? u == 1 : wave >= 2;
                uint32_t w[9];
#pragma unroll
                for (int i = 0; i < 9; ++i) w[i] = raw[u][i];
                const bool odd = u_blk & 1;  // d in the upper half of the first word, quants from the second on
                float d = (float)__builtin_bit_cast(_Float16, (uint16_t)(odd ? w[0] >> 16 : w[0]));
                uint32_t qw[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    qw[i] = odd ? w[i + 1] : __builtin_amdgcn_alignbyte(w[i + 1], w[i], 2);
                if (is_v) {
                    const bool bad = !(fabsf(d) < INFINITY);
                    d = bad ? 0.0f : d;
                    const uint64_t bads = __ballot(bad);
                    const float big = wave_max(fabsf(d));
                    const int e = max((int)(__builtin_bit_cast(uint32_t, big) >> 23), 1);
                    if (lane == 0) {
                        v_bad[0][wave] = bads;
                        if constexpr (NB == 4) v_exp[wave] = e;
                        else v_exp[2 * (wave - 2)] = v_exp[2 * (wave - 2) + 1] = e;
                    }
                    const float x = __builtin_amdgcn_ldexpf(d, 127 - e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        half8 h, l;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int q = (int)(int8_t)(qw[2 * i + j / 4] >> 8 * (j % 4));
                            _Float16 a, b;
                            split_f16(x * (float)q, a, b);
                            h[j] = a;
                            l[j] = b;
                        }
                        const int at = u_row * T::ROW + 16 * pv_slot<KVT, HD>(u_row, 4 * u_blk + i);
                        *reinterpret_cast<half8 *>(&lds[0][1][at]) = h;
                        *reinterpret_cast<half8 *>(&lds[0][SETS - 1][at]) = l;
                    }
                } else {
                    k_scale[u_blk][u_row] = d;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        half8 h;
#pragma unroll
                        for (int j = 0; j < 8; ++j) h[j] = (_Float16)(int)(int8_t)(qw[2 * i + j / 4] >> 8 * (j % 4));
                        *reinterpret_cast<half8 *>(&lds[0][0][u_row * T::ROW + 16 * pk_slot<KVT, HD>(u_row, 4 * u_blk + i)]) = h;
                    }
                }
            }
        }
    };

    // probabilities are 2^(s f - base), base kSplitShift below the row's running
    // maximum (F32: at it); l sums this lane's
    constexpr float SHIFT = kF32 ? 0.0f : (float)kSplitShift;
    float base = -INFINITY, l = 0.0f;
    int unit_exp = 1;  // Q8_0: o is in units of 2^(unit_exp - 127), the largest V scale's so far
    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    Src src = {}, next = {};
    if (t0 < t1) src = issue(t0, 0);
    int buf = 0;
    for (int t = t0; t < t1; ++t, buf ^= BUFS - 1, src = next) {
        // masked where a row of the workgroup does not see the whole tile
        const int end = src.first + TP - 1;
        const bool masked = (src.from > 0) | (src.to < TP) |
                            (!src.sink & ((end > first) | ((src.first <= last - p.window) & (end >= p.n_sink))));
        if constexpr (kQ8) {
            __syncthreads();  // the last tile has been read
            stage();
            if (t + 1 < t1) next = issue(t + 1, 0);
            __syncthreads();
        } else {
            wait_loads<0>();
            // a value that is not finite would reach rows that do not see it, as
            // 0 times it: the wave looks its quarter of V over
            if (masked) {
                bool any = false;
#pragma unroll
                for (int i = 0; i < T::NI; ++i) {
                    const int ch = (T::NI * wave + i) * 64 + lane;
                    intx4 *const at = reinterpret_cast<intx4 *>(&lds[buf][1][16 * ch]);
                    intx4 x = *at;
                    uint32_t bits = 0;
#pragma unroll
                    for (int j = 0; j < (kF32 ? 4 : 8); ++j) {
                        const uint32_t e = kF32 ? (uint32_t)x[j & 3] >> 23 & 255 : (uint32_t)x[j / 2] >> (j % 2 ? 26 : 10) & 31;
                        bits |= (e == (kF32 ? 255u : 31u) ? 1u : 0u) << j;
                    }
                    if (bits != 0) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (kF32) x[j] = bits >> j & 1 ? 0 : x[j];
                            else x[j] &= (bits >> 2 * j & 1 ? 0 : 0xffff) | (bits >> (2 * j + 1) & 1 ? 0 : (int)0xffff0000);
                        }
                        *at = x;
                        any = true;
                    }
                    v_bits[buf][ch] = (uint8_t)bits;
                }
                const uint64_t who = __ballot(any);
                if (lane == 0) v_bad[buf][wave] = who;
            }
            __syncthreads();  // this tile is there, and the other buffer has been read
            if (t + 1 < t1) next = issue(t + 1, buf ^ 1);
        }
        if (!wave_ok || !src.there) continue;
        const uint8_t *const kt = lds[kQ8 ? 0 : buf][0], *const vt = lds[kQ8 ? 0 : buf][1];
        // This lane's first operand addresses; a step's are these with its chunk
        // XORed in (the slots are XORs too) and its rows added.  The empty asm
        // keeps the compiler from holding every step's address over the loop.
        int k_at = n * T::ROW + 16 * pk_slot<KVT, HD>(n, hh), v_at0 = 0;
        const int li = lane & 15;
        if constexpr (kF32) {
            v_at0 = 4 * hh * T::ROW + 16 * pv_slot<KVT, HD>(4 * hh, n / 4) + 4 * (n & 3);
        } else {
            const int r = 4 * hh + (li >> 2);
            v_at0 = r * T::ROW + 16 * pv_slot<KVT, HD>(r, 2 * (lane >> 4 & 1) + ((li & 3) >> 1)) + 8 * (li & 1);
        }
        asm("" : "+v"(k_at), "+v"(v_at0));

        floatx16 s[PB];
#pragma unroll
        for (int b = 0; b < PB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
        if constexpr (kF32) {
            pipelined<2 * KC, 3>([&](int c) { return *reinterpret_cast<const floatx4 *>(kt + (k_at ^ (32 * c))); },
                                 [&](int c, floatx4 a) {
#pragma unroll
                                     for (int i = 0; i < 4; ++i)
                                         s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], qf[c / 2][c % 2 * 4 + i], s[0], 0, 0, 0);
                                 });
        } else if constexpr (!kQ8) {
            pipelined<KC * PB, 3>(
                [&](int i) {
                    return *reinterpret_cast<const half8 *>(kt + (k_at ^ (32 * (i / PB))) + i % PB * 32 * T::ROW);
                },
                [&](int i, half8 a) {
                    const int c = i / PB, b = i % PB;
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], s[b], 0, 0, 0);
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], s[b], 0, 0, 0);
                });
        } else {
            // two steps a block, then the block's scales
            floatx16 x;
            pipelined<KC * PB, 3>(
                [&](int i) {
                    const int b = i / 2 % PB, c = i / (2 * PB) * 2 + i % 2;
                    return *reinterpret_cast<const half8 *>(kt + (k_at ^ (32 * c)) + b * 32 * T::ROW);
                },
                [&](int i, half8 a) {
                    const int b = i / 2 % PB, nb = i / (2 * PB), c = 2 * nb + i % 2;
                    if (i % 2 == 0)
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = 0.0f;
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], x, 0, 0, 0);
                    if (i % 2 == 0) return;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const floatx4 d = *reinterpret_cast<const floatx4 *>(&k_scale[nb][32 * b + 8 * i4 + 4 * hh]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[b][4 * i4 + j] = fmaf(x[4 * i4 + j], d[j], s[b][4 * i4 + j]);
                    }
                });
        }

        if (masked) {
#pragma unroll
            for (int i = 0; i < 16 * PB; ++i) {
                const int r = i / 16 * 32 + i / 4 % 4 * 8 + 4 * hh + i % 4, pos = src.first + r;
                const bool see = (r >= src.from) & (r < src.to) & (pos <= tpos) & (src.sink | (pos > tpos - p.window) | (pos < p.n_sink));
                s[i / 16][i % 16] = see ? s[i / 16][i % 16] : -INFINITY;
            }
        }
        float mx = -INFINITY, ma, mb;
#pragma unroll
        for (int b = 0; b < PB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
        swap_halves(mx, ma, mb);
        mx = fmaxf(ma, mb) * f - SHIFT;
        if (__ballot(mx > base) != 0) {
            const float nb = fmaxf(mx, base);
            const float a = nb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - nb);
            l *= a;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= a;
            base = nb;
        }
        const float sub = base == -INFINITY ? 0.0f : base;
#pragma unroll
        for (int b = 0; b < PB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], f, -sub));
                l += s[b][i];
            }

        // A value that is not finite, in a position that some rows may not see:
        // the products take it as zero; the rows that see it get what it comes
        // to, NaN.
        auto spoil = [&]() {
            for (int r = src.from; r < src.to; ++r) {
                const int pos = src.first + r;
                const bool see = (pos <= tpos) & (src.sink | (pos > tpos - p.window) | (pos < p.n_sink));
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    if constexpr (kQ8) {
                        const int u = r * NB + d;  // its unit, NB / 2 * 128 of them in the waves that hold V
                        const bool bad = v_bad[0][(NB == 4 ? 0 : 2) + u / 64] >> u % 64 & 1;
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] = bad && see ? NAN : o[d][i];
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = 32 * d + i / 4 * 8 + 4 * hh + i % 4;  // the dim of o[d][i]
                        constexpr int PC = kF32 ? 4 : 8;                    // values of a chunk
                        const bool bad = v_bits[buf][r * T::CPR + pv_slot<KVT, HD>(r, e / PC)] >> e % PC & 1;
                        o[d][i] = (bad & see) ? NAN : o[d][i];
                    }
                }
            }
        };
        if constexpr (kF32) {
            // rows 8 (i / 4) + 4 hh + i % 4: the slots of all are those of row 4 hh
            pipelined<16 * DB, 4>(
                [&](int i) { return *reinterpret_cast<const float *>(vt + (v_at0 ^ (128 * (i % DB))) + (i / DB / 4 * 8 + i / DB % 4) * T::ROW); },
                [&](int i, float a) { o[i % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[0][i / DB], o[i % DB], 0, 0, 0); });
        } else {
            constexpr int ST = TP / 16;  // 16-position steps
            float w16[ST];
            if constexpr (kQ8) {
                int e = unit_exp;
#pragma unroll
                for (int st = 0; st < ST; ++st) e = max(e, __builtin_amdgcn_readfirstlane(v_exp[st]));
                if (e > unit_exp) {
                    const float a = __builtin_amdgcn_ldexpf(1.0f, unit_exp - e);
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] *= a;
                    unit_exp = e;
                }
#pragma unroll
                for (int st = 0; st < ST; ++st)
                    w16[st] = __builtin_amdgcn_ldexpf(1.0f, __builtin_amdgcn_readfirstlane(v_exp[st]) - unit_exp);
            }
            half8 ph[ST], pl[ST];
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 a, b;
                    split_f16(kQ8 ? s[st / 2][st % 2 * 8 + j] * w16[st] : s[st / 2][st % 2 * 8 + j], a, b);
                    ph[st][j] = a;
                    pl[st][j] = b;
                }
            // operand of step st: positions 16 st + 4 hh .. and 16 st + 8 + 4 hh .., the lane's own
            // scores; four values a read, lane i of 16 gets dim i of the four rows its group names
            auto v_at = [&](const uint8_t *tile, int st, int d) {
                const uint8_t *const at = tile + (v_at0 ^ (64 * d)) + 16 * st * T::ROW;
                const half4 x = tr16_read(at), y = tr16_read(at + 8 * T::ROW);
                return half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            };
            pipelined<ST * DB, 3>([&](int i) { return v_at(vt, i / DB, i % DB); },
                                  [&](int i, half8 a) {
                                      const int st = i / DB, d = i % DB;
                                      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[st], o[d], 0, 0, 0);
                                      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[st], o[d], 0, 0, 0);
                                      if constexpr (kQ8) {
                                          const half8 b = v_at(lds[0][SETS - 1], st, d);
                                          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b, ph[st], o[d], 0, 0, 0);
                                      }
                                  });
        }
        if (kQ8 || masked) {
            const uint64_t *const vb = v_bad[buf];
            const uint64_t any = kQ8 && NB == 2 ? vb[2] | vb[3] : vb[0] | vb[1] | vb[2] | vb[3];
            if (__ballot(any != 0) != 0) spoil();
        }
    }
    if (!row_ok) return;
    float la, lb;
    swap_halves(l, la, lb);
    l = la + lb;
    float w = p.n_split > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (kQ8) w = w == 0.0f ? 0.0f : w * __builtin_amdgcn_ldexpf(1.0f, unit_exp - 127);
    const int64_t out_row = (int64_t)tok * p.n_head + head;
    float *const dst = p.n_split > 1 ? p.rec_o + (out_row * p.n_split + split) * HD : p.out + out_row * HD;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            floatx4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = o[d][4 * i4 + i] * w;
            *reinterpret_cast<floatx4 *>(dst + 32 * d + 8 * i4 + 4 * hh) = x;
        }
    if (p.n_split > 1 && hh == 0) p.rec_ml[out_row * p.n_split + split] = make_float2(base, l);
}

// Workgroups that share a row block's tiles: as many as fill the chip's CUs
// twice, at most one per two tiles of the block's span.
int window_prefill_splits(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T, int32_t window, int32_t n_sink) {
    const int tp = kv->kv_type == SFA_KV_F32 ? 32 : 64, g = kv->n_head / kv->n_head_kv;
    const int64_t blocks = ((int64_t)T * g + kRows - 1) / kRows, span = (int64_t)window + kRows / g + n_sink;
    const int64_t end = (int64_t)q_pos0 + T, tiles = ((span < end ? span : end) + tp - 1) / tp;
    int64_t n = 512 / (blocks * kv->n_head_kv);
    if (n > tiles / 2) n = tiles / 2;
    return n < 1 ? 1 : (int)n;
}

template <int KVT, int HD>
static void launch_g(const WindowParams &p, dim3 grid, hipStream_t s) {
    const dim3 block(256);
    switch (p.n_head / p.n_head_kv) {
    case 1: hipLaunchKernelGGL((window_prefill_kernel<KVT, HD, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((window_prefill_kernel<KVT, HD, 2>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((window_prefill_kernel<KVT, HD, 4>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((window_prefill_kernel<KVT, HD, 8>), grid, block, 0, s, p); break;
    }
}

template <int KVT>
static int launch_hd(const WindowParams &p, int head_dim, dim3 grid, hipStream_t s) {
    if (head_dim == 128) launch_g<KVT, 128>(p, grid, s);
    else if (head_dim == 64) launch_g<KVT, 64>(p, grid, s);
    else if constexpr (KVT != SFA_KV_Q8_0) launch_g<KVT, 32>(p, grid, s);
    else return SFA_ERR_UNSUPPORTED;
    return hipGetLastError() == hipSuccess ? SFA_OK : SFA_ERR_RUNTIME;
}

int window_prefill_launch(const WindowParams &p, const sfa_kv_desc *kv, hipStream_t s) {
    const int64_t rows = (int64_t)p.n_tok * kv->n_head;
    const int64_t blocks = ((int64_t)p.n_tok * (kv->n_head / kv->n_head_kv) + kRows - 1) / kRows;
    if (blocks > 65535 || rows > INT32_MAX) return SFA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)kv->n_head_kv, (unsigned)p.n_split, (unsigned)blocks);
    int rc;
    switch (kv->kv_type) {
    case SFA_KV_F32: rc = launch_hd<SFA_KV_F32>(p, kv->head_dim, grid, s); break;
    case SFA_KV_F16: rc = launch_hd<SFA_KV_F16>(p, kv->head_dim, grid, s); break;
    case SFA_KV_Q8_0: rc = launch_hd<SFA_KV_Q8_0>(p, kv->head_dim, grid, s); break;
    default: return SFA_ERR_UNSUPPORTED;
    }
    if (rc != SFA_OK || p.n_split == 1) return rc;
    return window_merge_launch(p, kv->head_dim, rows, s);
}

}  // namespace sfa
