// sfa_window_decode.hip - one new token per sequence over a sliding window and
// the sinks (sfa_attn_decode_window, include/sfa_window.h).
//
// Bound by memory: a sequence's visible K and V rows are read once.  They are
// cut into tiles of 4 KB to 8 KB a tensor; a wave streams its tiles through
// LDS of its own, with the running maximum and sum of the softmax.  The next
// K is under way from the end of the first product on and the next V from the
// end of the second, so that one buffer each does and LDS has room for twice
// the waves that two would leave (Q8_0, 8 sequences, window 8192, with append
// and merge: 48.0 -> 45.5 us; one F16 token 11.9 -> 11.5).  The waves of a
// workgroup, then the workgroups of a sequence (the merge kernel), join their
// (maximum, sum, output).
//
// Measured (32 / 8 heads of 128): F16, 64 sequences, window 4096: 185 us, 5.8
// TB/s.  Q8_0, 8 sequences, window 8192: 34.6 us of kernel, 4.0 TB/s; its loads
// alone take 30 (rows of 136 bytes), its arithmetic alone 26.
//
// S^T = K Q^T and O^T = V^T P^T on 16x16 matrix instructions: their 16 columns
// are the G query heads of a kv head, and lane l holds column l % 16 of both,
// so that a score becomes the operand of the second product in the lane that
// has it.  Q and P keep 32 bits: F32 caches multiply in f32; F16 and Q8_0
// caches, whose values f16 holds (a quant is one, its block's scale is kept
// apart), multiply by Q and P as two f16 each.  These kernels wait for memory,
// so the second product costs them nothing.
#include "sfa_window_dev.h"

namespace sfa {

constexpr int kWaves = 4;

// Positions of a tile and its bytes in LDS.
template <int KVT, int HD>
struct Tile {
    static constexpr int TP = KVT == SFA_KV_F32 ? 16 : 32;
    static constexpr int RB = KVT == SFA_KV_F32 ? HD * 4 : KVT == SFA_KV_F16 ? HD * 2 : HD / kQK * kQ8Bytes;
    static constexpr int CPR = (RB + 15) / 16;               // 16-byte chunks of a row (Q8_0 rows end inside one)
    static constexpr int ROW = CPR * 16;                     // row in LDS
    static constexpr int NI = (TP * CPR + kWave - 1) / kWave;  // load instructions
    static constexpr int BYTES = TP * CPR * 16;
    static constexpr int RP = 256 / ROW > 0 ? 256 / ROW : 1;  // rows under all LDS banks (a power of two but for Q8_0)
};

// Where chunk j of row r lies in its LDS row.  The reads of 16 rows at one
// chunk (K) and of 8 rows at two neighbouring chunks (V of F16) or 4 rows at
// four (V of F32) then cover the banks evenly.
template <int KVT, int HD>
__device__ inline int k_slot(int r, int j) {
    if constexpr (KVT == SFA_KV_Q8_0) return j;
    using T = Tile<KVT, HD>;
    return j ^ (r / T::RP % (T::CPR < 16 ? T::CPR : 16));
}
template <int KVT, int HD>
__device__ inline int v_slot(int r, int j) {
    using T = Tile<KVT, HD>;
    if constexpr (KVT == SFA_KV_F16) return j ^ (r / T::RP % (T::CPR / 2) * 2);
    if constexpr (KVT == SFA_KV_F32) return j ^ (r / 4 % (T::CPR / 4) * 4);
    return j;
}

// Workgroups of a CU: as many as LDS holds, but for Q8_0 of HD 128: a fourth
// would leave too few registers.
template <int KVT, int HD>
constexpr int kGroups = HD != 128 ? 4 : KVT == SFA_KV_Q8_0 ? 3 : 2;

template <int KVT, int HD, int G>
__global__ __launch_bounds__(64 * kWaves, (kGroups<KVT, HD>)) void window_decode_kernel(WindowParams p) {
    using T = Tile<KVT, HD>;
    constexpr int TP = T::TP, MT = TP / 16;  // 16-position blocks of a tile
    constexpr int KS = HD / 32, DB = HD / 16;
    constexpr int NB = HD / kQK;             // quantisation blocks of a row
    constexpr int TAB = KVT == SFA_KV_Q8_0 ? 2 * NB * TP * 4 : 0;  // a wave's scales of the tile, K and V
    constexpr int WAVE = 2 * T::BYTES + TAB;
    constexpr int JOIN = (int)sizeof(float) * kWaves * G * (HD + 2);
    __shared__ __attribute__((aligned(256))) uint8_t lds[kWaves * WAVE > JOIN ? kWaves * WAVE : JOIN];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, qd = lane >> 4;
    // Workgroups go round the eight XCDs.  The rows of neighbouring kv heads share
    // cache lines in a Q8_0 cache: there the heads of one split are eight apart,
    // in one L2 (8 sequences, window 8192: the step 59 -> 51 us).  Whole lines are
    // faster from all over the chip (F16, 64 sequences: 190 us against 200).
    constexpr bool kShared = KVT == SFA_KV_Q8_0;
    int kvh = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
    if constexpr (kShared) {
        kvh = blockIdx.y;
        const int part = blockIdx.z * 8 + blockIdx.x;
        b = (int)to_scalar((uint32_t)part / (uint32_t)p.n_split);
        split = part - b * p.n_split;
        if (b >= p.n_tok) return;  // (the parts are rounded up to eight)
    }
    const int32_t *table = p.page_table + (int64_t)b * p.max_pages;
    const int len = max(p.seq_len[b], 0);

    // Q of column c: rows past G are zero columns
    float amax = 0.0f;
    float qx[KS][8];
    const float *qrow = p.q + ((int64_t)b * p.n_head + kvh * G + (c < G ? c : 0)) * HD;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        // F32: dims 16 j + 4 qd of chunk j = 2 ks and 2 ks + 1; else dims 32 ks + 8 qd
        const int d0 = KVT == SFA_KV_F32 ? 32 * ks + 4 * qd : 32 * ks + 8 * qd;
        const int d1 = KVT == SFA_KV_F32 ? d0 + 16 : d0 + 4;
        const floatx4 u = *reinterpret_cast<const floatx4 *>(qrow + d0);
        const floatx4 v = *reinterpret_cast<const floatx4 *>(qrow + d1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            qx[ks][j] = c < G ? u[j] : 0.0f;
            qx[ks][4 + j] = c < G ? v[j] : 0.0f;
        }
    }

    // what the token attends: [0, ns) and [lo, hi], as tiles: the first n_sink
    // ones, then those of the window
    const int64_t cap = (int64_t)p.max_pages * p.page_size;
    const int pos = len - 1;
    const int lo = pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
    const int hi = pos < cap ? pos : (int)(cap - 1);
    const int ns = min(min(p.n_sink, lo), hi + 1);
    const int sink_tiles = pos < 0 ? 0 : tiles_of(ns, TP);
    const int n_tiles = pos < 0 ? 0 : sink_tiles + (hi >= lo ? hi / TP - lo / TP + 1 : 0);
    int t0, t1;
    split_range(n_tiles, split, p.n_split, t0, t1);

    const int col_bytes = p.n_head_kv * T::RB;
    int k_off[T::NI], v_off[T::NI];
#pragma unroll
    for (int i = 0; i < T::NI; ++i) {
        const int ch = 64 * i + lane, r = ch / T::CPR, j = ch % T::CPR;
        k_off[i] = r * col_bytes + 16 * k_slot<KVT, HD>(r, j);
        v_off[i] = r * col_bytes + 16 * v_slot<KVT, HD>(r, j);
    }
    uint8_t *const mine = lds + wave * WAVE;
    const uint32_t mine_at = lds_addr(mine);
    PageWindow pages;
    // A tile: its first visible rows in the pools, their bytes, and which rows of
    // the tile they are.  The buffer holds the visible rows alone: what else the
    // tile's place in the page holds is not read.
    struct Src {
        const uint8_t *k, *v;
        int bytes, back, from, to;
    };
    auto source = [&](int t) {
        const bool sink = t < sink_tiles;
        const int first = (sink ? t : lo / TP + t - sink_tiles) * TP;
        Src s;
        s.from = max(sink ? 0 : lo - first, 0);
        s.to = min((sink ? ns : hi + 1) - first, TP);
        const int lp = page_of(p, first);
        const int32_t id = pages.get(table, p.max_pages, lp, lane);
        const uint8_t *kb = page_base(id, p.k_pages, p.n_pages, p.k_cold, p.n_cold, p.page_bytes);
        const uint8_t *vb = page_base(id, p.v_pages, p.n_pages, p.v_cold, p.n_cold, p.page_bytes);
        const bool there = kb != nullptr && vb != nullptr;
        const int64_t row = (int64_t)(first - lp * p.page_size + s.from) * col_bytes + kvh * T::RB;
        s.k = there ? kb + row : nullptr;
        s.v = there ? vb + row : nullptr;
        s.bytes = there ? (s.to - s.from - 1) * col_bytes + T::RB : 0;
        s.back = s.from * col_bytes;
        if (!there) s.to = 0;
        return s;
    };
    // (the last instruction of Q8_0 by the lanes that have a chunk left)
    constexpr int LAST = TP * T::CPR - 64 * (T::NI - 1);
    auto load = [&](const uint8_t *rows, const Src &s, const int (&off)[T::NI], uint32_t at) {
        const auto r = buffer_of(rows, s.bytes);
#pragma unroll
        for (int i = 0; i < T::NI; ++i)
            if (i < T::NI - 1 || LAST == 64 || lane < LAST) load_to_lds(r, at + 1024 * i, off[i] - s.back);
    };
    Src cur = {}, next = {};
    int t = t0 + wave;
    if (t < t1) {
        pages.load(table, p.max_pages, page_of(p, (t < sink_tiles ? t : lo / TP + t - sink_tiles) * TP), lane);
        cur = source(t);
        load(cur.k, cur, k_off, mine_at);
        load(cur.v, cur, v_off, mine_at + T::BYTES);
    }

    // Q as two f16 under a power of two of its row, or as it is
    float up = 1.0f;
    half8 qh[KS], ql[KS];
    if constexpr (KVT != SFA_KV_F32) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[ks][j]));
        float down;
        row_exponent(quarters_max(amax), down, up);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 h, l;
                split_f16(qx[ks][j] * down, h, l);
                qh[ks][j] = h;
                ql[ks][j] = l;
            }
    }
    const float f = KVT == SFA_KV_F32 ? p.scale_log2 : score_factor(p.scale_log2, up);

    // probabilities are 2^(s f - base), base kSplitShift below the column's
    // running maximum (F32: at it); l sums this lane's
    constexpr float SHIFT = KVT == SFA_KV_F32 ? 0.0f : (float)kSplitShift;
    float base = -INFINITY, l = 0.0f;
    // Q8_0: V's scales are taken down by the power of two of the largest so far,
    // in whose units o is: a probability times a scale fits an f16 then
    int unit = 1;
    floatx4 o[DB];                  // O^T: dims 16 db + 4 qd + i (Q8_0: see there) of column c
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    const uint8_t *const ks0 = mine, *const vs0 = mine + T::BYTES;
    for (; t < t1; t += kWaves, cur = next) {
        const bool more = t + kWaves < t1;
        wait_loads<T::NI>();  // K is there
        floatx4 s[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (KVT == SFA_KV_F16) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int r = 16 * mt + c;
                    const half8 a = *reinterpret_cast<const half8 *>(ks0 + r * T::ROW + 16 * k_slot<KVT, HD>(r, 4 * ks + qd));
                    s[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[ks], s[mt], 0, 0, 0);
                    s[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[ks], s[mt], 0, 0, 0);
                }
        } else if constexpr (KVT == SFA_KV_F32) {
#pragma unroll
            for (int ks = 0; ks < 2 * KS; ++ks) {
                const floatx4 a = *reinterpret_cast<const floatx4 *>(ks0 + c * T::ROW + 16 * k_slot<KVT, HD>(c, 4 * ks + qd));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], qx[ks / 2][ks % 2 * 4 + i], s[0], 0, 0, 0);
            }
        } else {
            // the blocks' scales as f32 [block][position]: a lane needs those of its eight
            // score rows, whose K rows are other lanes' operands
            float *const tab = reinterpret_cast<float *>(mine + 2 * T::BYTES);
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) {
                const int nb = NB / 2 * (lane >> 5) + i;
                tab[nb * TP + (lane & 31)] = (float)*reinterpret_cast<const _Float16 *>(ks0 + (lane & 31) * T::ROW + kQ8Bytes * nb);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint8_t *const blk = ks0 + (16 * mt + c) * T::ROW + kQ8Bytes * nb + 2 + 8 * qd;
                    uint32_t w[3];
                    half8 a;
                    if (nb % 2) {  // the quants of odd blocks start at a multiple of 4, those of even ones 2 after one
                        __builtin_memcpy(w, __builtin_assume_aligned(blk, 4), 8);
                        a = quants8(w[0], w[1]);
                    } else {
                        __builtin_memcpy(w, __builtin_assume_aligned(blk - 2, 4), 12);
                        a = quants8(__builtin_amdgcn_alignbyte(w[1], w[0], 2), __builtin_amdgcn_alignbyte(w[2], w[1], 2));
                    }
                    floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[nb], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[nb], x, 0, 0, 0);
                    const floatx4 d = *reinterpret_cast<const floatx4 *>(tab + nb * TP + 16 * mt + 4 * qd);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][i] = fmaf(x[i], d[i], s[mt][i]);
                }
        }
        // K's reads are done: the next tile's
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            next = source(t + kWaves);
            load(next.k, next, k_off, mine_at);
        }
        const int from = cur.from, to = cur.to;
        if (from > 0 || to < TP) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 16 * mt + 4 * qd + i;
                    if (r < from || r >= to) s[mt][i] = -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
            mx = fmaxf(mx, fmaxf(fmaxf(s[mt][0], s[mt][1]), fmaxf(s[mt][2], s[mt][3])));
        mx = quarters_max(mx) * f - SHIFT;
        if (__ballot(mx > base) != 0) {
            const float nb = fmaxf(mx, base);
            const float a = nb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - nb);
            l *= a;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= a;
            base = nb;
        }
        const float sub = base == -INFINITY ? 0.0f : base;
        float pr[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pr[mt][i] = __builtin_amdgcn_exp2f(fmaf(s[mt][i], f, -sub));
                l += pr[mt][i];
            }
        // V is there
        if (more) wait_loads<T::NI>();
        else wait_loads<0>();
        if constexpr (KVT == SFA_KV_F32) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * qd + i;
                    const float a = *reinterpret_cast<const float *>(vs0 + r * T::ROW + 16 * v_slot<KVT, HD>(r, 4 * d + c / 4) + 4 * (c & 3));
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, pr[0][i], o[d], 0, 0, 0);
                }
        } else if constexpr (KVT == SFA_KV_F16) {
            half8 ph, pl;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 h, lo16;
                split_f16(pr[j / 4][j % 4], h, lo16);
                ph[j] = h;
                pl[j] = lo16;
            }
            // operand positions 4 qd .. and 16 + 4 qd ..: the lane's own scores
            const int rr = 4 * qd + (c >> 2);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const int at = 16 * v_slot<KVT, HD>(rr, 2 * d + ((c & 3) >> 1)) + 8 * (c & 1);
                const int at2 = 16 * v_slot<KVT, HD>(rr + 16, 2 * d + ((c & 3) >> 1)) + 8 * (c & 1);
                const half4 x = tr16_read(vs0 + rr * T::ROW + at), y = tr16_read(vs0 + (rr + 16) * T::ROW + at2);
                const half8 a = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[d], 0, 0, 0);
            }
        } else {
            float *const tab = reinterpret_cast<float *>(mine + 2 * T::BYTES) + NB * TP;
            float d[NB / 2], dmax = 0.0f;
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) {
                d[i] = (float)*reinterpret_cast<const _Float16 *>(vs0 + (lane & 31) * T::ROW + kQ8Bytes * (NB / 2 * (lane >> 5) + i));
                dmax = fmaxf(dmax, fabsf(d[i]));
            }
            const int e = max(__builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, wave_max(dmax)) >> 23)), 1);
            if (e > unit) {
                const float a = __builtin_amdgcn_ldexpf(1.0f, unit - e);
#pragma unroll
                for (int i = 0; i < DB; ++i) o[i] *= a;
                unit = e;
            }
            const float down = __builtin_amdgcn_ldexpf(1.0f, 127 - unit);
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) tab[(NB / 2 * (lane >> 5) + i) * TP + (lane & 31)] = d[i] * down;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                // a position's block scale goes with its probability
                half8 ph, pl;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const floatx4 d = *reinterpret_cast<const floatx4 *>(tab + nb * TP + 16 * mt + 4 * qd);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        half2v h, lo16;
                        float u = pr[mt][i] * d[i], v = pr[mt][i + 1] * d[i + 1];
                        asm("" : "+v"(u), "+v"(v));  // (see split_f16)
                        split2_f16(u, v, h, lo16);
                        ph[4 * mt + i] = h[0], ph[4 * mt + i + 1] = h[1];
                        pl[4 * mt + i] = lo16[0], pl[4 * mt + i + 1] = lo16[1];
                    }
                }
                // rows of two products: dims 2 c and 2 c + 1 of the block, one 16-bit read a position
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int ra = j < 2 ? 4 * qd + 2 * j : 16 + 4 * qd + 2 * (j - 2);
                    const uint8_t *const src = vs0 + ra * T::ROW + kQ8Bytes * nb + 2 + 2 * c;
                    w[j] = *reinterpret_cast<const uint16_t *>(src) | (uint32_t)*reinterpret_cast<const uint16_t *>(src + T::ROW) << 16;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    half8 a;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const half2v h = quants2((e ? w[j] >> 8 : w[j]) & 0x00ff00ffu);
                        a[2 * j] = h[0];
                        a[2 * j + 1] = h[1];
                    }
                    o[2 * nb + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[2 * nb + e], 0, 0, 0);
                    o[2 * nb + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[2 * nb + e], 0, 0, 0);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load(next.v, next, v_off, mine_at + T::BYTES);
        }
    }

    // the four waves join
    l = quarters_sum(l);
    if constexpr (KVT == SFA_KV_Q8_0) {
        const float back = __builtin_amdgcn_ldexpf(1.0f, unit - 127);
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= back;
    }
    float *const jm = reinterpret_cast<float *>(lds), *const jl = jm + kWaves * G, *const jo = jl + kWaves * G;
    __syncthreads();
    if (c < G) {
        if (qd == 0) {
            jm[wave * G + c] = base;
            jl[wave * G + c] = l;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = KVT == SFA_KV_Q8_0 ? d / 2 * 32 + 2 * (4 * qd + i) + d % 2 : 16 * d + 4 * qd + i;
                jo[(wave * G + c) * HD + e] = o[d][i];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * HD; i += 64 * kWaves) {
        const int g = i / HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, jm[w * G + g]);
        const float mb = mm == -INFINITY ? 0.0f : mm;
        float L = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float x = __builtin_amdgcn_exp2f(jm[w * G + g] - mb);
            L = fmaf(jl[w * G + g], x, L);
            acc = fmaf(jo[w * G * HD + i], x, acc);
        }
        const int64_t row = (int64_t)b * p.n_head + kvh * G + g;
        if (p.n_split == 1) {
            p.out[row * HD + i % HD] = L == 0.0f ? 0.0f : acc / L;
        } else {
            p.rec_o[(row * p.n_split + split) * HD + i % HD] = acc;
            if (i % HD == 0) p.rec_ml[row * p.n_split + split] = make_float2(mm, L);
        }
    }
}

// Joins a row's split records: a thread has four dims of every GR-th split,
// GR groups of HD / 4 threads a row.
template <int HD, int GR>
__global__ __launch_bounds__(256) void window_merge_kernel(WindowParams p, int64_t rows) {
    constexpr int LN = HD / 4, NG = 256 / LN;
    __shared__ float jm[NG], jl[NG];
    __shared__ floatx4 jo[NG][LN];
    const int grp = threadIdx.x / LN, e = threadIdx.x % LN;
    const int64_t row = (int64_t)blockIdx.x * (NG / GR) + grp / GR;
    const bool ok = row < rows;
    const float2 *const ml = p.rec_ml + row * p.n_split;
    const float *const rec = p.rec_o + row * p.n_split * HD + 4 * e;
    float m = -INFINITY, l = 0.0f;
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    // four splits' loads at a time (a split past the last: the last, of no weight)
    for (int s = grp % GR; ok && s < p.n_split; s += 4 * GR) {
        float2 r[4];
        floatx4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = min(s + i * GR, p.n_split - 1);
            r[i] = ml[at];
            x[i] = *reinterpret_cast<const floatx4 *>(rec + (int64_t)at * HD);
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) mn = fmaxf(mn, r[i].x);
        const float mb = mn == -INFINITY ? 0.0f : mn, a = __builtin_amdgcn_exp2f(m - mb);
        l *= a;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] *= a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s + i * GR >= p.n_split) continue;
            const float w = __builtin_amdgcn_exp2f(r[i].x - mb);
            l = fmaf(r[i].y, w, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(x[i][j], w, o[j]);
        }
        m = mn;
    }
    if constexpr (GR > 1) {
        if (e == 0) jm[grp] = m, jl[grp] = l;
        jo[grp][e] = o;
        __syncthreads();
        if (grp % GR != 0) return;
        float mm = -INFINITY;
#pragma unroll
        for (int g = 0; g < GR; ++g) mm = fmaxf(mm, jm[grp + g]);
        if (mm == -INFINITY) mm = 0.0f;
        l = 0.0f;
        o = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < GR; ++g) {
            const float w = __builtin_amdgcn_exp2f(jm[grp + g] - mm);
            l = fmaf(jl[grp + g], w, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(jo[grp + g][e][j], w, o[j]);
        }
    }
    if (!ok) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = l == 0.0f ? 0.0f : o[j] / l;
    *reinterpret_cast<floatx4 *>(p.out + row * HD + 4 * e) = o;
}

template <int HD>
static void launch_merge(const WindowParams &p, int64_t rows, hipStream_t s) {
    constexpr int NG = 256 / (HD / 4);
    // few splits are read by one group of threads in one round of loads
    if (p.n_split <= 4)
        hipLaunchKernelGGL((window_merge_kernel<HD, 1>), dim3((unsigned)((rows + NG - 1) / NG)), dim3(256), 0, s, p, rows);
    else
        hipLaunchKernelGGL((window_merge_kernel<HD, 8>), dim3((unsigned)((rows + NG / 8 - 1) / (NG / 8))), dim3(256), 0, s, p, rows);
}

int window_merge_launch(const WindowParams &p, int head_dim, int64_t rows, hipStream_t s) {
    if (head_dim == 128) launch_merge<128>(p, rows, s);
    else if (head_dim == 64) launch_merge<64>(p, rows, s);
    else launch_merge<32>(p, rows, s);
    return hipGetLastError() == hipSuccess ? SFA_OK : SFA_ERR_RUNTIME;
}

// Workgroups of one sequence and kv head: as many as give every CU one (F16
// and F32 of HD 128) or two, at most one per four tiles of the longest span.
// More records cost more than a fuller chip gives: F16, one sequence, window
// 4096 (32 / 8 heads of 128): 12.2 / 11.5 / 12.0 / 12.5 us with 16 / 24 / 32 /
// 48; 64 sequences 182 / 193 with 1 / 2; Q8_0, 8 sequences, window 8192: 53 /
// 46.4 / 46.5 / 48.7 with 4 / 8 / 12 / 16.
// Short spans stay with one, whose rounds of a tile a wave take `round` us each,
// against a second launch: 2 us, and 2.7 more where the host issues every call.
// Measured (two sequences; one workgroup / split, GPU alone): F16, heads of
// 128: window 124 6.5 / 7.2, 252 7.7 / 7.6, 508 9.9 / 7.7; Q8_0 124 8.7 / 8.5,
// 252 10.9 / 8.7; F32 heads of 32: 252 6.7 / 6.4, 508 10.0 / 6.6.
int window_decode_splits(const sfa_kv_desc *kv, int32_t B, int32_t max_seq_len, int32_t window, int32_t n_sink) {
    const bool f32 = kv->kv_type == SFA_KV_F32, f16 = kv->kv_type == SFA_KV_F16;
    const int tp = f32 ? 16 : 32;
    const int64_t seen = (int64_t)window + n_sink < max_seq_len ? (int64_t)window + n_sink : max_seq_len;
    const double width = kv->head_dim / 128.0, round = f32 ? 0.3 + 1.5 * width : f16 ? 0.6 + 0.55 * width : 1.1 + 1.1 * width;
    if (((double)seen / (tp * kWaves) - 1.0) * round <= 2.1) return 1;
    const int64_t tiles = (seen + tp - 1) / tp + 2;
    const int64_t room = kv->head_dim == 128 && kv->kv_type != SFA_KV_Q8_0 ? 256 : 512;
    int64_t n = room / ((int64_t)B * kv->n_head_kv);
    if (n > (tiles + kWaves - 1) / kWaves) n = (tiles + kWaves - 1) / kWaves;
    return n < 1 ? 1 : (int)n;
}

template <int KVT, int HD>
static void launch_g(const WindowParams &p, dim3 grid, hipStream_t s) {
    const dim3 block(64 * kWaves);
    switch (p.n_head / p.n_head_kv) {
    case 1: hipLaunchKernelGGL((window_decode_kernel<KVT, HD, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((window_decode_kernel<KVT, HD, 2>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((window_decode_kernel<KVT, HD, 4>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((window_decode_kernel<KVT, HD, 8>), grid, block, 0, s, p); break;
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

int window_decode_launch(const WindowParams &p, const sfa_kv_desc *kv, int32_t B, hipStream_t s) {
    const int64_t rows = (int64_t)B * kv->n_head;
    if (B > 65535 || kv->n_head_kv > 65535 || rows > INT32_MAX) return SFA_ERR_UNSUPPORTED;
    const dim3 grid = kv->kv_type == SFA_KV_Q8_0 ? dim3(8, (unsigned)kv->n_head_kv, (unsigned)(((int64_t)B * p.n_split + 7) / 8))
                                                 : dim3((unsigned)kv->n_head_kv, (unsigned)p.n_split, (unsigned)B);
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
