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
//
// Measured (32 / 8 heads of 128): F16, 4096 tokens on 8192, window 4096: 503 us,
// 547 TFLOP/s of what the tokens see, which is 1095 on the matrix cores (a large
// f16 product of the library: 1073; the clock falls to 1.7 GHz to 2 GHz under
// either).  Q8_0, 777 tokens on 6000, window 1024: 68 us; F32 (16 / 4 heads),
// 1500 tokens, window 512: 47 us: bound by the chain of a tile (its values into
// halves, a barrier, products, a barrier) on two workgroups a CU, matrix cores
// busy 21 % and 15 %.
#include <type_traits>

#include "sfa_window_dev.h"

namespace sfa {

constexpr int kRows = 128;         // of a workgroup
constexpr int kMostSplits = 64;    // of a row block's tiles
constexpr int kMostBlocks = 1024;  // workgroups where there are splits

template <int KVT, int HD>
struct PTile {
    static constexpr int TP = KVT == SFA_KV_F32 ? 32 : 64;  // positions
    static constexpr int RB = KVT == SFA_KV_F32 ? HD * 4 : KVT == SFA_KV_F16 ? HD * 2 : HD / kQK * kQ8Bytes;
    static constexpr int ROW = HD * 2;                      // a row in LDS: f16, or f16 halves of wider values
    static constexpr int CPR = ROW / 16;
    static constexpr int BYTES = TP * ROW;
    static constexpr int NI = BYTES / 4096;                 // F16: load instructions of a wave, a tensor
    static constexpr int RP = 256 / ROW > 0 ? 256 / ROW : 1;  // rows under all LDS banks
    static constexpr int NG = ROW / 64 > 0 ? ROW / 64 : 1;
};

// Where chunk j of row r lies in its LDS row.  K's reads are 16 rows at one
// chunk, V's four rows at 64 neighbouring bytes; writes of Q8_0 and F32 rows
// are one chunk of every block of neighbouring rows: all of these fall in
// different banks.
template <int HD>
__device__ inline int pk_slot(int r, int j) {
    using T = PTile<SFA_KV_F16, HD>;
    return j ^ (r / T::RP % T::CPR);
}
template <int HD>
__device__ inline int pv_slot(int r, int j) {
    using T = PTile<SFA_KV_F16, HD>;
    const int q = r / T::RP;
    return j ^ (q % T::NG * 4) ^ (q % (HD == 32 ? 2 : 4));
}

// Runs the N steps of a product loop with the operand reads AHEAD steps before
// their use; left to itself the compiler waits for every operand right before
// it is used.  Vector and scalar arithmetic may move over the fences, reads and
// matrix instructions may not.
template <int N, int AHEAD, int FENCE = 0x406, typename Read, typename Use>
__device__ inline void pipelined(Read read, Use use) {
    decltype(read(0)) a[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD && i < N; ++i) a[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const auto now = a[i % AHEAD];
        if (i + AHEAD < N) a[i % AHEAD] = read(i + AHEAD);
        __builtin_amdgcn_sched_barrier(FENCE);
        use(i, now);
        __builtin_amdgcn_sched_barrier(FENCE);
    }
}

// A lane's row, and its workgroup's rows and tiles.
struct Block {
    int kvh, split;
    int tok, head, tpos;   // the lane's row: its token (a row past the chunk: the last), head and position
    bool row_ok, wave_ok;  // the lane has a row, the wave has any
    int first, last;       // positions of the workgroup's tokens
    int lo, hi, ns;        // what any of them sees: sinks before the window [0, ns), then [lo, hi]
    int sink_tiles, t0, t1;
};
template <int G, int TP>
__device__ inline Block block_of(const WindowParams &p, int wave, int n) {
    Block b;
    // Workgroups go round the eight XCDs: with Hkv a multiple of 8 a kv head's
    // tiles stay in one L2.  The last rows, which see the most, come first.
    const int blk = gridDim.z - 1 - blockIdx.z;
    b.kvh = blockIdx.x;
    b.split = blockIdx.y;
    const int row = blk * kRows + wave * 32 + n;  // token row / G, head row % G of the group
    b.row_ok = row < p.n_tok * G;
    b.tok = b.row_ok ? row / G : p.n_tok - 1;
    b.head = b.kvh * G + row % G;
    b.tpos = p.q_pos0 + b.tok;
    b.wave_ok = blk * kRows + wave * 32 < p.n_tok * G;
    const int64_t cap = (int64_t)p.max_pages * p.page_size;
    b.first = p.q_pos0 + blk * kRows / G;
    b.last = p.q_pos0 + min((blk * kRows + kRows - 1) / G, p.n_tok - 1);
    b.lo = b.first - p.window + 1 > 0 ? b.first - p.window + 1 : 0;
    b.hi = b.last < cap ? b.last : (int)(cap - 1);
    b.ns = min(min(p.n_sink, b.lo), b.hi + 1);
    b.sink_tiles = tiles_of(b.ns, TP);
    const int n_tiles = b.sink_tiles + (b.hi >= b.lo ? b.hi / TP - b.lo / TP + 1 : 0);
    split_range(n_tiles, b.split, p.n_split, b.t0, b.t1);
    return b;
}

// A tile: where it lies and which of its rows any token of the workgroup sees.
struct Src {
    int first, from, to;       // position of its row 0, its visible rows
    bool sink, there, masked;  // masked: some row of the workgroup does not see all of it
    const uint8_t *k, *v;      // its first visible rows
    int bytes, back;           // of the visible rows; offset of the first from row 0
};
template <int TP, int RB>
__device__ inline Src source(const WindowParams &p, const Block &b, PageWindow &pages, int t, int lane) {
    const int col_bytes = p.n_head_kv * RB;
    Src s;
    s.sink = t < b.sink_tiles;
    s.first = (s.sink ? t : b.lo / TP + t - b.sink_tiles) * TP;
    s.from = max(s.sink ? 0 : b.lo - s.first, 0);
    s.to = min((s.sink ? b.ns : b.hi + 1) - s.first, TP);
    const int lp = page_of(p, s.first);
    const int32_t id = pages.get(p.page_table, p.max_pages, lp, lane);
    const uint8_t *kb = page_base(id, p.k_pages, p.n_pages, p.k_cold, p.n_cold, p.page_bytes);
    const uint8_t *vb = page_base(id, p.v_pages, p.n_pages, p.v_cold, p.n_cold, p.page_bytes);
    s.there = kb != nullptr && vb != nullptr;
    const int64_t at = (int64_t)(s.first - lp * p.page_size + s.from) * col_bytes + b.kvh * RB;
    s.k = s.there ? kb + at : nullptr;
    s.v = s.there ? vb + at : nullptr;
    s.bytes = s.there ? (s.to - s.from - 1) * col_bytes + RB : 0;
    s.back = s.from * col_bytes;
    const int end = s.first + TP - 1;
    s.masked = (s.from > 0) | (s.to < TP) | !s.there |
               (!s.sink & ((end > b.first) | ((s.first <= b.last - p.window) & (end >= p.n_sink))));
    return s;
}
template <int TP>
__device__ inline void page_window(const WindowParams &p, const Block &b, PageWindow &pages, int lane) {
    const int t = b.t0;
    if (t < b.t1)
        pages.load(p.page_table, p.max_pages, page_of(p, (t < b.sink_tiles ? t : b.lo / TP + t - b.sink_tiles) * TP), lane);
}

// The rows of a tile that the token at tpos sees, a bit each.
__device__ inline uint64_t seen_rows(const WindowParams &p, const Src &s, int tpos) {
    auto below = [](int n) { return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1; };
    const int at = tpos - s.first;
    uint64_t m = below(min(s.to, at + 1)) & ~below(s.from);
    if (!s.sink) m &= ~below(max(at, 0) + 1 - p.window) | below(p.n_sink - s.first);
    return m;
}

// Scores [32 x][16], rows 32 x + 8 (i / 4) + 4 hh + i % 4, of the rows that are
// not seen become -inf: three instructions a score (by comparisons of positions: 15).
template <int PB>
__device__ inline void mask_scores(const WindowParams &p, const Src &src, int tpos, int hh, floatx16 (&s)[PB]) {
    asm("" : "+v"(tpos), "+v"(hh));  // (nothing of them held over the loop)
    const uint64_t m = seen_rows(p, src, tpos) >> (4 * hh);
#pragma unroll
    for (int i = 0; i < 16 * PB; ++i) {
        const uint32_t word = (uint32_t)(i < 16 ? m : m >> 32);
        s[i / 16][i % 16] = word >> (i / 4 % 4 * 8 + i % 4) & 1 ? s[i / 16][i % 16] : -INFINITY;
    }
}

// A value of V that is not finite would reach rows that do not see it, as 0
// times it.  Each wave looks its quarter of a masked tile over: such values
// become zeros and get a bit, and the rows that see one are NaN afterwards.
template <int HD>
__device__ inline void look_over(uint8_t *v, uint8_t *bits_of, uint64_t *bad, int wave, int lane) {
    using T = PTile<SFA_KV_F16, HD>;
    bool any = false;
#pragma unroll
    for (int i = 0; i < T::NI; ++i) {
        const int ch = (T::NI * wave + i) * 64 + lane;
        intx4 *const at = reinterpret_cast<intx4 *>(v + 16 * ch);
        intx4 x = *at;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) bits |= (((uint32_t)x[j / 2] >> (j % 2 ? 26 : 10) & 31) == 31 ? 1u : 0u) << j;
        if (bits != 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] &= (bits >> 2 * j & 1 ? 0 : 0xffff) | (bits >> (2 * j + 1) & 1 ? 0 : (int)0xffff0000);
            *at = x;
            any = true;
        }
        bits_of[ch] = (uint8_t)bits;
    }
    const uint64_t who = __ballot(any);
    if (lane == 0) bad[wave] = who;
}

__device__ inline bool any_bad(const uint64_t *bad) { return __ballot((bad[0] | bad[1] | bad[2] | bad[3]) != 0) != 0; }

// The lane's outputs that a value set to zero has a part in, a bit for each
// o[d][i] at 16 d + i; was(r, e): whether V's value e of row r was.  A small loop
// that leaves o alone: it hardly ever runs, and the registers are full.
template <int HD, typename Was>
__device__ inline uint64_t spoiled(const WindowParams &p, const Src &s, int tpos, int hh, Was was) {
    asm("" : "+v"(tpos));  // (nothing of it held over the tile's products)
    uint64_t bits = 0;
    const uint64_t seen = seen_rows(p, s, tpos);
    for (int r = s.from; r < s.to; ++r) {
        if ((seen >> r & 1) == 0) continue;
#pragma unroll 1
        for (int j = 0; j < HD / 2; ++j)
            bits |= (uint64_t)was(r, j / 16 * 32 + j % 16 / 4 * 8 + 4 * hh + j % 4) << j;
    }
    return bits;
}

// The lane's outputs, NaN where a bit of `bad` is set, or its split record.
template <int HD, typename O>
__device__ inline void store_row(const WindowParams &p, const Block &b, int hh, const O &o, float base, float l, float unit, uint64_t bad) {
    if (!b.row_ok) return;
    float la, lb;
    swap_halves(l, la, lb);
    l = la + lb;
    const float w = p.n_split > 1 ? unit : l == 0.0f ? 0.0f : unit / l;
    const int64_t row = (int64_t)b.tok * p.n_head + b.head;
    float *const dst = p.n_split > 1 ? p.rec_o + (row * p.n_split + b.split) * HD : p.out + row * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            floatx4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = bad >> (16 * d + 4 * i4 + i) & 1 ? NAN : o[d][4 * i4 + i] * w;
            *reinterpret_cast<floatx4 *>(dst + 32 * d + 8 * i4 + 4 * hh) = x;
        }
    if (p.n_split > 1 && hh == 0) p.rec_ml[row * p.n_split + b.split] = make_float2(base, l);
}

// Q of a lane's row, dims 16 c + 8 hh + j, as two f16 under a power of two of
// the row; returns that power's inverse.
template <int HD>
__device__ inline float split_q(const float *q, half8 (&qh)[HD / 16], half8 (&ql)[HD / 16]) {
    float x[HD / 16][8], amax = 0.0f, a, b, down, up;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
        const floatx4 u = *reinterpret_cast<const floatx4 *>(q + 16 * c);
        const floatx4 v = *reinterpret_cast<const floatx4 *>(q + 16 * c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[c][j] = u[j], x[c][4 + j] = v[j];
    }
#pragma unroll
    for (int c = 0; c < HD / 16; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[c][j]));
    swap_halves(amax, a, b);
    row_exponent(fmaxf(a, b), down, up);
#pragma unroll
    for (int c = 0; c < HD / 16; ++c)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            half2v h, l;
            split2_f16(x[c][j] * down, x[c][j + 1] * down, h, l);
            qh[c][j] = h[0], qh[c][j + 1] = h[1];
            ql[c][j] = l[0], ql[c][j + 1] = l[1];
        }
    return up;
}

// The F16 kernel.
template <int HD, int G>
__global__ __launch_bounds__(256, 2) void window_prefill_f16_kernel(WindowParams p) {
    using T = PTile<SFA_KV_F16, HD>;
    constexpr int TP = T::TP, PB = TP / 32, DB = HD / 32, KC = HD / 16, ST = TP / 16;
    __shared__ __attribute__((aligned(256))) uint8_t lds[4][T::BYTES];  // K, K, V, V
    __shared__ uint64_t v_bad[2][4];  // (two of each: a slow wave may still read the last tile's)
    __shared__ uint8_t v_bits[2][TP * T::CPR];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5;
    const Block b = block_of<G, TP>(p, wave, n);
    PageWindow pages;
    page_window<TP>(p, b, pages, lane);

    half8 qh[KC], ql[KC];
    const float f = score_factor(p.scale_log2, split_q<HD>(p.q + ((int64_t)b.tok * p.n_head + b.head) * HD + 8 * hh, qh, ql));

    // This wave's quarter of a tile, lane by lane: load i has RPI rows more than
    // load 0, which flips bit 2 of K's slots i times and leaves V's (few registers:
    // what the compiler cannot hold it would reload behind the tile's loads).
    constexpr int RPI = 64 / T::CPR;
    static_assert(RPI % (4 * T::RP) == 0 || T::NI == 1, "the slots of load i");
    const int col_bytes = p.n_head_kv * T::RB;
    const int r_0 = T::NI * RPI * wave + lane / T::CPR;
    const int row_off = r_0 * col_bytes;
    const int k_chunk = 16 * pk_slot<HD>(r_0, lane % T::CPR), v_chunk = 16 * pv_slot<HD>(r_0, lane % T::CPR);
    const uint32_t my_lds = lds_addr(lds[0]) + 1024 * T::NI * wave;
    auto load_k = [&](const Src &s, int buf) {
        const auto r = buffer_of(s.k, s.bytes);
#pragma unroll
        for (int i = 0; i < T::NI; ++i)
            load_to_lds(r, my_lds + buf * T::BYTES + 1024 * i, row_off + (i * RPI * col_bytes - s.back) + (k_chunk ^ (64 * i)));
    };
    auto load_v = [&](const Src &s, int buf) {
        const auto r = buffer_of(s.v, s.bytes);
#pragma unroll
        for (int i = 0; i < T::NI; ++i)
            load_to_lds(r, my_lds + buf * T::BYTES + 1024 * i, row_off + (i * RPI * col_bytes - s.back) + v_chunk);
    };

    // probabilities are 2^(s f - base), base kSplitShift below the row's running
    // maximum; l sums this lane's
    float base = -INFINITY, l = 0.0f;
    uint64_t bad = 0;
    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    floatx16 s[PB];

    // Operand addresses: a step's are these with its chunk XORed in (the slots
    // are XORs too) and its rows added.
    const int li = lane & 15, vr = 4 * hh + (li >> 2);
    const int k_row = n * T::ROW + 16 * pk_slot<HD>(n, hh);
    const int v_row = vr * T::ROW + 16 * pv_slot<HD>(vr, 2 * (lane >> 4 & 1) + ((li & 3) >> 1)) + 8 * (li & 1);
    // Operand of step (st, d): positions 16 st + 4 hh .. and 16 st + 8 + 4 hh ..,
    // the lane's own scores; four values a read, lane i of 16 gets dim i of the
    // four rows its group names.
    auto v_at = [&](int v_base, int i) {
        const uint8_t *const at = &lds[0][0] + (v_base ^ (64 * (i % DB))) + 16 * (i / DB) * T::ROW;
        const half4 x = tr16_read(at), y = tr16_read(at + 8 * T::ROW);
        return half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    auto tile = [&](const Src &src, int par) {
        int k_base = k_row + par * T::BYTES;
        asm("" : "+v"(k_base));  // keeps the compiler from holding every step's address
#pragma unroll
        for (int x = 0; x < PB; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
        pipelined<KC * PB, 3>(
            [&](int i) { return *reinterpret_cast<const half8 *>(&lds[0][0] + (k_base ^ (32 * (i / PB))) + i % PB * 32 * T::ROW); },
            [&](int i, half8 a) {
                const int c = i / PB, x = i % PB;
                s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], s[x], 0, 0, 0);
                s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], s[x], 0, 0, 0);
            });
        if (src.masked) mask_scores<PB>(p, src, b.tpos, hh, s);
        float mx = -INFINITY, x, y;
#pragma unroll
        for (int i = 0; i < 16 * PB; ++i) mx = fmaxf(mx, s[i / 16][i % 16]);
        swap_halves(mx, x, y);
        mx = fmaxf(x, y) * f - (float)kSplitShift;
        if (__ballot(mx > base) != 0) {
            const float nb = fmaxf(mx, base);
            const float a = nb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - nb);
            l *= a;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= a;
            base = nb;
        }
        const float sub = base == -INFINITY ? 0.0f : base;
        half8 ph[ST], pl[ST];
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int e = 8 * st + j;
                float u = __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], f, -sub));
                float v = __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16 + 1], f, -sub));
                l += u + v;
                asm("" : "+v"(u), "+v"(v) : "v"(l));
                half2v h, r;
                split2_f16(u, v, h, r);
                ph[st][j] = h[0], ph[st][j + 1] = h[1];
                pl[st][j] = r[0], pl[st][j + 1] = r[1];
            }
        int v_base = v_row + (2 + par) * T::BYTES;
        asm("" : "+v"(v_base));
        pipelined<ST * DB, 3>([&](int i) { return v_at(v_base, i); },
                              [&](int i, half8 a) {
                                  const int st = i / DB, d = i % DB;
                                  o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[st], o[d], 0, 0, 0);
                                  o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[st], o[d], 0, 0, 0);
                              });
        if (src.masked && any_bad(v_bad[par]))
            bad |= spoiled<HD>(p, src, b.tpos, hh, [&](int r, int e) { return v_bits[par][r * T::CPR + pv_slot<HD>(r, e / 8)] >> e % 8 & 1; });
    };

    Src cur = {}, next = {};
    auto issue = [&](int t, int par) {
        const Src src = source<TP, T::RB>(p, b, pages, t, lane);
        load_k(src, par);
        load_v(src, 2 + par);
        return src;
    };
    if (b.t0 < b.t1) cur = issue(b.t0, 0);
    int par = 0;
    for (int t = b.t0; t < b.t1; ++t, par ^= 1, cur = next) {
        wait_loads<0>();
        if (cur.masked) look_over<HD>(lds[2 + par], v_bits[par], v_bad[par], wave, lane);
        __syncthreads();  // this tile is there, and the other buffers have been read
        if (t + 1 < b.t1) next = issue(t + 1, par ^ 1);
        if (b.wave_ok && cur.there) tile(cur, par);
    }
    store_row<HD>(p, b, hh, o, base, l, 1.0f, bad);
}

// The F32 and Q8_0 kernel: caches whose values are wider than an f16.  A tile
// waits in registers while the last one is computed and goes to LDS as f16:
// - F32: K and V as two f16 each, a row of K and eight rows of V under the
//   power of two of their largest value;
// - Q8_0: K's quants, whose blocks' scales multiply the scores of a block; V's
//   values (a quant times its scale) as two f16, exactly.
// Three products then stand for one of 32 bits (hi hi, hi lo, lo hi; QK of
// Q8_0 needs two).  A 32-bit matrix instruction is 16 times slower than an f16
// one.
template <int KVT, int HD, int G>
__global__ __launch_bounds__(256, 2) void window_prefill_wide_kernel(WindowParams p) {
    using T = PTile<KVT, HD>;
    constexpr int TP = T::TP, PB = TP / 32, DB = HD / 32, KC = HD / 16, NB = HD / kQK, ST = TP / 16;
    constexpr bool kQ8 = KVT == SFA_KV_Q8_0;
    constexpr int SETS = kQ8 ? 3 : 4;               // K (F32: and its lower halves), V, V's lower halves
    constexpr int V_SHIFT = kQ8 ? 7 : kSplitShift;  // V's largest scale goes to 2^7, its largest value to 2^14
    constexpr int FENCE = kQ8 ? 0x7f6 : 0x406;      // Q8_0 has loads and arithmetic of its scales between the products
    __shared__ __attribute__((aligned(256))) uint8_t lds[SETS][T::BYTES];
    __shared__ __attribute__((aligned(16))) float k_scale[kQ8 ? NB : 1][TP];
    __shared__ int v_exp[4];                        // exponent of the largest of V: F32: of each 8 positions, Q8_0: of each 16
    __shared__ uint64_t v_bad[4];                   // lanes of a wave with values of V that are not finite, held as zeros
    __shared__ uint16_t v_bits[kQ8 ? 4 : 256];      // F32: a bit for each such value of a thread

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5;
    const Block b = block_of<G, TP>(p, wave, n);
    PageWindow pages;
    page_window<TP>(p, b, pages, lane);
    half8 qh[KC], ql[KC];
    const float f = score_factor(p.scale_log2, split_q<HD>(p.q + ((int64_t)b.tok * p.n_head + b.head) * HD + 8 * hh, qh, ql));

    // What a thread brings of a tile.  F32: 1/8 of a row of K and of V, four
    // neighbouring values of every 32, so that a load instruction reads whole
    // lines.  Q8_0: a block; with HD 128 one of K and one of V, with HD 64 the
    // first two waves have K's and the others V's.
    const int col_bytes = p.n_head_kv * T::RB;
    constexpr int FPT = HD / 8;
    constexpr int UN = kQ8 ? NB / 2 : 2, WORDS = kQ8 ? 9 : FPT;
    const int unit = kQ8 && NB == 2 ? threadIdx.x & 127 : threadIdx.x;
    const int u_row = kQ8 ? unit / NB : unit / 8, u_blk = kQ8 ? unit % NB : unit % 8;
    // (a block's nine words start at its first multiple of 4)
    const int u_off = u_row * col_bytes + (kQ8 ? kQ8Bytes * u_blk - 2 * (u_blk & 1) : 16 * u_blk);
    uint32_t raw[UN][WORDS];
    auto issue = [&](int t) {
        const Src s = source<TP, T::RB>(p, b, pages, t, lane);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const auto r = buffer_of((UN == 2 ? u == 0 : wave < 2) ? s.k : s.v, s.bytes);
#pragma unroll
            for (int i = 0; i + 4 <= WORDS; i += 4) {
                const intx4 x = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(r, u_off - s.back, (kQ8 ? 4 : 32) * i, 0));
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[u][i + j] = x[j];
            }
            if constexpr (WORDS % 4 != 0) raw[u][WORDS - 1] = __builtin_amdgcn_raw_buffer_load_b32(r, u_off - s.back, 4 * (WORDS - 1), 0);
        }
        return s;
    };
    auto stage_q8 = [&]() {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const bool is_v = UN == 2 ? u == 1 : wave >= 2;
            const uint32_t *const w = raw[u];
            const bool odd = u_blk & 1;  // d in the upper half of the first word, quants from the second on
            float d = (float)__builtin_bit_cast(_Float16, (uint16_t)(odd ? w[0] >> 16 : w[0]));
            uint32_t qw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) qw[i] = odd ? w[i + 1] : __builtin_amdgcn_alignbyte(w[i + 1], w[i], 2);
            if (is_v) {
                const bool bad = !(fabsf(d) < INFINITY);
                d = bad ? 0.0f : d;
                const uint64_t who = __ballot(bad);
                const int e = max((int)(__builtin_bit_cast(uint32_t, wave_max(fabsf(d))) >> 23), 1);
                if (lane == 0) {
                    v_bad[wave] = who;
                    if constexpr (NB == 4) v_exp[wave] = e;
                    else v_exp[2 * (wave - 2)] = v_exp[2 * (wave - 2) + 1] = e;
                }
                // a scale of 11 bits times a quant of 8: an f16 and what it leaves, which is an f16 too
                const _Float16 x = (_Float16)__builtin_amdgcn_ldexpf(d, 127 + V_SHIFT - e);
                const half2v x2 = {x, x};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const half8 q = quants8(qw[2 * i], qw[2 * i + 1]);
                    half8 h, r;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const half2v q2 = {q[j], q[j + 1]}, h2 = q2 * x2, r2 = __builtin_elementwise_fma(q2, x2, -h2);
                        h[j] = h2[0], h[j + 1] = h2[1];
                        r[j] = r2[0], r[j + 1] = r2[1];
                    }
                    const int at = u_row * T::ROW + 16 * pv_slot<HD>(u_row, 4 * u_blk + i);
                    *reinterpret_cast<half8 *>(&lds[SETS - 2][at]) = h;
                    *reinterpret_cast<half8 *>(&lds[SETS - 1][at]) = r;
                }
            } else {
                k_scale[u_blk][u_row] = d;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<half8 *>(&lds[0][u_row * T::ROW + 16 * pk_slot<HD>(u_row, 4 * u_blk + i)]) = quants8(qw[2 * i], qw[2 * i + 1]);
            }
        }
    };
    auto stage_f32 = [&]() {
        auto put = [&](const float (&x)[FPT], uint8_t *hi, uint8_t *lo, bool v) {
#pragma unroll
            for (int i = 0; i < FPT; i += 4) {
                half2v h0, h1, r0, r1;
                split2_f16(x[i], x[i + 1], h0, r0);
                split2_f16(x[i + 2], x[i + 3], h1, r1);
                const int ch = i + u_blk / 2;
                const int at = u_row * T::ROW + 16 * (v ? pv_slot<HD>(u_row, ch) : pk_slot<HD>(u_row, ch)) + 8 * (u_blk & 1);
                *reinterpret_cast<half4 *>(hi + at) = half4{h0[0], h0[1], h1[0], h1[1]};
                *reinterpret_cast<half4 *>(lo + at) = half4{r0[0], r0[1], r1[0], r1[1]};
            }
        };
        float x[FPT], amax = 0.0f, down, up;
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            x[i] = __builtin_bit_cast(float, raw[0][i]);
            amax = fmaxf(amax, fabsf(x[i]));
        }
        amax = fmaxf(amax, dpp_row<0xB1>(amax));  // the row's eight lanes
        amax = fmaxf(amax, dpp_row<0x4E>(amax));
        amax = fmaxf(amax, dpp_row<0x141>(amax));
        row_exponent(amax, down, up);
        if (u_blk == 0) k_scale[0][u_row] = up;
#pragma unroll
        for (int i = 0; i < FPT; ++i) x[i] *= down;
        put(x, lds[0], lds[1], false);
        uint32_t bits = 0;
        amax = 0.0f;
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            x[i] = __builtin_bit_cast(float, raw[UN - 1][i]);
            const bool bad = !(fabsf(x[i]) < INFINITY);
            bits |= (bad ? 1u : 0u) << i;
            x[i] = bad ? 0.0f : x[i];
            amax = fmaxf(amax, fabsf(x[i]));
        }
        const uint64_t who = __ballot(bits != 0);
        const int e = max((int)(__builtin_bit_cast(uint32_t, wave_max(amax)) >> 23), 1);
        if (lane == 0) v_bad[wave] = who, v_exp[wave] = e;
        if (who != 0) v_bits[threadIdx.x] = (uint16_t)bits;
#pragma unroll
        for (int i = 0; i < FPT; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], 127 + V_SHIFT - e);
        put(x, lds[SETS - 2], lds[SETS - 1], true);
    };

    // probabilities are 2^(s f - base), base kSplitShift below the row's running
    // maximum; l sums this lane's; o is in units of 2^(unit_exp - 127 - V_SHIFT),
    // unit_exp the exponent of the largest of V so far
    float base = -INFINITY, l = 0.0f;
    uint64_t bad = 0;
    int unit_exp = 1;
    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    struct Two {
        half8 hi, lo;
    };

    Src src = {}, next = {};
    if (b.t0 < b.t1) src = issue(b.t0);
    for (int t = b.t0; t < b.t1; ++t, src = next) {
        __syncthreads();  // the last tile has been read
        if constexpr (kQ8) stage_q8();
        else stage_f32();
        if (t + 1 < b.t1) next = issue(t + 1);
        __syncthreads();
        if (!b.wave_ok || !src.there) continue;
        // This lane's first operand addresses; a step's are these with its chunk
        // XORed in (the slots are XORs too) and its rows added.  The empty asm
        // keeps the compiler from holding every step's address over the loop.
        const int li = lane & 15, vr = 4 * hh + (li >> 2);
        int k_at = n * T::ROW + 16 * pk_slot<HD>(n, hh);
        int v_at = vr * T::ROW + 16 * pv_slot<HD>(vr, 2 * (lane >> 4 & 1) + ((li & 3) >> 1)) + 8 * (li & 1);
        asm("" : "+v"(k_at), "+v"(v_at));

        floatx16 s[PB];
#pragma unroll
        for (int x = 0; x < PB; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
        if constexpr (!kQ8) {
            pipelined<KC, 1, FENCE>(
                [&](int c) {
                    const uint8_t *const at = &lds[0][0] + (k_at ^ (32 * c));
                    return Two{*reinterpret_cast<const half8 *>(at), *reinterpret_cast<const half8 *>(at + T::BYTES)};
                },
                [&](int c, Two a) {
                    s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.hi, qh[c], s[0], 0, 0, 0);
                    s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.hi, ql[c], s[0], 0, 0, 0);
                    s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.lo, qh[c], s[0], 0, 0, 0);
                });
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const floatx4 d = *reinterpret_cast<const floatx4 *>(&k_scale[0][8 * i4 + 4 * hh]);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[0][4 * i4 + j] *= d[j];
            }
        } else {
            // two steps a block, then the block's scales
            floatx16 x;
            pipelined<KC * PB, 2, FENCE>(
                [&](int i) {
                    const int blk = i / 2 % PB, c = i / (2 * PB) * 2 + i % 2;
                    return *reinterpret_cast<const half8 *>(&lds[0][0] + (k_at ^ (32 * c)) + blk * 32 * T::ROW);
                },
                [&](int i, half8 a) {
                    const int blk = i / 2 % PB, nb = i / (2 * PB), c = 2 * nb + i % 2;
                    if (i % 2 == 0)
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = 0.0f;
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], x, 0, 0, 0);
                    if (i % 2 == 0) return;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const floatx4 d = *reinterpret_cast<const floatx4 *>(&k_scale[nb][32 * blk + 8 * i4 + 4 * hh]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[blk][4 * i4 + j] = fmaf(x[4 * i4 + j], d[j], s[blk][4 * i4 + j]);
                    }
                });
        }
        if (src.masked) mask_scores<PB>(p, src, b.tpos, hh, s);
        float mx = -INFINITY, ma, mb;
#pragma unroll
        for (int x = 0; x < PB; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[x][i]);
        swap_halves(mx, ma, mb);
        mx = fmaxf(ma, mb) * f - (float)kSplitShift;
        int exps[4], e = unit_exp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            exps[i] = __builtin_amdgcn_readfirstlane(v_exp[i]);
            e = max(e, exps[i]);
        }
        if (__ballot(mx > base) != 0 || e > unit_exp) {
            const float nb = fmaxf(mx, base);
            const float a = nb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - nb);
            const float a_o = __builtin_amdgcn_ldexpf(a, unit_exp - e);
            l *= a;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= a_o;
            base = nb;
            unit_exp = e;
        }
        const float sub = base == -INFINITY ? 0.0f : base;
        half8 ph[ST], pl[ST];
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int i = 8 * st + j;
                const float u = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16], f, -sub));
                const float v = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16 + 1], f, -sub));
                l += u + v;
                // to the units of o, by a power of two: F32: values j < 4 are of positions 16 st .. + 7
                const int w = exps[kQ8 ? st : 2 * st + j / 4] - unit_exp;
                half2v h, r;
                split2_f16(__builtin_amdgcn_ldexpf(u, w), __builtin_amdgcn_ldexpf(v, w), h, r);
                ph[st][j] = h[0], ph[st][j + 1] = h[1];
                pl[st][j] = r[0], pl[st][j + 1] = r[1];
            }
        // operand of step st: positions 16 st + 4 hh .. and 16 st + 8 + 4 hh .., the lane's own
        // scores; four values a read, lane i of 16 gets dim i of the four rows its group names
        auto v_read = [&](int set, int st, int d) {
            const uint8_t *const at = &lds[set][0] + (v_at ^ (64 * d)) + 16 * st * T::ROW;
            const half4 x = tr16_read(at), y = tr16_read(at + 8 * T::ROW);
            return half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        };
        pipelined<ST * DB, 1, FENCE>([&](int i) { return Two{v_read(SETS - 2, i / DB, i % DB), v_read(SETS - 1, i / DB, i % DB)}; },
                                     [&](int i, Two a) {
                                         const int st = i / DB, d = i % DB;
                                         o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.hi, ph[st], o[d], 0, 0, 0);
                                         o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.hi, pl[st], o[d], 0, 0, 0);
                                         o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.lo, ph[st], o[d], 0, 0, 0);
                                     });
        if constexpr (kQ8) {
            // units of V: NB / 2 * 128 of them in the waves that hold V
            constexpr int W0 = NB == 4 ? 0 : 2;
            if (__ballot((v_bad[W0] | v_bad[W0 + 1] | v_bad[2] | v_bad[3]) != 0) != 0)
                bad |= spoiled<HD>(p, src, b.tpos, hh, [&](int r, int e) {
                    const int u = r * NB + e / kQK;
                    return v_bad[W0 + u / 64] >> u % 64 & 1;
                });
        } else {
            if (any_bad(v_bad))
                bad |= spoiled<HD>(p, src, b.tpos, hh, [&](int r, int e) {
                    const int th = r * 8 + e % 32 / 4;
                    return (v_bad[th / 64] >> th % 64 & 1) & (v_bits[th] >> (e / 32 * 4 + e % 4) & 1);
                });
        }
    }
    store_row<HD>(p, b, hh, o, base, l, __builtin_amdgcn_ldexpf(1.0f, unit_exp - 127 - V_SHIFT), bad);
}

// Workgroups that share a row block's tiles: the number with the least estimated
// time.  A tile takes `tile` us where a CU has one workgroup, `pair` times that
// where two share it (and in proportion beyond); every split writes and reads
// its rows' records, at 3.5 TB/s.  Measured (us; 32 / 8 heads of 128): F16 93
// tokens on 20100, window 4096: 146 / 50 / 36 / 35 with 1 / 4 / 10 / 21; Q8_0
// 777 on 6000, window 1024: 90 / 78 / 87 with 1 / 2 / 3; F32 (16 / 4 heads) 1500
// tokens, window 512: 54 / 51 / 56 with 1 / 2 / 4.
int window_prefill_splits(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T, int32_t window, int32_t n_sink) {
    const bool f32 = kv->kv_type == SFA_KV_F32, f16 = kv->kv_type == SFA_KV_F16;
    const int tp = f32 ? 32 : 64, g = kv->n_head / kv->n_head_kv;
    const double tile = (f16 ? 2.5 : f32 ? 3.7 : 5.1) * kv->head_dim / 128, pair = f16 ? 1.6 : 1.4;
    const int64_t blocks = ((int64_t)T * g + kRows - 1) / kRows * kv->n_head_kv;
    const int64_t span = (int64_t)window + kRows / g + n_sink, end = (int64_t)q_pos0 + T;
    const int64_t tiles = ((span < end ? span : end) + tp - 1) / tp;
    const double record = 2.0 * T * kv->n_head * kv->head_dim * 4 / 3.5e6;
    int best = 1;
    double least = 0.0;
    for (int n = 1; n <= kMostSplits && n <= tiles && (n == 1 || blocks * n <= kMostBlocks); ++n) {
        const int64_t cu = (blocks * n + 255) / 256;
        const double us = (double)((tiles + n - 1) / n) * tile * (cu == 1 ? 1.0 : pair * cu / 2) + (n > 1 ? 3.0 + n * record : 0.0);
        if (n == 1 || us < least) {
            least = us;
            best = n;
        }
    }
    return best;
}

// The most (row, split) records that a call of up to max_T tokens may write.
int64_t window_prefill_most_records(const sfa_kv_desc *kv, int32_t max_T) {
    const int g = kv->n_head / kv->n_head_kv;
    int64_t most = 0;
    // the splits allowed fall where a row block is added: the last T of a block count
    for (int64_t block = 1;; ++block) {
        const int64_t T = block * kRows / g < max_T ? block * kRows / g : max_T;
        int64_t n = kMostBlocks / (block * kv->n_head_kv);
        n = n > kMostSplits ? kMostSplits : n;
        if (n > 1 && T * kv->n_head * n > most) most = T * kv->n_head * n;
        if (n <= 1 || T == max_T) return most;
    }
}

template <int KVT, int HD>
static void launch_g(const WindowParams &p, dim3 grid, hipStream_t s) {
    const dim3 block(256);
    if constexpr (KVT == SFA_KV_F16) {
        switch (p.n_head / p.n_head_kv) {
        case 1: hipLaunchKernelGGL((window_prefill_f16_kernel<HD, 1>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((window_prefill_f16_kernel<HD, 2>), grid, block, 0, s, p); break;
        case 4: hipLaunchKernelGGL((window_prefill_f16_kernel<HD, 4>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((window_prefill_f16_kernel<HD, 8>), grid, block, 0, s, p); break;
        }
        return;
    } else
    switch (p.n_head / p.n_head_kv) {
    case 1: hipLaunchKernelGGL((window_prefill_wide_kernel<KVT, HD, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((window_prefill_wide_kernel<KVT, HD, 2>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((window_prefill_wide_kernel<KVT, HD, 4>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((window_prefill_wide_kernel<KVT, HD, 8>), grid, block, 0, s, p); break;
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
