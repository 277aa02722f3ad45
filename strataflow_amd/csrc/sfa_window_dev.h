// sfa_window_dev.h - parameters and device helpers of the windowed attention
// kernels (sfa_window_decode.hip, sfa_window_prefill.hip).
#pragma once

#include "sfa_common.h"
#include "sfa_window.h"

namespace sfa {

// Both factors that are split into two f16 are scaled up first, the row of
// queries and the probabilities to 2^14: the lower half of a value 2^17 times
// smaller than the largest is a normal f16 then (the matrix cores need not
// keep subnormal ones).
constexpr int kSplitShift = 14;

struct WindowParams {
    const float *q;
    float *out;
    const uint8_t *k_pages, *v_pages, *k_cold, *v_cold;
    int64_t page_bytes;
    int n_pages, n_cold, page_size, max_pages;
    int page_shift;          // log2(page_size), -1 where there is none
    int n_head, n_head_kv, row_bytes;
    const int32_t *page_table;
    const int32_t *seq_len;  // decode; null for a chunk
    int q_pos0;              // chunk
    int n_tok;               // of the chunk; decode: sequences
    int window, n_sink;
    float scale_log2;        // scale * log2(e): probabilities are powers of two
    int n_split;
    float *rec_o;            // split records: outputs [row][split][HD] not yet divided,
    float2 *rec_ml;          // and (running maximum, sum) [row][split]
};

int window_decode_splits(const sfa_kv_desc *kv, int32_t B, int32_t max_seq_len, int32_t window, int32_t n_sink);
int window_decode_launch(const WindowParams &p, const sfa_kv_desc *kv, int32_t B, hipStream_t s);
int window_prefill_splits(const sfa_kv_desc *kv, int32_t q_pos0, int32_t T, int32_t window, int32_t n_sink);
int64_t window_prefill_most_records(const sfa_kv_desc *kv, int32_t max_T);
int window_prefill_launch(const WindowParams &p, const sfa_kv_desc *kv, hipStream_t s);
int window_merge_launch(const WindowParams &p, int head_dim, int64_t rows, hipStream_t s);

// x, the same in every lane, in a scalar register.  Without the empty asm the
// compiler drops the readfirstlane of a value that it knows to be uniform and
// may keep what follows in vector registers, where the operands of load_to_lds
// cannot be.
__device__ inline uint32_t to_scalar(uint32_t x) {
    asm("" : "+v"(x));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// The tiles of a split: n / splits, and one more for the first n % splits.
// (Divisions run on the vector side: back to scalars, for scalar branches.)
__device__ inline void split_range(int n, int split, int splits, int &t0, int &t1) {
    const int each = (int)to_scalar((uint32_t)n / (uint32_t)splits), more = n - each * splits;
    t0 = split * each + min(split, more);
    t1 = t0 + each + (split < more ? 1 : 0);
}

// Tiles of n positions from a tile's first one (n up to INT32_MAX).
__device__ inline int tiles_of(int n, int tp) { return n / tp + (n % tp != 0); }

// Factor of the scores in the exponent of two, under a row's power of two
// (row_exponent).  Never zero: a masked score stays -inf.  (Where it would be,
// the row's scores differ by less than 2^-80.)
__device__ inline float score_factor(float scale_log2, float up) { return fmaxf(scale_log2 * up, 0x1p-126f); }

// Logical page of a position.
__device__ inline int page_of(const WindowParams &p, int pos) {
    return p.page_shift >= 0 ? pos >> p.page_shift : (int)to_scalar((uint32_t)pos / (uint32_t)p.page_size);
}

// A raw buffer over [base, base + bytes): loads outside it give zeros, also
// those at "negative" offsets, which are large unsigned ones.
__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *base, int bytes) {
    const uint64_t u = reinterpret_cast<uint64_t>(base);
    uint32_t lo = to_scalar((uint32_t)u), hi = to_scalar((uint32_t)(u >> 32)), n = to_scalar((uint32_t)bytes);
    // a load may read a scalar register five states after a vector instruction
    // wrote it, and the compiler does not see the load in load_to_lds
    asm volatile("s_nop 4" : "+s"(lo), "+s"(hi), "+s"(n));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>((uint64_t)hi << 32 | lo), 0, (int)n, kBufferRsrcWord3);
}

__device__ inline uint32_t lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)p;
}

// 16 bytes a lane from a buffer straight into LDS at lds_base + 16 * lane.
// The compiler does not count these loads: the caller waits with wait_loads
// before it reads what they wrote.  M0 holds the LDS base.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // "m0 is reserved": the kernels use M0 for nothing else
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds_base, int offset) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(lds_base), "v"(offset), "s"(rsrc)
        : "memory", "m0");
}
#pragma clang diagnostic pop

// Waits until at most N of the wave's loads are in flight (they end in order).
template <int N>
__device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Maximum and sum over the lanes l % 16 + {0, 16, 32, 48}, in all four.
__device__ inline void swap_rows16(float x, float &a, float &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                    false, false);
    static_assert(sizeof(r) == 8, "two 32-bit values");
    unsigned u0, u1;
    __builtin_memcpy(&u0, reinterpret_cast<const char *>(&r), 4);
    __builtin_memcpy(&u1, reinterpret_cast<const char *>(&r) + 4, 4);
    a = __builtin_bit_cast(float, u0);
    b = __builtin_bit_cast(float, u1);
}
__device__ inline float quarters_max(float x) {
    float a, b;
    swap_rows16(x, a, b);
    x = fmaxf(a, b);
    swap_halves(x, a, b);
    return fmaxf(a, b);
}
__device__ inline float quarters_sum(float x) {
    float a, b;
    swap_rows16(x, a, b);
    x = a + b;
    swap_halves(x, a, b);
    return a + b;
}

// x as two f16: hi its nearest, lo the nearest of what is left.  The empty asm
// keeps a product that x comes from out of the conversions: fused with one of
// them only, it gave a hi and a lo of two different roundings now and then.
__device__ inline void split_f16(float x, _Float16 &hi, _Float16 &lo) {
    asm("" : "+v"(x));
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}

// Two values split so, in four instructions: what is left of x is h (-1) + x as
// a dot product with the pair, exact (the other half meets a zero).
__device__ inline void split2_f16(float x, float y, half2v &hi, half2v &lo) {
    const half2v h = {(_Float16)x, (_Float16)y};
    const half2v first = {(_Float16)-1.0f, (_Float16)0.0f}, second = {(_Float16)0.0f, (_Float16)-1.0f};
    hi = h;
    lo = half2v{(_Float16)__builtin_amdgcn_fdot2(h, first, x, false), (_Float16)__builtin_amdgcn_fdot2(h, second, y, false)};
}

// Power of two that takes a row's largest value into [2^14, 2^15), and its
// inverse.
__device__ inline void row_exponent(float amax, float &down, float &up) {
    int e = (int)(__builtin_bit_cast(uint32_t, amax) >> 23) & 255;
    e = e < kSplitShift + 2 ? kSplitShift + 2 : e > 252 ? 252 : e;  // zeros and the ends of the range
    down = __builtin_bit_cast(float, (uint32_t)(254 + kSplitShift - e) << 23);
    up = __builtin_bit_cast(float, (uint32_t)(e - kSplitShift) << 23);
}

// Quants as f16 (exact): byte b is 1024 + (b + 128) under the exponent of 1024.
__device__ inline half2v quants2(uint32_t two) {  // bytes 0 and 2, the others 0
    const half2v base = {(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(half2v, two ^ 0x64806480u) - base;
}
__device__ inline half8 quants8(uint32_t a, uint32_t b) {
    const half2v base = {(_Float16)1152.0f, (_Float16)1152.0f};
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t w[4] = {__builtin_amdgcn_perm(0x64646464u, a, 0x04010400), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402),
                           __builtin_amdgcn_perm(0x64646464u, b, 0x04010400), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402)};
    half8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2v h = __builtin_bit_cast(half2v, w[i]) - base;
        r[2 * i] = h[0], r[2 * i + 1] = h[1];
    }
    return r;
}

}  // namespace sfa
