// What the kernels over the 4-bit key/value cache share: the view of the cache, integers and scales out of its bytes, where a row lies.
//
// A value is n s g: n + 8 in 4 bits, s in e4m3 for 16 dims of a row, g in f32 for a kv head.  n s has 8 bits and is exact in f16, so the products of queries and weights with the cache lose
// nothing on the cache's side; g goes into the scores' factor and into what the sums are multiplied by at the end.
#pragma once
#include "lc_kv8.cuh"

namespace lc {

// k, v: two integers to a byte; k_scale, v_scale: [n_kv]
struct Kv4Pool : Kv8Pool {
    uint8_t* k_block;
    uint8_t* v_block;
};
// kv4.cu: the arguments that all calls over the cache have
int32_t kv4_check(const char* call, const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, Kv4Pool* view, Kv8Seqs* seqs);

struct AttnArgs;
struct TilePlan;
// attention_kv4_tiles.cu: many rows per sequence, by the plan of kv8_tiles_plan
int32_t launch_kv4_tiles(const Kv4Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const TilePlan& plan, cudaStream_t s);

constexpr float kUnit4 = 8.0f;  // what the f16 values below are to be multiplied by

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_fma4(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t h2_const(uint32_t bits) { return bits | bits << 16; }
// Two block scales (bytes, in bits 0-6 and 16-22 of b) as what turns 4 bits into values.  The byte's bits, 7 up, are the f16 number s / 256 (f16's exponent is 8 larger, and what has none means the
// same in both).  0x6400 | u is 1024 + u and 0x6400 | 16 u is 1024 + 16 u, so one multiplication and addition gives (u - 8) s / 8, whose 8 bits are exact, as is every constant here: 1032 = 8 x 129,
// and 129 times a scale's 4 bits are at most 1935.
struct Scale4 {
    uint32_t lo, lo_less, hi, hi_less;   // s / 8, -1032 s / 8; s / 128, -72 s / 8
};
__device__ __forceinline__ Scale4 scale4(uint32_t b) {
    const uint32_t raw = (b & 0x007f007fu) << 7;
    Scale4 r;
    r.lo = h2_mul(raw, h2_const(0x5000));        // 32
    r.lo_less = h2_mul(raw, h2_const(0xf808));   // -33024
    r.hi = h2_mul(raw, h2_const(0x4000));        // 2
    r.hi_less = h2_mul(raw, h2_const(0xe880));   // -2304
    return r;
}
// the integers in bits 0-3 and 16-19, 4-7 and 20-23 of x (and 8 higher, after a shift) as values
__device__ __forceinline__ uint32_t value_lo(uint32_t x, const Scale4& s) { return h2_fma4((x & 0x000f000fu) | 0x64006400u, s.lo, s.lo_less); }
__device__ __forceinline__ uint32_t value_hi(uint32_t x, const Scale4& s) { return h2_fma4((x & 0x00f000f0u) | 0x64006400u, s.hi, s.hi_less); }
// eight neighbouring dims: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void values8(uint32_t x, const Scale4& s, uint32_t (&v)[4]) {
    v[0] = value_lo(x, s);
    v[1] = value_hi(x, s);
    v[2] = value_lo(x >> 8, s);
    v[3] = value_hi(x >> 8, s);
}
template <int N> __device__ __forceinline__ void lds_words(const unsigned char* p, uint32_t (&w)[N]) {  // N: 1, 2, 4 or 8 words, aligned to 16 bytes or their size
    if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
    }
}
// the same, aligned to 8 bytes
template <int N> __device__ __forceinline__ void lds_words8(const unsigned char* p, uint32_t (&w)[N]) {
    if constexpr (N <= 2) lds_words<N>(p, w);
    else
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 u = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = u.x; w[2 * i + 1] = u.y;
        }
}

// a block scale as a number
__device__ __forceinline__ float scale4_f(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)((b & 0x7fu) << 7))) * 256.0f; }

// A row of the call: its sequence (-1: none, or one that leaves its table), page (-1: outside the pool) and slot in it, position.
struct RowPlace {
    int seq, page, slot, index;   // index: of the row within its sequence
};
// By one whole warp.
__device__ __forceinline__ RowPlace row_place(const Kv8Seqs& s, const Kv8Pool& p, int r) {
    RowPlace at;
    int next, first, n;
    at.seq = kv8_seq_of_row(s, r, next);
    at.page = at.slot = -1;
    at.index = 0;
    if (at.seq < 0) return at;
    kv8_span(s, at.seq, first, n);
    const int ctx = s.ctx[at.seq];
    at.index = r - first;
    if (!kv8_in_table(s, p, ctx, n)) return at;
    const int place = ctx + at.index, number = s.table[(size_t)at.seq * s.width + (place >> p.page_shift)];
    at.slot = place & ((1 << p.page_shift) - 1);
    at.page = number >= 0 && number < p.n_pages ? number : -1;
    return at;
}
#endif

}  // namespace lc
