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
// What a row's scores are multiplied by: the scale times log2 e, what undoes the row's power of two, the head's scale.  0 as 2^-100, so that a masked score of minus infinity stays one; beyond f32, where a
// row of zeros has no power of two that brings it back, as f32's largest: its scores stay 0.
__device__ __forceinline__ float score_factor(float scale_log2, float down, float head) {
    const float f = max_nan(scale_log2 * down * head, 0x1p-100f);
    return f == INFINITY ? 0x1.fffffep127f : f;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_fma4(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t h2_const(uint32_t bits) { return bits | bits << 16; }
// Block scales as what turns 4 bits into values.  A byte's bits, 7 up, are the f16 number s / 256 (f16's exponent is 8 larger, and what has none means the same in both).  0x6400 | u is
// 1024 + u and 0x5400 | 16 u is 64 + u, so one multiplication and addition gives (u - 8) s / 8, whose 8 bits are exact, as is every constant here: 1032 = 8 x 129, and 129 times a scale's 4 bits are at
// most 1935.
struct Scale4 {
    uint32_t by, lo_less, hi_less;   // s / 8, -1032 s / 8, -72 s / 8
};
__device__ __forceinline__ Scale4 scale4_of(uint32_t raw) {   // two numbers s / 256
    Scale4 r;
    r.by = h2_mul(raw, h2_const(0x5000));        // 32
    r.lo_less = h2_mul(raw, h2_const(0xf808));   // -33024
    r.hi_less = h2_mul(raw, h2_const(0xe880));   // -2304
    return r;
}
// byte j of b, twice (its top bit is not looked at); b has no top bits: b & 0x7f7f7f7f
__device__ __forceinline__ Scale4 scale4_both(uint32_t b, int j) { return scale4_of(__byte_perm(b, 0, j * 0x0101 + 0x4040) * 128u); }
// two keys' scales, a byte each
__device__ __forceinline__ Scale4 scale4_pair(uint32_t a, uint32_t b) { return scale4_of((a * 128u + b * 0x800000u) & 0x3f803f80u); }
// the integers in bits 0-3 and 16-19, 4-7 and 20-23 of x (and 8 higher, after a shift) as values
// (x & keep) | with, in one instruction: left to itself the compiler takes two
template <uint32_t KEEP> __device__ __forceinline__ uint32_t bits_with(uint32_t x, uint32_t with) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(KEEP), "r"(with));
    return r;
}
__device__ __forceinline__ uint32_t value_lo(uint32_t x, const Scale4& s) { return h2_fma4(bits_with<0x000f000fu>(x, 0x64006400u), s.by, s.lo_less); }
__device__ __forceinline__ uint32_t value_hi(uint32_t x, const Scale4& s) { return h2_fma4(bits_with<0x00f000f0u>(x, 0x54005400u), s.by, s.hi_less); }
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

// Keys (and values) of a warp's steps of 16, through a ring of S places in shared memory of its own.  A place has the keys' bytes, the values', and their scales' (HD bytes each).
// Which pages the steps lie on is looked up for 32 of them at a time, one per lane; a page outside the pool is not copied, and `any_bad` then says that some step has one.
template <int HD, bool FULL, bool VALUES, int S>
struct Ring4 {
    static_assert((S & (S - 1)) == 0, "places are counted with a mask");
    static constexpr int kRows = 16, kHalf = kRows * HD / 2, kScales = (VALUES ? 2 : 1) * kHalf, kPlace = kScales + (VALUES ? 2 : 1) * HD;
    static constexpr int KW = HD / 32;
    static constexpr uint32_t kBad = 0xffffffffu;
    const Kv4Pool& pool;
    const int hd;
    const int32_t* table;
    const int8_t* k_from;         // the lane's part of row 0
    const int8_t* v_from;
    const uint8_t* s_from;
    uint32_t to, v_to, s_to;      // the lane's places in the ring; of its scales: 0 where it has none
    uint32_t where = kBad;        // of step (at + lane): the number of its 16 rows in the pools
    int step0, end, kvh, lane;
    bool any_bad = false;

    __device__ __forceinline__ Ring4(const Kv4Pool& p, int hd_, const int32_t* t, int kvh_, int step0_, uint32_t smem, int lane_)
        : pool(p), hd(hd_), table(t), step0(step0_), kvh(kvh_), lane(lane_) {
        k_from = pool.k + lane * 16;
        v_from = pool.v + lane * 16;
        to = smem + lane * 16;
        v_to = smem + kHalf + (FULL ? value_chunk(lane / KW, lane % KW) : lane) * 16;
        const int pieces = hd >> 4;
        const bool v = VALUES && lane >= pieces;
        s_from = (v ? pool.v_block : pool.k_block) + (v ? lane - pieces : lane) * 16;
        s_to = lane < (VALUES ? 2 : 1) * pieces ? smem + kScales + (v ? HD : 0) + (v ? lane - pieces : lane) * 16 : 0;
    }
    // Where values' 16-byte chunk ch of row r lies (in chunks), so that the threads of a quad, whose keys are 2c, 2c + 1, 8 + 2c, 9 + 2c, read other banks: rows in the
    // order of the quads, and chunks swapped where two of these rows begin at the same bank.
    static __device__ __forceinline__ int value_chunk(int r, int ch) {
        const int slot = (r >> 1) + (r & 1) * 8;
        return slot * KW + (HD == 256 ? ch ^ ((slot & 3) * 2) : HD == 128 ? ch ^ (slot & 2) : ch);
    }
    __device__ __forceinline__ int page_of(int st) const { return table[((step0 + st) * kRows) >> pool.page_shift]; }
    __device__ __forceinline__ bool outside(int st) const {  // for the steps that the warp has begun
        const int number = page_of(st);
        return number < 0 || number >= pool.n_pages;
    }
    // steps at .. at + 31; true where some page is outside the pool
    __device__ __forceinline__ bool look_up(int first, int at) {
        const int st = at + lane;
        where = kBad;
        bool bad = false;
        if (st >= first && st < end) {
            const int number = page_of(st);
            bad = number < 0 || number >= pool.n_pages;
            if (!bad) where = (((uint32_t)number * (uint32_t)pool.n_kv + (uint32_t)kvh) << (pool.page_shift - 4)) + (((uint32_t)(step0 + st) * kRows & ((1u << pool.page_shift) - 1)) >> 4);
        }
        bad = __any_sync(0xffffffffu, bad);
        any_bad = any_bad || bad;
        return bad;
    }
    __device__ __forceinline__ bool begin(int first, int end_) {
        end = end_;
        return look_up(first, first & ~31);
    }
    // a commit for every step, whether it is there or not; true where a page outside the pool was met
    __device__ __forceinline__ bool fetch(int st, bool first = false) {
        bool bad = false;
        if (!first && (st & 31) == 0) bad = look_up(st, st);
        const uint32_t row16 = __shfl_sync(0xffffffffu, where, st & 31);
        if (st < end && row16 != kBad) {
            const uint32_t place = (uint32_t)(st & (S - 1)) * kPlace;
            const int8_t* const ks = k_from + (uint64_t)row16 * (uint32_t)(8 * hd);
            const int8_t* const vs = v_from + (uint64_t)row16 * (uint32_t)(8 * hd);
            if (FULL) {
#pragma unroll
                for (int i = 0; i < KW * kRows / 32; i++) {
                    cp16(to + place + i * 512, ks + i * 512);
                    if (VALUES) {
                        // chunk i * 32 + lane: for HD of 64 and 128 the lane's row plus an even number, whose places are a constant apart
                        if (HD == 256) cp16(v_to - (uint32_t)value_chunk(lane / KW, lane % KW) * 16 + (uint32_t)value_chunk((i * 32 + lane) / KW, lane % KW) * 16 + place, vs + i * 512);
                        else cp16(v_to + place + i * (value_chunk(8, 0) * 16), vs + i * 512);
                    }
                }
            } else {
                for (int ch = 0; ch < hd >> 1; ch += 32)
                    if (ch + lane < hd >> 1) {
                        cp16(to + place + ch * 16, ks + ch * 16);
                        if (VALUES) cp16(v_to + place + ch * 16, vs + ch * 16);
                    }
            }
            if (s_to) cp16(s_to + place, s_from + (uint64_t)row16 * (uint32_t)hd);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return bad;
    }
    static __device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
};

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
