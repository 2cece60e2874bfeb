// What the two attention kernels over the 8-bit key/value cache share: arguments, operands of the matrix unit, the units of a call.
#pragma once
#include <algorithm>
#include "lc_kv8.cuh"
#include "lc_tma.cuh"

namespace lc {

struct AttnArgs {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int typ, group, window;
    bool q_vec, out_vec;             // 16-byte accesses
    float scale_log2;                // scale * log2(e)
    float* part;                     // partial results of runs that end inside a unit
    struct UnitRecord* records;      // one per run: the unit that begins in it and goes on behind it
    float* lse = nullptr;            // ln sum exp of the rows' scores, or null; the weights that were summed are 2^lse_less too large
    int64_t lse_stride = 0;
    float lse_less = 0.0f;
};
struct __align__(16) UnitRecord {
    int first, kvh, row_lo, row_n;   // the sequence's first row, kv head, rows; row_n 0: none
    int last, pad0, pad1, pad2;      // the run with the unit's end
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same from nothing
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// 16 x 8 sums of 32 products of integers of 8 bits, exact in 32
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ uint32_t h2_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) as f16 and what that rounding lost, as f16
__device__ __forceinline__ void h2_split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = h2_pack(a - __low2float(h), b - __high2float(h));
}
// Bytes 0, 1 (or 2, 3) of x = integers + 128 as f16 integers + 1152: 0x64 is the high byte of 1024.0, and 1152 = 1024 + 128; then without the 1152.
__device__ __forceinline__ uint32_t biased01(uint32_t x) { return __byte_perm(x, 0x64646464u, 0x4140u); }
__device__ __forceinline__ uint32_t biased23(uint32_t x) { return __byte_perm(x, 0x64646464u, 0x4342u); }
__device__ __forceinline__ uint32_t minus_1152(uint32_t v) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t ints01(uint32_t x) { return minus_1152(biased01(x)); }
__device__ __forceinline__ uint32_t ints23(uint32_t x) { return minus_1152(biased23(x)); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// sixteen elements in a row as f32, and back
template <typename T> __device__ __forceinline__ void load16(const T* p, bool vec, float* v) {
    constexpr int E = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int u = 0; u < 16 / E; u++) {
            __align__(16) T t[E];
            *reinterpret_cast<uint4*>(t) = reinterpret_cast<const uint4*>(p)[u];
#pragma unroll
            for (int e = 0; e < E; e++) v[u * E + e] = elem_f(t[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = elem_f(p[e]);
    }
}
__device__ __forceinline__ void load16(const void* p, int64_t at, int typ, bool vec, float* v) {
    if (typ == LC_TYPE_F32) load16((const float*)p + at, vec, v);
    else if (typ == LC_TYPE_F16) load16((const __half*)p + at, vec, v);
    else load16((const __nv_bfloat16*)p + at, vec, v);
}
template <int N, typename T> __device__ __forceinline__ void store_run(T* p, bool vec, const float* v) {
    constexpr int E = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int u = 0; u < N / E; u++) {
            __align__(16) T t[E];
#pragma unroll
            for (int e = 0; e < E; e++) t[e] = to_elem<T>(v[u * E + e]);
            reinterpret_cast<uint4*>(p)[u] = *reinterpret_cast<const uint4*>(t);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = to_elem<T>(v[e]);
    }
}
template <int N> __device__ __forceinline__ void store_run(void* p, int64_t at, int typ, bool vec, const float* v) {
    if (typ == LC_TYPE_F32) store_run<N>((float*)p + at, vec, v);
    else if (typ == LC_TYPE_F16) store_run<N>((__half*)p + at, vec, v);
    else store_run<N>((__nv_bfloat16*)p + at, vec, v);
}
__device__ __forceinline__ void store16(float* p, bool vec, const float* v) { store_run<16>(p, vec, v); }
__device__ __forceinline__ void store16(void* p, int64_t at, int typ, bool vec, const float* v) { store_run<16>(p, at, typ, vec, v); }
__device__ __forceinline__ void store1(void* p, int64_t at, int typ, float v) {
    if (typ == LC_TYPE_F32) ((float*)p)[at] = v;
    else if (typ == LC_TYPE_F16) ((__half*)p)[at] = to_elem<__half>(v);
    else ((__nv_bfloat16*)p)[at] = to_elem<__nv_bfloat16>(v);
}
// a power of two that brings the largest magnitude of a row into [2^14, 2^15), and its inverse; 1 for a row of zeros or with infinities
__device__ __forceinline__ void row_scale(float top, float& up, float& down) {
    const int e = (__float_as_int(top) >> 23) & 0xff;
    int s = 127 + 14 - (e - 127);
    s = s < 1 ? 1 : s > 253 ? 253 : s;
    if (top == 0.0f || e == 255) s = 127;
    up = __int_as_float(s << 23);
    down = __int_as_float((254 - s) << 23);
}

constexpr float kNegInf = -INFINITY;
constexpr int kStep = 16;            // keys of a step of the line: one page's, or a part of one page's
constexpr int kUnitCost = 4;         // steps that a unit's beginning and end take as long as

// A unit is (sequence, kv head, row block of RB rows = tokens x heads of the group).
struct SeqWork {
    int first, n, ctx, blocks, step0, steps;  // rows, context, row blocks, first step, steps per unit
    bool inside;
};
template <int RB>
__device__ __forceinline__ SeqWork seq_work(const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, int i) {
    SeqWork w;
    w.inside = false;
    w.blocks = w.step0 = w.steps = 0;
    w.ctx = s.ctx[i];
    if (!kv8_span(s, i, w.first, w.n) || w.n == 0) { w.n = 0; return w; }
    w.blocks = (w.n * a.group + RB - 1) / RB;
    w.inside = kv8_in_table(s, p, w.ctx, w.n);
    if (w.inside) {
        const int lo = a.window > 0 ? max(0, w.ctx - a.window + 1) : 0;
        w.step0 = lo / kStep;
        w.steps = (w.ctx + w.n + kStep - 1) / kStep - w.step0;
    } else {
        w.steps = 1;  // one step that writes NaN
    }
    return w;
}
// Sums that stop at 2^31 - 1: the calls' checks keep those of ascending rows below it, and rows given to several sequences must not make a place of the line another's.
__device__ __forceinline__ uint32_t add_places(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }
// cum[i] = the line's places before sequence i (kUnitCost and its steps for every unit), cum[n_seqs] = all; units[i] (if wanted) the units before i; by one block, returns the total
template <int RB>
__device__ __forceinline__ uint32_t line_up(const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, uint32_t* cum, uint32_t* units, uint2* warp_sums) {
    const int per = (s.n_seqs + blockDim.x - 1) / blockDim.x, i0 = min((int)threadIdx.x * per, s.n_seqs), i1 = min(i0 + per, s.n_seqs);
    uint32_t sum = 0, usum = 0;
    for (int i = i0; i < i1; i++) {
        const SeqWork w = seq_work<RB>(s, p, a, i);
        cum[i] = sum;
        if (units) units[i] = usum;
        sum = add_places(sum, (uint32_t)w.blocks * (uint32_t)p.n_kv * (uint32_t)(w.steps + kUnitCost));
        usum = add_places(usum, (uint32_t)w.blocks * (uint32_t)p.n_kv);
    }
    uint32_t incl = sum, uincl = usum;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o), u = __shfl_up_sync(0xffffffffu, uincl, o);
        if (lane >= o) { incl = add_places(incl, v); uincl = add_places(uincl, u); }
    }
    if (lane == 31) warp_sums[warp] = make_uint2(incl, uincl);
    __syncthreads();
    uint32_t before = __shfl_up_sync(0xffffffffu, incl, 1), ubefore = __shfl_up_sync(0xffffffffu, uincl, 1), total = 0, utotal = 0;
    if (lane == 0) before = ubefore = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        const uint2 v = warp_sums[w];
        if (w < warp) { before = add_places(before, v.x); ubefore = add_places(ubefore, v.y); }
        total = add_places(total, v.x);
        utotal = add_places(utotal, v.y);
    }
    for (int i = i0; i < i1; i++) {
        cum[i] = add_places(cum[i], before);
        if (units) units[i] = add_places(units[i], ubefore);
    }
    if (threadIdx.x == 0) {
        cum[s.n_seqs] = total;
        if (units) units[s.n_seqs] = utotal;
    }
    __syncthreads();
    return total;
}
__device__ __forceinline__ int seq_at(const uint32_t* cum, int n_seqs, uint32_t t) {  // the sequence that has place t
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}
constexpr int kRunWarps = 4;
// The line of `total` steps in equal runs, none of them empty, and none shorter than kLeast where that leaves warps without one.
constexpr uint32_t kLeast = 4;
struct Runs {
    uint32_t n, per, more;  // the first `more` runs have a step more than `per`
    __device__ __forceinline__ Runs(uint32_t total, uint32_t warps) {
        n = min((total + kLeast - 1) / kLeast, warps);
        per = n ? total / n : 0;
        more = total - per * n;
    }
    __device__ __forceinline__ uint32_t start(uint32_t b) const { return b * per + min(b, more); }
    __device__ __forceinline__ uint32_t run_of(uint32_t t) const {  // the run that step t is in
        const uint32_t longer = more * (per + 1);
        return t < longer ? t / (per + 1) : more + (t - longer) / per;
    }
};

// floats of one partial result: maxima, sums and rows of HD
template <int HD, int RB> __host__ __device__ constexpr int part_floats() { return RB * (HD + 2); }

// Where a place of the line lies: `in` of its unit, whose first kUnitCost places are no steps.
struct Place {
    int seq, kvh, rb, in;
    SeqWork w;
};
template <int RB>
__device__ __forceinline__ void place_at(Place& at, const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, const uint32_t* cum, uint32_t t) {
    at.seq = seq_at(cum, s.n_seqs, t);
    at.w = seq_work<RB>(s, p, a, at.seq);
    const uint32_t cost = at.w.steps + kUnitCost, in = t - cum[at.seq], unit = in / cost;
    at.in = in - unit * cost;
    at.kvh = unit / at.w.blocks;
    at.rb = unit - at.kvh * at.w.blocks;
}

// Whether the places of the line, with row blocks of so many rows, are sure to stay in 31 bits: every context as long as its table.
inline bool line_fits(const Kv8Pool& pool, const Kv8Seqs& seqs, int group, int block_rows) {
    const double steps = (double)((int64_t)seqs.width << pool.page_shift) / kStep + 2 + kUnitCost;
    const double blocks = (double)seqs.n_rows * group / block_rows + std::min(seqs.n_seqs, seqs.n_rows);
    return steps * blocks * pool.n_kv < 2147483648.0;
}
// attention_kv8_tiles.cu: many rows per sequence, in tiles of 256 rows on tcgen05; heads of up to 128
constexpr int kTileRows2 = 256;       // of a unit
struct TilePlan {
    int units, splits;               // blocks: at most so many units; every unit's keys in so many parts
    size_t bytes;
};
bool kv8_tiles_plan(const Kv8Pool& pool, const Kv8Seqs& seqs, int group, TilePlan* plan);                                                          // whether they can
bool kv8_tiles_pay(const Kv8Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows, const TilePlan& plan);                          // whether they are faster
size_t kv8_tiles_most_bytes(const Kv8Pool& pool, int64_t rows);                                                                                     // of any call with at most so many rows (tokens x heads of a group) per sequence
int32_t launch_kv8_tiles(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const TilePlan& plan, cudaStream_t s);

}  // namespace lc
