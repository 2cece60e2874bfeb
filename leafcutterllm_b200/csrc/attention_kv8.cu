// Attention over the key/value cache in 8 bits: out = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the positions j up to the row's own.
//
// A cached element is q8 * S with one scale S per page and head, and an integer of 8 bits is exact in f16: scores and weighted sums are
// products on the matrix unit (mma.sync m16n8k16, f16 in, f32 out) of f16 integers with the queries and the weights, and the scales are
// applied outside, S_k to the scores and S_v to a block's sums.
//
// Queries are scaled by a power of two per row, so that their largest element is in [2^14, 2^15) whatever its size.  The weights are
// 2^(s - max + 8).  In the split form (RB = 8 rows to a tile of 16) rows 0 .. 7 of the tile hold the f16 value and rows 8 .. 15 what its
// rounding lost, 22 bits together: the two halves of a sum lie in the same thread.  In the plain form (RB = 16) a tile holds 16 rows, weights
// rounded to f16 (2^-12 of each).
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include "lc_tma.cuh"

namespace lc {

namespace {

constexpr int kStep = 16;            // keys of a warp's step: one page's, or a part of one page's
constexpr int kRunWarps = 4;
constexpr int kChunk = kStep * kRunWarps;  // keys of a block's step
constexpr float kNegInf = -INFINITY;

struct AttnArgs {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int n_heads, group, window;
    float scale_log2;                // scale * log2(e)
    float* part;                     // partial results of runs that end inside a unit
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// Bytes 0, 1 (or 2, 3) of x = integers + 128 as f16 integers: 0x64 is the high byte of 1024.0, and 1152 = 1024 + 128.
__device__ __forceinline__ uint32_t minus_1152(uint32_t v) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t ints01(uint32_t x) { return minus_1152(__byte_perm(x, 0x64646464u, 0x4140u)); }
__device__ __forceinline__ uint32_t ints23(uint32_t x) { return minus_1152(__byte_perm(x, 0x64646464u, 0x4342u)); }
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
// a power of two that brings the largest magnitude of a row into [2^14, 2^15), and its inverse; 1 for a row of zeros or with infinities
__device__ __forceinline__ void row_scale(float top, float& up, float& down) {
    const int e = (__float_as_int(top) >> 23) & 0xff;
    int s = 127 + 14 - (e - 127);
    s = s < 1 ? 1 : s > 253 ? 253 : s;
    if (top == 0.0f || e == 255) s = 127;
    up = __int_as_float(s << 23);
    down = __int_as_float((254 - s) << 23);
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Runs: few rows per sequence.  A unit is (sequence, kv head, row block of RB rows = tokens x heads of the group); its keys are cut into
// chunks of 64.  All chunks of all units stand in one line, which is cut into equal runs, one per block, so that
// contexts of any lengths keep all blocks equally long at work.  A unit that lies in several runs leaves partial results, which the next kernel
// joins.  A warp takes 16 keys of a chunk; keys and values come through a ring of its own in shared memory (cp.async, no block-wide waits).
// ------------------------------------------------------------------------------------------------------------------------------------

// The line: chunks before each sequence, its chunks per unit and first chunk follow from ctx and rows.
struct SeqWork {
    int first, n, ctx, blocks, chunk0, chunks;  // rows, context, row blocks, first chunk, chunks per unit
    bool inside;
};
template <int RB>
__device__ __forceinline__ SeqWork seq_work(const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, int i) {
    SeqWork w;
    w.inside = false;
    w.blocks = w.chunk0 = w.chunks = 0;
    w.ctx = s.ctx[i];
    if (!kv8_span(s, i, w.first, w.n) || w.n == 0) { w.n = 0; return w; }
    w.blocks = (w.n * a.group + RB - 1) / RB;
    w.inside = kv8_in_table(s, p, w.ctx, w.n);
    if (w.inside) {
        const int lo = a.window > 0 ? max(0, w.ctx - a.window + 1) : 0;
        w.chunk0 = lo / kChunk;
        w.chunks = (w.ctx + w.n + kChunk - 1) / kChunk - w.chunk0;
    } else {
        w.chunks = 1;  // one step that writes NaN
    }
    return w;
}
// cum[i] = chunks of the sequences before i, cum[n_seqs] = all; by one block, returns the total
template <int RB>
__device__ __forceinline__ uint32_t line_up(const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, uint32_t* cum, uint32_t* warp_sums) {
    const int per = (s.n_seqs + blockDim.x - 1) / blockDim.x, i0 = threadIdx.x * per, i1 = min(i0 + per, s.n_seqs);
    uint32_t sum = 0;
    for (int i = i0; i < i1; i++) {
        const SeqWork w = seq_work<RB>(s, p, a, i);
        cum[i] = sum;
        sum += (uint32_t)w.blocks * (uint32_t)p.n_kv * (uint32_t)w.chunks;
    }
    uint32_t incl = sum;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    uint32_t before = incl - sum, total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    for (int i = i0; i < i1; i++) cum[i] += before;
    if (threadIdx.x == 0) cum[s.n_seqs] = total;
    __syncthreads();
    return total;
}
__device__ __forceinline__ int seq_at(const uint32_t* cum, int n_seqs, uint32_t t) {  // the sequence whose chunks t is one of
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ uint32_t run_start(uint32_t total, int b, int blocks) { return (uint32_t)((unsigned long long)total * b / blocks); }

// floats of one partial result: maxima, sums and rows of HD
template <int HD, int RB> __host__ __device__ constexpr int part_floats() { return RB * (HD + 2); }

// Where a place of the line lies.
struct Place {
    int seq, kvh, rb, chunk;       // chunk: index within the unit
    SeqWork w;
    uint32_t unit_start;           // place of the unit's first chunk
};
template <int RB>
__device__ __forceinline__ void place_at(Place& at, const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, const uint32_t* cum, uint32_t t) {
    at.seq = seq_at(cum, s.n_seqs, t);
    at.w = seq_work<RB>(s, p, a, at.seq);
    const uint32_t in = t - cum[at.seq], unit = in / at.w.chunks;
    at.chunk = in - unit * at.w.chunks;
    at.unit_start = t - at.chunk;
    at.kvh = unit / at.w.blocks;
    at.rb = unit - at.kvh * at.w.blocks;
}

template <typename T, int HD, int RB> struct RunShape {
    static constexpr int kStageBytes = 2 * kStep * HD + 16;   // keys, values, their two scales
    static constexpr int kStages = HD == 64 ? 4 : 3;
    static constexpr int kRing = kRunWarps * kStages * kStageBytes;
    static constexpr int kJoin = kRunWarps * part_floats<HD, RB>() * 4;
};

template <typename T, int HD, int RB>
__global__ void __launch_bounds__(kRunWarps * 32, HD == 256 ? 2 : RB == 8 ? 4 : 3)
kv8_runs_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a) {
    constexpr bool SPLIT = RB == 8;
    constexpr int NT = HD / 8;              // tiles of 8 dims of the output; a thread's values of a key are NT in a row
    constexpr int KS = HD / 16;             // k steps of the scores
    constexpr int OC = SPLIT ? 2 : 4;
    using Shape = RunShape<T, HD, RB>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t warp_sums[kRunWarps];
    float* join = reinterpret_cast<float*>(smem);                 // shares its place with the ring between segments' ends
    uint32_t* cum = reinterpret_cast<uint32_t*>(smem + (Shape::kRing > Shape::kJoin ? Shape::kRing : Shape::kJoin));
    pdl_launch_dependents();
    if (blockIdx.x == 0) kv8_check_seqs(seqs, pool);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const uint32_t total = line_up<RB>(seqs, pool, a, cum, warp_sums);
    uint32_t t = run_start(total, blockIdx.x, gridDim.x);
    const uint32_t t_end = run_start(total, blockIdx.x + 1, gridDim.x);
    const uint32_t ring = smem_u32(smem) + warp * Shape::kStages * Shape::kStageBytes;
    const int hd = pool.hd, page_mask = (1 << pool.page_shift) - 1;

    while (t < t_end) {
        // a segment: this run's chunks of one unit
        Place at;
        place_at<RB>(at, seqs, pool, a, cum, t);
        const SeqWork& w = at.w;
        const int c0 = at.chunk, c1 = min(w.chunks, c0 + (int)(t_end - t));
        const int32_t* table = seqs.table + (size_t)at.seq * seqs.width;
        const int row_lo = at.rb * RB, row_n = min(RB, w.n * a.group - row_lo);
        const int key_end = w.ctx + w.n;    // exclusive

        auto page_of = [&](int chunk) -> int {  // the page of this warp's keys of a chunk
            const int key = (w.chunk0 + chunk) * kChunk + warp * kStep;
            if (!w.inside || chunk >= c1 || key >= key_end) return -1;
            return table[key >> pool.page_shift];
        };
        auto fetch = [&](int chunk, int number) {
            const int key = (w.chunk0 + chunk) * kChunk + warp * kStep;
            if (w.inside && chunk < c1 && key < key_end) {
                const uint32_t st = ring + (uint32_t)(chunk % Shape::kStages) * Shape::kStageBytes;
                const bool held = number >= 0 && number < pool.n_pages;
                if (!held) { if (lane == 0) kv8_raise(seqs, at.seq); }
                else {
                    const size_t ph = (size_t)number * pool.n_kv + at.kvh;
                    const size_t off = ((ph << pool.page_shift) + (key & page_mask)) * hd;
                    const int pieces = hd >> 4;
#pragma unroll
                    for (int e = lane; e < kStep * (HD / 16); e += 32) {
                        const int row = e / (HD / 16), ch = e % (HD / 16);
                        if (ch < pieces) {
                            cp_async16(st + row * HD + ((ch ^ ((row & 1) << 2)) & (HD / 16 - 1)) * 16, pool.k + off + (size_t)row * hd + ch * 16);
                            cp_async16(st + kStep * HD + row * HD + ((ch ^ (row & 6)) & (HD / 16 - 1)) * 16, pool.v + off + (size_t)row * hd + ch * 16);
                        }
                    }
                    if (lane < 2) cp_async4(st + 2 * kStep * HD + lane * 4, (lane ? pool.v_scale : pool.k_scale) + ph);
                }
            }
            cp_async_commit();
        };

        int next_page = page_of(c0);
#pragma unroll
        for (int k = 0; k < Shape::kStages - 1; k++) {
            const int now = next_page;
            next_page = page_of(c0 + k + 1);
            fetch(c0 + k, now);
        }

        // the queries as operand fragments: dims of step ks = 4 j + wd: chunk j of 64, 16 c .. in it, word wd
        uint32_t qf[KS][4];
        float rf[SPLIT ? 1 : 2];
        int limit[SPLIT ? 1 : 2];            // last position that the row sees (-1: no row)
#pragma unroll
        for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) {
            const int r = g + 8 * hf;
            const bool has = r < row_n;
            const int tok = has ? (row_lo + r) / a.group : 0, hq = has ? (row_lo + r) % a.group : 0;
            const T* src = (const T*)a.q + (int64_t)(w.first + tok) * a.q_stride + (int64_t)(at.kvh * a.group + hq) * hd;
            limit[hf] = has ? w.ctx + tok : -1;
            float top = 0.0f;
            if (has)
                for (int j = 0; j < HD / 64; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int d = 64 * j + 16 * c + e;
                        if (d < hd) top = fmaxf(top, fabsf(elem_f(src[d])));
                    }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float up, down;
            row_scale(top, up, down);
            rf[hf] = a.scale_log2 * down;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d = 64 * (ks >> 2) + 16 * c + 4 * (ks & 3);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = has && d + e < hd ? elem_f(src[d + e]) * up : 0.0f;
                if (SPLIT) {
                    h2_split(v[0], v[1], qf[ks][0], qf[ks][1]);
                    h2_split(v[2], v[3], qf[ks][2], qf[ks][3]);
                } else {
                    qf[ks][hf] = h2_pack(v[0], v[1]);
                    qf[ks][2 + hf] = h2_pack(v[2], v[3]);
                }
            }
        }

        float o[NT][OC];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < OC; e++) o[n][e] = 0.0f;
        float m[SPLIT ? 1 : 2], l[SPLIT ? 1 : 2];
#pragma unroll
        for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) { m[hf] = kNegInf; l[hf] = 0.0f; }
        bool poisoned = !w.inside;

        for (int chunk = c0; chunk < c1; chunk++) {
            const int now = next_page;
            next_page = page_of(chunk + Shape::kStages);
            cp_async_wait<Shape::kStages - 2>();
            __syncwarp();
            const int key0 = (w.chunk0 + chunk) * kChunk + warp * kStep;
            const unsigned char* st = smem + (warp * Shape::kStages + chunk % Shape::kStages) * Shape::kStageBytes;
            const bool any = w.inside && key0 < key_end;
            if (any) {
                const int number = table[key0 >> pool.page_shift];
                if (number < 0 || number >= pool.n_pages) poisoned = true;
                else {
                    const float ksc = *reinterpret_cast<const float*>(st + 2 * kStep * HD), vsc = *reinterpret_cast<const float*>(st + 2 * kStep * HD + 4);
                    float s[2][4];
#pragma unroll
                    for (int tl = 0; tl < 2; tl++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) s[tl][e] = 0.0f;
#pragma unroll
                        for (int j = 0; j < HD / 64; j++) {
                            const int row = 8 * tl + g, ch = 4 * j + c;
                            uint4 kw = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                            if (ch * 16 < hd) {
                                kw = *reinterpret_cast<const uint4*>(st + row * HD + ((ch ^ ((row & 1) << 2)) & (HD / 16 - 1)) * 16);
                                kw.x ^= 0x80808080u; kw.y ^= 0x80808080u; kw.z ^= 0x80808080u; kw.w ^= 0x80808080u;
                            }
                            mma_f16(s[tl], qf[4 * j + 0], ints01(kw.x), ints23(kw.x));
                            mma_f16(s[tl], qf[4 * j + 1], ints01(kw.y), ints23(kw.y));
                            mma_f16(s[tl], qf[4 * j + 2], ints01(kw.z), ints23(kw.z));
                            mma_f16(s[tl], qf[4 * j + 3], ints01(kw.w), ints23(kw.w));
                        }
                    }
                    uint32_t pf[4];
#pragma unroll
                    for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) {
                        float v[4];
                        const float f = rf[hf] * ksc;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int tl = e >> 1, k = e & 1, key = key0 + 8 * tl + 2 * c + k;
                            v[e] = (SPLIT ? s[tl][k] + s[tl][2 + k] : s[tl][2 * hf + k]) * f;
                            if (key > limit[hf] || (a.window > 0 && key <= limit[hf] - a.window)) v[e] = kNegInf;
                        }
                        float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        mx = fmaxf(mx, m[hf]);
                        const float ref = mx == kNegInf ? 0.0f : mx;
                        if (__any_sync(0xffffffffu, mx > m[hf])) {
                            const float corr = exp2_fast(m[hf] - ref);
                            l[hf] *= corr;
#pragma unroll
                            for (int n = 0; n < NT; n++) { o[n][2 * hf] *= corr; o[n][2 * hf + 1] *= corr; }
                            m[hf] = mx;
                        }
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) p[e] = exp2_fast(v[e] - ref + 8.0f);
                        l[hf] += (p[0] + p[1]) + (p[2] + p[3]);
                        if (SPLIT) {
                            h2_split(p[0], p[1], pf[0], pf[1]);
                            h2_split(p[2], p[3], pf[2], pf[3]);
                        } else {
                            pf[hf] = h2_pack(p[0], p[1]);
                            pf[2 + hf] = h2_pack(p[2], p[3]);
                        }
                    }
                    // values: a thread's keys are 2c, 2c + 1, 8 + 2c, 9 + 2c; its dims NT in a row (HD 256: 16 and 16 more 128 further)
                    const unsigned char* vs = st + kStep * HD;
                    constexpr int WORDS = HD == 64 ? 2 : 4;
#pragma unroll
                    for (int gr = 0; gr < (HD == 256 ? 2 : 1); gr++) {
                        const int ch = HD == 64 ? g >> 1 : 8 * gr + g;
                        uint32_t kv[4][WORDS];
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int row = (x >> 1) * 8 + 2 * c + (x & 1);
                            const unsigned char* at16 = vs + row * HD + ((ch ^ (row & 6)) & (HD / 16 - 1)) * 16;
                            if (HD == 64) {
                                uint2 u = make_uint2(0, 0);
                                if (ch * 16 < hd) u = *reinterpret_cast<const uint2*>(at16 + (g & 1) * 8);
                                kv[x][0] = u.x ^ 0x80808080u; kv[x][1] = u.y ^ 0x80808080u;
                            } else {
                                uint4 u = make_uint4(0, 0, 0, 0);
                                if (ch * 16 < hd) u = *reinterpret_cast<const uint4*>(at16);
                                kv[x][0] = u.x ^ 0x80808080u; kv[x][1] = u.y ^ 0x80808080u;
                                kv[x][WORDS - 2] = u.z ^ 0x80808080u; kv[x][WORDS - 1] = u.w ^ 0x80808080u;
                            }
                        }
#pragma unroll
                        for (int wd = 0; wd < WORDS; wd++) {
                            const uint32_t a01 = __byte_perm(kv[0][wd], kv[1][wd], 0x5140), a23 = __byte_perm(kv[0][wd], kv[1][wd], 0x7362);
                            const uint32_t b01 = __byte_perm(kv[2][wd], kv[3][wd], 0x5140), b23 = __byte_perm(kv[2][wd], kv[3][wd], 0x7362);
#pragma unroll
                            for (int b = 0; b < 4; b++) {
                                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                const uint32_t va = b < 2 ? a01 : a23, vb = b < 2 ? b01 : b23;
                                mma_f16(acc, pf, b & 1 ? ints23(va) : ints01(va), b & 1 ? ints23(vb) : ints01(vb));
                                float(&oo)[OC] = o[16 * gr + 4 * wd + b];
                                if (SPLIT) {
                                    oo[0] = fmaf(acc[0] + acc[2], vsc, oo[0]);
                                    oo[1] = fmaf(acc[1] + acc[3], vsc, oo[1]);
                                } else {
#pragma unroll
                                    for (int e = 0; e < OC; e++) oo[e] = fmaf(acc[e], vsc, oo[e]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            fetch(chunk + Shape::kStages - 1, now);
        }
        cp_async_wait<0>();

        // join the warps: maxima, sums, rows
        if (poisoned) {
#pragma unroll
            for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) l[hf] = __int_as_float(0x7fffffff);
        }
#pragma unroll
        for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
        }
        __syncthreads();  // all warps have done with the ring
        float* mine = join + warp * part_floats<HD, RB>();
#pragma unroll
        for (int hf = 0; hf < (SPLIT ? 1 : 2); hf++) {
            const int r = g + 8 * hf;
            if (c == 0) { mine[r] = m[hf]; mine[RB + r] = l[hf]; }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                // tile n = byte n of the dims that a thread's column owns
                const int gr = HD == 256 ? n >> 4 : 0, byte = HD == 256 ? n & 15 : n;
                const int width = HD == 64 ? 8 : 16;
                mine[2 * RB + r * HD + 128 * gr + (2 * c) * width + byte] = o[n][2 * hf];
                mine[2 * RB + r * HD + 128 * gr + (2 * c + 1) * width + byte] = o[n][2 * hf + 1];
            }
        }
        __syncthreads();
        const bool starts = c0 == 0, ends = c1 == w.chunks;
        float* part = a.part + (size_t)(2 * blockIdx.x + (starts ? 1 : 0)) * part_floats<HD, RB>();
        for (int e = tid; e < RB * HD; e += kRunWarps * 32) {
            const int r = e / HD, d = e % HD;
            if (r >= row_n) continue;
            float mx = kNegInf;
#pragma unroll
            for (int x = 0; x < kRunWarps; x++) mx = fmaxf(mx, join[x * part_floats<HD, RB>() + r]);
            const float ref = mx == kNegInf ? 0.0f : mx;
            float sum = 0.0f, val = 0.0f;
#pragma unroll
            for (int x = 0; x < kRunWarps; x++) {
                const float* px = join + x * part_floats<HD, RB>();
                const float f = exp2_fast(px[r] - ref);
                // a warp without a key has weight 0 and sum 0; a poisoned one has a NaN sum
                sum += px[RB + r] == 0.0f ? 0.0f : isnan(px[RB + r]) ? px[RB + r] : f * px[RB + r];
                val = fmaf(f, px[2 * RB + r * HD + d], val);
            }
            if (starts && ends) {
                if (d < hd) {
                    const int tok = (row_lo + r) / a.group, hq = (row_lo + r) % a.group;
                    const float y = sum == 0.0f ? 0.0f : val / sum;
                    ((T*)a.out)[(int64_t)(w.first + tok) * a.out_stride + (int64_t)(at.kvh * a.group + hq) * hd + d] = to_elem<T>(isnan(sum) ? sum : y);
                }
            } else {
                if (d == 0) { part[r] = mx; part[RB + r] = sum; }
                part[2 * RB + e] = val;
            }
        }
        __syncthreads();
        t += (uint32_t)(c1 - c0);
    }
}

// Joins the partial results of units that lie in several runs.  Block b looks at the border between runs b and b + 1 and serves the unit
// across it, if run b is where that unit begins.
template <typename T, int HD, int RB>
__global__ void __launch_bounds__(128) kv8_join_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a, int runs) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t warp_sums[4];
    uint32_t* cum = reinterpret_cast<uint32_t*>(smem);
    const uint32_t total = line_up<RB>(seqs, pool, a, cum, warp_sums);
    pdl_wait();  // every block: this kernel's end then means that of the one before
    const int b = blockIdx.x;
    const uint32_t border = run_start(total, b + 1, runs), start = run_start(total, b, runs);
    if (border >= total || border == start) return;  // no unit there, or the run is empty
    Place at;
    place_at<RB>(at, seqs, pool, a, cum, border - 1);
    const uint32_t u0 = at.unit_start, u1 = u0 + at.w.chunks;
    if (u1 <= border || u0 < start) return;          // ends with the run; or began in an earlier one
    int last = b + 1;                                // the run with the unit's last chunk
    while (run_start(total, last + 1, runs) < u1) last++;
    const int row_lo = at.rb * RB, row_n = min(RB, at.w.n * a.group - row_lo);
    constexpr int P = part_floats<HD, RB>();
    for (int e = threadIdx.x; e < row_n * HD; e += blockDim.x) {
        const int r = e / HD, d = e % HD;
        if (d >= pool.hd) continue;
        const float* p = a.part + (size_t)(2 * b + 1) * P;
        float mx = p[r], sum = p[RB + r], val = p[2 * RB + e];
        for (int x = b + 1; x <= last; x++) {
            if (run_start(total, x, runs) == run_start(total, x + 1, runs)) continue;  // an empty run leaves nothing
            p = a.part + (size_t)(2 * x) * P;
            const float m2 = fmaxf(mx, p[r]), ref = m2 == kNegInf ? 0.0f : m2;
            const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(p[r] - ref);
            sum = (isnan(sum) ? sum : f0 * sum) + (isnan(p[RB + r]) ? p[RB + r] : f1 * p[RB + r]);
            val = fmaf(f0, val, f1 * p[2 * RB + e]);
            mx = m2;
        }
        const int tok = (row_lo + r) / a.group, hq = (row_lo + r) % a.group;
        const float y = isnan(sum) ? sum : sum == 0.0f ? 0.0f : val / sum;
        ((T*)a.out)[(int64_t)(at.w.first + tok) * a.out_stride + (int64_t)(at.kvh * a.group + hq) * pool.hd + d] = to_elem<T>(y);
    }
}

struct RunPlan {
    int hd, rb, blocks;
    size_t bytes;
};
// Rows of at most 8 per unit, and everything in f32, in the split form: its 22 bits come at no more products.
RunPlan plan_runs(const Kv8Pool& pool, uint32_t typ, int group, int max_rows) {
    RunPlan p;
    p.hd = pool.hd <= 64 ? 64 : pool.hd <= 128 ? 128 : 256;
    p.rb = typ == LC_TYPE_F32 || group * (max_rows < 1 ? 1 : max_rows) <= 8 ? 8 : 16;
    p.blocks = sm_count() * (p.hd == 256 ? 2 : p.rb == 8 ? 4 : 3);
    p.bytes = (size_t)2 * p.blocks * p.rb * (p.hd + 2) * sizeof(float);
    return p;
}

template <typename T, int HD, int RB>
int32_t runs_as(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int blocks, cudaStream_t s) {
    using Shape = RunShape<T, HD, RB>;
    const size_t cum = (size_t)(seqs.n_seqs + 1) * 4;
    const size_t smem = (Shape::kRing > Shape::kJoin ? Shape::kRing : Shape::kJoin) + cum;
    LC_CUDA(ensure_smem_limit((const void*)kv8_runs_kernel<T, HD, RB>, smem));
    kv8_runs_kernel<T, HD, RB><<<blocks, kRunWarps * 32, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    LC_CUDA(launch_pdl(kv8_join_kernel<T, HD, RB>, dim3((unsigned)(blocks - 1)), dim3(128), cum, s, pool, seqs, a, blocks));
    return LC_OK;
}
template <typename T>
int32_t runs_of(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const RunPlan& p, cudaStream_t s) {
    if (p.rb == 8) {
        if (p.hd == 64) return runs_as<T, 64, 8>(pool, seqs, a, p.blocks, s);
        if (p.hd == 128) return runs_as<T, 128, 8>(pool, seqs, a, p.blocks, s);
        return runs_as<T, 256, 8>(pool, seqs, a, p.blocks, s);
    }
    if (p.hd == 64) return runs_as<T, 64, 16>(pool, seqs, a, p.blocks, s);
    if (p.hd == 128) return runs_as<T, 128, 16>(pool, seqs, a, p.blocks, s);
    return runs_as<T, 256, 16>(pool, seqs, a, p.blocks, s);
}

int32_t check_heads(const char* call, const Kv8Pool& pool, const Kv8Seqs& seqs, int32_t n_heads) {
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    // places of the line, row blocks of 8 at worst, in 31 bits
    const double chunks = (double)((int64_t)seqs.width << pool.page_shift) / kChunk + 2, blocks = (double)seqs.n_rows * (n_heads / pool.n_kv) / 8 + seqs.n_seqs;
    LC_CHECK(chunks * blocks * pool.n_kv < 2147483648.0, LC_ERR_INVALID, "%s: %d rows of %d heads over tables of %d pages are too many for one call", call, seqs.n_rows, n_heads, seqs.width);
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_attention_kv8_workspace(const lc_kv8_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, int32_t n_heads,
                                   size_t* out_bytes) {
    Kv8Pool pool;
    Kv8Seqs seqs;
    LC_CHECK(out_bytes, LC_ERR_INVALID, "lc_attention_kv8_workspace: null output");
    LC_TRY(kv8_check("lc_attention_kv8_workspace", cache, rows, typ, n_rows, &pool, &seqs));
    LC_TRY(check_heads("lc_attention_kv8_workspace", pool, seqs, n_heads));
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_attention_kv8_workspace: cache"));
    *out_bytes = plan_runs(pool, typ, n_heads / pool.n_kv, rows->max_rows).bytes;
    return LC_OK;
}

int32_t lc_attention_kv8_dev(const lc_kv8_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, const void* q_dev,
                             int64_t q_stride, int32_t n_heads, float scale, int32_t window, void* out_dev, int64_t out_stride,
                             void* workspace_dev, size_t workspace_bytes, void* stream_) {
    Kv8Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv8_check("lc_attention_kv8_dev", cache, rows, typ, n_rows, &pool, &seqs));
    LC_TRY(check_heads("lc_attention_kv8_dev", pool, seqs, n_heads));
    LC_CHECK(window >= 0, LC_ERR_INVALID, "lc_attention_kv8_dev: window=%d", window);
    LC_CHECK(scale >= 0.0f && scale <= 3.0e38f, LC_ERR_INVALID, "lc_attention_kv8_dev: scale=%g", scale);
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(q_dev && out_dev, LC_ERR_INVALID, "lc_attention_kv8_dev: null queries or output");
    LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && out_stride >= (int64_t)n_heads * pool.hd, LC_ERR_INVALID, "lc_attention_kv8_dev: rows overlap");
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_attention_kv8_dev: cache"));
    const int group = n_heads / pool.n_kv;
    const RunPlan plan = plan_runs(pool, typ, group, rows->max_rows);
    LC_CHECK(workspace_dev && workspace_bytes >= plan.bytes && (uintptr_t)workspace_dev % 16 == 0, LC_ERR_INVALID,
             "lc_attention_kv8_dev: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", plan.bytes, workspace_bytes);
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    AttnArgs a{q_dev, out_dev, q_stride, out_stride, n_heads, group, window, scale * 1.44269504088896f, (float*)workspace_dev};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return runs_of<float>(pool, seqs, a, plan, s);
    if (typ == LC_TYPE_F16) return runs_of<__half>(pool, seqs, a, plan, s);
    return runs_of<__nv_bfloat16>(pool, seqs, a, plan, s);
}

}  // extern "C"
