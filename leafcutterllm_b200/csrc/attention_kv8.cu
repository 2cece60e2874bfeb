// Attention over the key/value cache in 8 bits: out = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the positions j up to the row's own.
//
// A cached element is an integer times the scale of its page and head, so both products are taken of the integers as they are, and the scales are applied outside.
//   Scores  on the matrix unit's integers (mma.sync m16n8k32, exact): a row of queries is whole numbers in units of its largest / (127 x 256), f32: / (127 x 65,536), and
//           these are digits of 8 bits, in rows of their own of the operand, so that keys go in as they lie in the cache.  16 bits are as good as f16 or bf16
//           queries ask for: a score of size 1 is off by 3e-5; 24 bits for f32.  Rows whose largest element is above 32 times the mean get a digit more.
//   Values  an integer of 8 bits is exact in f16 (m16n8k16, f32 out): values are the operand of 16 rows (dims) and weights that of 8 columns (rows of queries), which the
//           scores' layout already is.  The weights are 2^(s - max + 6) in f16, 2^-11 of each off, times their page's scale over a reference that follows the scales, so that sums stay
//           in the matrix unit's accumulators.  For f32 they are the f16 value and what its rounding lost, 22 bits together, in two products; a step's sums are multiplied by the page's
//           scale and added in f32, so that what the matrix unit cuts off when it adds stays within 16 keys.
// What bounds it: single tokens, the instructions' waits for one another at 16 warps an SM (64 sequences of 128 - 4,096 tokens, 32 heads over 8, bf16: 43 us, 154 MB at 4.1 TB/s, half of the issue slots);
// more rows, the same with 8 warps of 255 registers (32 rows behind 60,000 - 131,000: 152 us, 392 MB at 2.7 TB/s, 39 % of the slots); one sequence, the two launches' beginnings and ends (700 tokens 10 us).
#include <algorithm>
#include <type_traits>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

// ------------------------------------------------------------------------------------------------------------------------------------
// Runs: few rows per sequence.  A unit is (sequence, kv head, row block of RB rows = tokens x heads of the group); its keys are cut into
// steps of 16.  All steps of all units, and some places for what a unit costs besides, stand in one line, which is cut into equal runs, one per WARP, so that
// contexts of any lengths keep all warps equally long at work and none waits for another.  A unit that lies in several runs leaves partial results, which the next kernel
// joins.  Keys and values come through a ring of the warp's own in shared memory (cp.async).
//
// Operand layouts, so that nothing is transposed: the dims of a score and the keys of a weighted sum are sums' indexes and may stand in any
// order, so a thread takes 16 neighbouring dims of its key (one 16-byte read) for four steps of the scores, and its columns of
// the weighted sum are 16 neighbouring dims of its four keys.  What it ends with is 32 neighbouring dims (HD 64: 16) of its row.
// ------------------------------------------------------------------------------------------------------------------------------------

// NG groups of 8 rows; F32: queries of 24 bits and weights of 22
template <int HD, int NG, bool F32> struct RunShape {
    static constexpr int kRows = 8 * NG;
    static constexpr int kStageBytes = 2 * kStep * HD + 16;   // keys, values, their two scales
    static constexpr int kStages = HD == 64 ? 4 : HD == 128 && !(F32 && NG == 4) ? 3 : 2;
    static constexpr bool kQueriesShared = HD == 256 || NG > 1;  // operand fragments of the queries in shared memory, not in registers
    static constexpr int kQueries = kQueriesShared ? NG * (F32 ? 2 : 1) * (HD / 32) * 512 : 0;
    static constexpr int kWarp = kStages * kStageBytes + kQueries;
    static constexpr int kByRegisters = HD == 256 ? (NG == 1 ? 3 : 2) : NG == 1 ? 4 : NG == 2 ? 3 : 2;
    static constexpr int kByMemory = (220 << 10) / (kRunWarps * kWarp + 2048);
    static constexpr int kBlocks = kByRegisters < kByMemory ? kByRegisters : kByMemory;
};

// The unit of a row's numbers, of its scaled largest element.
template <bool F32> __device__ __forceinline__ float query_unit(float top) { return top > 0.0f ? top * (F32 ? 1.0f / (127.0f * 65536.0f) : 1.0f / (127.0f * 256.0f)) : 1.0f; }

// What the scores of 16 keys gain by the digit behind the units, in units: keys 2c, 2c + 1 and 8 + 2c, 9 + 2c of row g.  hd: 0 for no row.  Few rows need it, so it is taken
// from the queries again.
template <int HD, bool F32>
__device__ __forceinline__ float4 next_digit(const void* q, int64_t src, int typ, bool vec, int hd, const unsigned char* kp) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float v[HD / 64][16], top = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 64; j++) {
        const int d = 64 * j + 16 * c;
        if (d < hd) load16(q, src + d, typ, vec, v[j]);
        else
#pragma unroll
            for (int e = 0; e < 16; e++) v[j][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) top = max_nan(top, fabsf(v[j][e]));
    }
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up, down;
    row_scale(top, up, down);
    const float per = 1.0f / query_unit<F32>(top * up);
    int dot[2][4] = {};
#pragma unroll
    for (int j = 0; j < HD / 64; j++) {
        uint32_t f[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            int n[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float u = v[j][4 * x + e] * up * per;  // as above
                n[e] = min(127, __float2int_rn((u - rintf(u)) * 256.0f));
            }
            f[x] = pack4(n[0], n[1], n[2], n[3]);
        }
#pragma unroll
        for (int tl = 0; tl < 2; tl++) {
            const int row = 8 * tl + g, ch = 4 * j + c;
            const uint4 kw = *reinterpret_cast<const uint4*>(kp + row * HD + ((ch ^ ((row & 1) << 2)) & (HD / 16 - 1)) * 16);
            mma_s8(dot[tl], f[0], 0u, f[1], 0u, kw.x, kw.y);
            mma_s8(dot[tl], f[2], 0u, f[3], 0u, kw.z, kw.w);
        }
    }
    return make_float4((float)dot[0][0] / 256.0f, (float)dot[0][1] / 256.0f, (float)dot[1][0] / 256.0f, (float)dot[1][1] / 256.0f);
}

template <int HD, int NG, bool F32, bool FULL>
__global__ void __launch_bounds__(kRunWarps * 32, RunShape<HD, NG, F32>::kBlocks)
kv8_runs_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a) {
    using Shape = RunShape<HD, NG, F32>;
    constexpr int ND = F32 ? 2 : 1;         // tiles of a group's digits
    constexpr int RB = Shape::kRows;
    constexpr int NT = HD / 16;             // tiles of 16 dims of the output: a thread has two neighbouring ones of each, NT pairs in a row
    constexpr int KS = HD / 32;             // k steps of the scores
    constexpr int S = Shape::kStages;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint2 warp_sums[kRunWarps];
    uint32_t* cum = reinterpret_cast<uint32_t*>(smem + kRunWarps * Shape::kWarp);
    pdl_launch_dependents();
    if (blockIdx.x == 0) kv8_check_seqs(seqs, pool);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t total = line_up<RB>(seqs, pool, a, cum, nullptr, warp_sums);
    const Runs runs(total, gridDim.x * kRunWarps);
    const uint32_t run = blockIdx.x * kRunWarps + warp;
    if (lane == 0) a.records[run].row_n = 0;
    if (run >= runs.n) return;
    uint32_t t = runs.start(run);
    const uint32_t t_end = runs.start(run + 1);
    unsigned char* const mine = smem + warp * Shape::kWarp;
    const uint32_t ring = smem_u32(mine);
    uint4* const qs = reinterpret_cast<uint4*>(mine + S * Shape::kStageBytes);
    const int hd = FULL ? HD : pool.hd, page_mask = (1 << pool.page_shift) - 1;
    // a lane's part of every copy: chunk lch of rows lrow, lrow + kRowsPer, ...; chunks behind hd repeat the last one (their queries are 0, their sums not stored)
    constexpr int kChunks = HD / 16, kRowsPer = 32 / kChunks;
    const int lrow = lane / kChunks, lch = lane % kChunks;
    const int lsrc = lrow * hd + (FULL ? lch : min(lch, (hd >> 4) - 1)) * 16;

    while (t < t_end) {
        // a segment: this run's steps of one unit
        Place at;
        place_at<RB>(at, seqs, pool, a, cum, t);
        const SeqWork& w = at.w;
        const int end = min(w.steps + kUnitCost, at.in + (int)(t_end - t)), s0 = max(0, at.in - kUnitCost), s1 = end - kUnitCost;
        t += (uint32_t)(end - at.in);
        if (s1 <= s0) continue;  // the unit's steps are the next run's
        if (s0 == 0 && s1 < w.steps && lane == 0) {
            a.records[run].last = (int)min(runs.run_of(t + (uint32_t)(w.steps - s1) - 1), runs.n - 1);
            *reinterpret_cast<int4*>(&a.records[run]) = make_int4(w.first, at.kvh, at.rb * RB, min(RB, w.n * a.group - at.rb * RB));
        }
        const int32_t* table = seqs.table + (size_t)at.seq * seqs.width;
        const int row_lo = at.rb * RB, row_n = min(RB, w.n * a.group - row_lo);

        // pages of 32 steps on, one per lane
        int pages_at = s0, pages = -1;
        auto look_up = [&]() {
            const int st = pages_at + lane;
            pages = w.inside && st < s1 ? table[((w.step0 + st) * kStep) >> pool.page_shift] : -1;
        };
        look_up();
        auto fetch = [&](int st) {
            if (st - pages_at == 32) { pages_at += 32; look_up(); }
            if (st < s1 && w.inside) {
                const int number = __shfl_sync(0xffffffffu, pages, st - pages_at);
                if (number < 0 || number >= pool.n_pages) {
                    // a page outside the pool: with a scale of NaN the scores of rows that see it are, those of others are masked; its values, whatever is in their place, count nothing
                    if (lane < 2) *reinterpret_cast<float*>(mine + (st % S) * Shape::kStageBytes + 2 * kStep * HD + lane * 4) = lane ? 0.0f : __int_as_float(0x7fffffff);
                    if (lane == 0) kv8_raise(seqs, at.seq);
                } else {
                    const uint32_t dst = ring + (uint32_t)(st % S) * Shape::kStageBytes;
                    const size_t ph = (size_t)number * pool.n_kv + at.kvh;
                    const size_t off = ((ph << pool.page_shift) + (((w.step0 + st) * kStep) & page_mask)) * hd + lsrc;
                    const int8_t* ks = pool.k + off;
                    const int8_t* vs = pool.v + off;
#pragma unroll
                    for (int i = 0; i < kStep / kRowsPer; i++) {
                        const int row = lrow + i * kRowsPer;
                        cp_async16(dst + row * HD + ((lch ^ ((row & 1) << 2)) & (kChunks - 1)) * 16, ks + i * kRowsPer * hd);
                        cp_async16(dst + (kStep + row) * HD + ((lch ^ (row & 6)) & (kChunks - 1)) * 16, vs + i * kRowsPer * hd);
                    }
                    if (lane < 2) cp_async4(dst + 2 * kStep * HD + lane * 4, (lane ? pool.v_scale : pool.k_scale) + ph);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int k = 0; k < S - 1; k++) fetch(s0 + k);

        // the queries as operand fragments: step ks = 2 j + x of the scores takes dims 64 j + 16 c + 8 x .. + 7.  A group's first tile has the highest digit in rows
        // 0 .. 7 and the next in rows 8 .. 15, its second tile the lowest in rows 0 .. 7.
        uint32_t qf[Shape::kQueriesShared ? 1 : NG * ND * KS][4];
        float rf[NG];                        // exponent of a unit of the queries' numbers
        int limit[NG];                       // last position that the row sees (-1: no row)
        bool fine = false;                   // some row's numbers get a digit more
#pragma unroll
        for (int group = 0; group < NG; group++) {
                const int r = 8 * group + g;
                const bool has = r < row_n;
                const int tok = has ? (row_lo + r) / a.group : 0, hq = has ? (row_lo + r) - tok * a.group : 0;
                const int64_t src = (int64_t)(w.first + tok) * a.q_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                limit[group] = has ? w.ctx + tok : -1;
                float v[HD / 64][16], top = 0.0f, all = 0.0f;
#pragma unroll
                for (int j = 0; j < HD / 64; j++) {
                    const int d = 64 * j + 16 * c;
                    if (has && (FULL || d < hd)) load16(a.q, src + d, a.typ, a.q_vec, v[j]);
                    else
#pragma unroll
                        for (int e = 0; e < 16; e++) v[j][e] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) { top = max_nan(top, fabsf(v[j][e])); all += fabsf(v[j][e]); }
                }
                all += __shfl_xor_sync(0xffffffffu, all, 1);
                all += __shfl_xor_sync(0xffffffffu, all, 2);
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float up, down;
                row_scale(top, up, down);
                const float unit = query_unit<F32>(top * up), per = 1.0f / unit;
                fine = fine || top * (float)hd > 32.0f * all;
                rf[group] = top < INFINITY ? a.scale_log2 * down * unit : __int_as_float(0x7fffffff);  // not finite: the row is NaN
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t digit[3][2];    // [highest first][four dims]
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        int n[4], lo[4], mid[4], hi[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            n[e] = __float2int_rn(v[ks >> 1][8 * (ks & 1) + 4 * x + e] * up * per);
                            lo[e] = (int)(int8_t)n[e];
                            mid[e] = (n[e] - lo[e]) >> 8;
                            hi[e] = (mid[e] - (int)(int8_t)mid[e]) >> 8;
                        }
                        digit[0][x] = F32 ? pack4(hi[0], hi[1], hi[2], hi[3]) : pack4(mid[0], mid[1], mid[2], mid[3]);
                        digit[1][x] = F32 ? pack4(mid[0], mid[1], mid[2], mid[3]) : pack4(lo[0], lo[1], lo[2], lo[3]);
                        digit[2][x] = pack4(lo[0], lo[1], lo[2], lo[3]);
                    }
#pragma unroll
                    for (int nd = 0; nd < ND; nd++) {
                        const uint32_t f0 = digit[2 * nd][0], f1 = nd ? 0u : digit[1][0], f2 = digit[2 * nd][1], f3 = nd ? 0u : digit[1][1];
                        const int at_f = (group * ND + nd) * KS + ks;
                        if (Shape::kQueriesShared) qs[at_f * 32 + lane] = make_uint4(f0, f1, f2, f3);
                        else {
                            uint32_t(&f)[4] = qf[Shape::kQueriesShared ? 0 : at_f];
                            f[0] = f0; f[1] = f1; f[2] = f2; f[3] = f3;
                        }
                    }
                }
            }

        // o: dims (a thread's 2 t, 2 t + 1 of tile t) x rows 2c, 2c + 1 of the group; m, l: of row g
        float o[NG][NT][4], m[NG], l[NG];
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[gr][t][e] = 0.0f;
            m[gr] = kNegInf;
            l[gr] = 0.0f;
        }
        auto is_far = [](float top) { return fabsf(top) > 65536.0f && top != kNegInf; };  // so far from 0 that a reference has no bits left for what is added to it
        bool far = false;                    // some row of the warp's has such a reference
        float vref = 0.0f, vtop = 0.0f;      // 16-bit types: what the sums' scales are relative to; the largest that was

        // rows see all keys up to the first row's position (with a window, from the last row's on)
        const int sees = w.ctx + row_lo / a.group, from = a.window > 0 ? w.ctx + (row_lo + row_n - 1) / a.group - a.window : -1;
        auto steps = [&](auto finer) {
        for (int st = s0; st < s1; st++) {
            cp_async_wait<S - 2>();
            __syncwarp();
            fetch(st + S - 1);  // into the place of the step before
            const int key0 = (w.step0 + st) * kStep;
            const bool plain = key0 + kStep - 1 <= sees && key0 > from;
            const unsigned char* kp = mine + (st % S) * Shape::kStageBytes;
            const float2 scales = *reinterpret_cast<const float2*>(kp + 2 * kStep * HD);
            const float ksc = scales.x, vsc = scales.y;
            constexpr int TL = kStep / 8;    // tiles of 8 keys
            float s[NG][TL][2];              // [group][tile][two keys]
            {
                int dot[NG * ND][TL][4];
#pragma unroll
                for (int j = 0; j < HD / 64; j++) {
                    uint4 kw[TL];
#pragma unroll
                    for (int tl = 0; tl < TL; tl++) {
                        const int row = 8 * tl + g, ch = 4 * j + c;
                        kw[tl] = *reinterpret_cast<const uint4*>(kp + row * HD + ((ch ^ ((row & 1) << 2)) & (kChunks - 1)) * 16);
                    }
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int ks = 2 * j + x;
#pragma unroll
                        for (int gd = 0; gd < NG * ND; gd++) {
                            uint4 f;
                            if (Shape::kQueriesShared) f = qs[(gd * KS + ks) * 32 + lane];
                            else {
                                const uint32_t(&q4)[4] = qf[Shape::kQueriesShared ? 0 : gd * KS + ks];
                                f = make_uint4(q4[0], q4[1], q4[2], q4[3]);
                            }
#pragma unroll
                            for (int tl = 0; tl < TL; tl++) {
                                const uint32_t b0 = x ? kw[tl].z : kw[tl].x, b1 = x ? kw[tl].w : kw[tl].y;
                                if (ks == 0) mma_s8_first(dot[gd][tl], f.x, f.y, f.z, f.w, b0, b1);
                                else mma_s8(dot[gd][tl], f.x, f.y, f.z, f.w, b0, b1);
                            }
                        }
                    }
                }
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
#pragma unroll
                    for (int tl = 0; tl < TL; tl++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const float high = (float)(256 * dot[gr * ND][tl][k] + dot[gr * ND][tl][2 + k]);
                            s[gr][tl][k] = F32 ? fmaf(high, 256.0f, (float)dot[gr * ND + ND - 1][tl][k]) : high;
                        }
            }
            if (decltype(finer)::value) {
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const int r = 8 * gr + g, rr = r < row_n ? r : 0, tok = (row_lo + rr) / a.group;
                    const int64_t src = (int64_t)(w.first + tok) * a.q_stride + (int64_t)(at.kvh * a.group + row_lo + rr - tok * a.group) * hd;
                    const float4 more = next_digit<HD, F32>(a.q, src, a.typ, a.q_vec, r < row_n ? hd : 0, kp);
                    s[gr][0][0] += more.x; s[gr][0][1] += more.y; s[gr][1][0] += more.z; s[gr][1][1] += more.w;
                }
            }
            float to_weight = 1.0f;
            if (!F32) {
                // within 2^-8 and 2^4 of the reference a scale goes to the weights; others make a reference of themselves (of 0 nothing is added), but none below 2^-64 of the
                // largest: the sums, 2^10 x 2^4 x 127 a key, would pass f32's range there
                const float ratio = fabsf(vsc) / vref;
                if (vsc != 0.0f && !(ratio >= 0x1p-8f && ratio <= 0x1p4f)) {
                    vtop = fmaxf(vtop, fabsf(vsc));
                    const float now = fmaxf(fabsf(vsc), vtop * 0x1p-64f), by = vref > 0.0f ? vref / now : 0.0f;
#pragma unroll
                    for (int gr = 0; gr < NG; gr++)
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[gr][t][e] *= by;
                    vref = now;
                }
                to_weight = vref > 0.0f ? vsc / vref : 0.0f;
                if (isnan(vsc)) to_weight = vsc;
            }
            float mx[NG];
            bool raise = false;
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                const float f = rf[gr] * ksc;
#pragma unroll
                for (int e = 0; e < 4; e++) s[gr][e >> 1][e & 1] *= f;
                if (!plain) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = key0 + 8 * (e >> 1) + 2 * c + (e & 1);
                        if (key > limit[gr] || (a.window > 0 && key <= limit[gr] - a.window)) s[gr][e >> 1][e & 1] = kNegInf;
                    }
                }
                mx[gr] = fmaxf(fmaxf(s[gr][0][0], s[gr][0][1]), fmaxf(s[gr][1][0], s[gr][1][1]));
            }
#pragma unroll
            for (int gr = 0; gr < NG; gr++) mx[gr] = fmaxf(mx[gr], __shfl_xor_sync(0xffffffffu, mx[gr], 1));
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                mx[gr] = fmaxf(mx[gr], __shfl_xor_sync(0xffffffffu, mx[gr], 2));
                raise = raise || mx[gr] - m[gr] > 4.0f;   // the difference: far from 0, m + 4 may be rounded up to the next number, which mx may be
            }
            // the references are raised when a row's maximum has grown by more than 2^4, so that a weight is 2^10 at most (with its scale 2^14); one vote for all
            // groups, whose chains of instructions then run side by side
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const float top = fmaxf(mx[gr], m[gr]), corr = top == kNegInf ? 1.0f : exp2_fast(m[gr] - top);
                    l[gr] *= corr;
                    m[gr] = top;
                    far = far || is_far(top);
                    const float c0 = __shfl_sync(0xffffffffu, corr, 8 * c), c1 = __shfl_sync(0xffffffffu, corr, 8 * c + 4);
#pragma unroll
                    for (int t = 0; t < NT; t++) { o[gr][t][0] *= c0; o[gr][t][1] *= c1; o[gr][t][2] *= c0; o[gr][t][3] *= c1; }
                }
                far = __any_sync(0xffffffffu, far);
            }
            uint32_t ph[NG][2], pl[NG][2];   // weights, and what their rounding lost: keys 2c, 2c + 1 and 8 + 2c, 9 + 2c of row g
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                const float less = m[gr] == kNegInf ? 6.0f : 6.0f - m[gr];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = s[gr][e >> 1][e & 1] + less;
                if (far && is_far(m[gr])) {  // 6 - m may be 4 off there, and as much the other way for another m: the difference first, of rounded scores, as m is; it is exact near m
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = __fadd_rn(__fsub_rn(s[gr][e >> 1][e & 1], m[gr]), 6.0f);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = exp2_fast(v[e]);
                l[gr] += (v[0] + v[1]) + (v[2] + v[3]);
                if (F32) {
                    h2_split(v[0], v[1], ph[gr][0], pl[gr][0]);
                    h2_split(v[2], v[3], ph[gr][1], pl[gr][1]);
                } else {
                    ph[gr][0] = h2_pack(v[0] * to_weight, v[1] * to_weight);
                    ph[gr][1] = h2_pack(v[2] * to_weight, v[3] * to_weight);
                }
            }
            // values: a thread's keys are 2c, 2c + 1, 8 + 2c, 9 + 2c; its dims 2 NT in a row (HD 256: 16 and 16 more 128 further)
            const unsigned char* vp = kp + kStep * HD;
            constexpr int WORDS = HD == 64 ? 2 : 4;
#pragma unroll
            for (int half = 0; half < (HD == 256 ? 2 : 1); half++) {
                const int ch = HD == 64 ? g >> 1 : 8 * half + g;
                uint32_t kv[4][WORDS];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int row = (x >> 1) * 8 + 2 * c + (x & 1);
                    const unsigned char* at16 = vp + row * HD + ((ch ^ (row & 6)) & (kChunks - 1)) * 16;
                    if (HD == 64) {
                        const uint2 u = *reinterpret_cast<const uint2*>(at16 + (g & 1) * 8);
                        kv[x][0] = u.x ^ 0x80808080u; kv[x][1] = u.y ^ 0x80808080u;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(at16);
                        kv[x][0] = u.x ^ 0x80808080u; kv[x][1] = u.y ^ 0x80808080u;
                        kv[x][WORDS - 2] = u.z ^ 0x80808080u; kv[x][WORDS - 1] = u.w ^ 0x80808080u;
                    }
                }
#pragma unroll
                for (int wd = 0; wd < WORDS; wd++)
#pragma unroll
                    for (int b = 0; b < 2; b++) {  // bytes 2b, 2b + 1: dims of a tile's rows g, g + 8
                        const uint32_t va = __byte_perm(kv[0][wd], kv[1][wd], b ? 0x7362 : 0x5140), vb = __byte_perm(kv[2][wd], kv[3][wd], b ? 0x7362 : 0x5140);
                        const uint32_t vf[4] = {ints01(va), ints23(va), ints01(vb), ints23(vb)};
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) {
                            float(&oo)[4] = o[gr][8 * half + 2 * wd + b];
                            if (F32) {
                                float acc[4];
                                mma_f16_first(acc, vf, pl[gr][0], pl[gr][1]);
                                mma_f16(acc, vf, ph[gr][0], ph[gr][1]);
#pragma unroll
                                for (int e = 0; e < 4; e++) oo[e] = fmaf(acc[e], vsc, oo[e]);
                            } else {
                                mma_f16(oo, vf, ph[gr][0], ph[gr][1]);
                            }
                        }
                    }
            }
        }
        };
        // the loop twice, as the digit's values took other calls' registers in one (4 tokens x 8 heads of a group, two sequences behind 60,000 and more: 161 us instead of 152)
        if (__any_sync(0xffffffffu, fine)) steps(std::true_type{});
        else steps(std::false_type{});
        cp_async_wait<0>();

        const bool starts = s0 == 0, ends = s1 == w.steps;
        float* part = a.part + (size_t)(2 * run + (starts ? 1 : 0)) * part_floats<HD, RB>();
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
            float sum = l[gr];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (!w.inside) sum = __int_as_float(0x7fffffff);
            const bool whole = starts && ends;
            if (!whole && c == 0 && 8 * gr + g < row_n) { part[8 * gr + g] = m[gr]; part[RB + 8 * gr + g] = sum; }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int r = 8 * gr + 2 * c + x;
                const float total = __shfl_sync(0xffffffffu, sum, 8 * c + 4 * x);
                if (r >= row_n) continue;
                // a NaN sum makes all of the row NaN
                const float inv = whole ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f, unit = F32 ? 1.0f : vref;  // their product may be below the smallest number
                const int tok = (row_lo + r) / a.group, hq = (row_lo + r) - tok * a.group;
                const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                constexpr int N = HD == 64 ? 8 : 16;  // dims in a row
#pragma unroll
                for (int half = 0; half < (HD == 256 ? 2 : 1); half++) {
                    float v[N];
#pragma unroll
                    for (int e = 0; e < N; e++) v[e] = o[gr][8 * half + (e >> 1)][2 * (e & 1) + x] * inv * unit;
                    const int d = HD == 64 ? 8 * g : 128 * half + 16 * g;
                    if (!whole) store_run<N>(part + 2 * RB + r * HD + d, true, v);
                    else if (FULL || d < hd) store_run<N>(a.out, dst + d, a.typ, a.out_vec, v);
                }
            }
        }
        __syncwarp();
    }
}

// Joins the partial results of units that lie in several runs.  grid: (runs, slices of kJoinRows rows); a run's record says which unit begins in it.  Threads
// take four dims of a row each, and what threads are left over shares of the partial results.
constexpr int kJoinThreads = 128, kJoinRows = 4;
template <int HD, int RB>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(AttnArgs a, int hd) {
    __shared__ float4 s_val[kJoinThreads];
    __shared__ float s_m[kJoinThreads], s_sum[kJoinThreads];
    constexpr int P = part_floats<HD, RB>(), Q = HD / 4;
    pdl_wait();  // every block: this kernel's end then means that of the one before
    const int b = blockIdx.x;
    const int4 at = *reinterpret_cast<const int4*>(&a.records[b]);
    const int last = a.records[b].last, row0 = blockIdx.y * kJoinRows, rows = min(kJoinRows, at.w - row0);
    if (rows <= 0) return;
    const int cells = rows * Q, per = min(cells, kJoinThreads), shares = kJoinThreads / per, share = threadIdx.x / per;
    for (int e0 = 0; e0 < cells; e0 += per) {
        const int e = e0 + threadIdx.x - share * per, r = row0 + e / Q, d = (e % Q) * 4;
        const bool here = share < shares && e < cells;
        float mx = kNegInf, sum = 0.0f;
        float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (here) {
            const float* p = a.part + (size_t)(2 * b + 1) * P;  // of the run itself the second place, of the later ones the first
#pragma unroll 8
            for (int x = b + share; x <= last; x += shares) {
                const float* q = x == b ? p : a.part + (size_t)(2 * x) * P;
                const float pm = q[r], ps = q[RB + r];
                const float4 v = *reinterpret_cast<const float4*>(q + 2 * RB + r * HD + d);
                const float m2 = fmaxf(mx, pm), ref = m2 == kNegInf ? 0.0f : m2;
                const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(pm - ref);
                sum = f0 * sum + (isnan(ps) ? ps : f1 * ps);
                val.x = fmaf(f0, val.x, f1 * v.x); val.y = fmaf(f0, val.y, f1 * v.y);
                val.z = fmaf(f0, val.z, f1 * v.z); val.w = fmaf(f0, val.w, f1 * v.w);
                mx = m2;
            }
        }
        if (shares > 1) {
            __syncthreads();
            s_val[threadIdx.x] = val; s_m[threadIdx.x] = mx; s_sum[threadIdx.x] = sum;
            __syncthreads();
            if (share == 0 && here) {
                for (int x = 1; x < shares; x++) {
                    const int k = x * per + threadIdx.x;
                    const float m2 = fmaxf(mx, s_m[k]), ref = m2 == kNegInf ? 0.0f : m2;
                    const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(s_m[k] - ref);
                    const float4 v = s_val[k];
                    sum = f0 * sum + f1 * s_sum[k];
                    val.x = fmaf(f0, val.x, f1 * v.x); val.y = fmaf(f0, val.y, f1 * v.y);
                    val.z = fmaf(f0, val.z, f1 * v.z); val.w = fmaf(f0, val.w, f1 * v.w);
                    mx = m2;
                }
            }
        }
        if (share == 0 && here && d < hd) {
            const int tok = (at.z + r) / a.group, hq = (at.z + r) - tok * a.group;
            const int64_t dst = (int64_t)(at.x + tok) * a.out_stride + (int64_t)(at.y * a.group + hq) * hd + d;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            store1(a.out, dst, a.typ, val.x * inv);
            store1(a.out, dst + 1, a.typ, val.y * inv);
            store1(a.out, dst + 2, a.typ, val.z * inv);
            store1(a.out, dst + 3, a.typ, val.w * inv);
        }
    }
}

struct RunPlan {
    int hd, groups, blocks;
    size_t bytes;
};
template <int HD, bool F32> int run_blocks(int groups) {
    if (HD < 256 && groups == 4) return RunShape<HD, HD < 256 ? 4 : 1, F32>::kBlocks;
    return groups == 2 ? RunShape<HD, 2, F32>::kBlocks : RunShape<HD, 1, F32>::kBlocks;
}
// As many groups of 8 rows share a step's keys and values as a unit has rows for: four at most, whose sums are 128 registers (two for heads of 256).
int run_groups(const Kv8Pool& pool, int group, int max_rows) {
    const int64_t rows = (int64_t)group * (max_rows < 1 ? 1 : max_rows);
    return rows <= 8 ? 1 : rows <= 16 || pool.hd > 128 ? 2 : 4;
}
RunPlan plan_runs(const Kv8Pool& pool, uint32_t typ, int groups) {
    RunPlan p;
    p.hd = pool.hd <= 64 ? 64 : pool.hd <= 128 ? 128 : 256;
    p.groups = groups;
    const bool f32 = typ == LC_TYPE_F32;
    p.blocks = sm_count() * (p.hd == 64    ? (f32 ? run_blocks<64, true>(p.groups) : run_blocks<64, false>(p.groups))
                             : p.hd == 128 ? (f32 ? run_blocks<128, true>(p.groups) : run_blocks<128, false>(p.groups))
                                           : (f32 ? run_blocks<256, true>(p.groups) : run_blocks<256, false>(p.groups)));
    p.bytes = (size_t)p.blocks * kRunWarps * (sizeof(UnitRecord) + (size_t)2 * 8 * p.groups * (p.hd + 2) * sizeof(float));
    return p;
}
int most_groups(const Kv8Pool& pool) { return pool.hd > 128 ? 2 : 4; }
bool tiles_fit(const Kv8Pool& pool, const Kv8Seqs& seqs, int group) {
    TilePlan tiles;
    return line_fits(pool, seqs, group, kTileRows2) && kv8_tiles_plan(pool, seqs, group, &tiles);
}
struct Plan {
    bool by_tiles;
    TilePlan tiles;
    RunPlan runs;
    size_t bytes() const { return by_tiles ? tiles.bytes : runs.bytes; }
};
// The faster kernel, unless its line does not fit: a call with many more rows than its max_rows says goes by tiles then, or by as many groups as it takes.
Plan plan_call(const Kv8Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows) {
    Plan p;
    int groups = run_groups(pool, group, max_rows);
    p.by_tiles = kv8_tiles_plan(pool, seqs, group, &p.tiles) && line_fits(pool, seqs, group, kTileRows2) &&
                 (kv8_tiles_pay(pool, seqs, typ, group, max_rows, p.tiles) || !line_fits(pool, seqs, group, 8 * groups));
    while (!p.by_tiles && groups < most_groups(pool) && !line_fits(pool, seqs, group, 8 * groups)) groups *= 2;
    p.runs = plan_runs(pool, typ, groups);
    return p;
}
// The most that a call with at most these arguments needs: fewer rows, sequences or pages may go by runs instead of tiles, take fewer groups (whose
// runs are more), or have their keys cut where larger ones are not, so the answer goes by none of them.
size_t most_bytes(const Kv8Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows) {
    const bool any = !line_fits(pool, seqs, group, 8);  // then a smaller max_rows may lead to every kernel
    size_t most = kv8_tiles_most_bytes(pool, any ? 1 << 30 : (int64_t)group * max_rows);
    for (int groups = any ? most_groups(pool) : run_groups(pool, group, max_rows); groups >= 1; groups /= 2) most = std::max(most, plan_runs(pool, typ, groups).bytes);
    return most;
}

template <int HD, int NG, bool F32, bool FULL>
int32_t runs_as(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int blocks, cudaStream_t s) {
    using Shape = RunShape<HD, NG, F32>;
    const size_t cum = (size_t)(seqs.n_seqs + 1) * 4, smem = kRunWarps * Shape::kWarp + cum;
    LC_CUDA(ensure_smem_limit((const void*)kv8_runs_kernel<HD, NG, F32, FULL>, smem));
    kv8_runs_kernel<HD, NG, F32, FULL><<<blocks, kRunWarps * 32, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    LC_CUDA(launch_pdl(kv8_join_kernel<HD, Shape::kRows>, dim3((unsigned)blocks * kRunWarps, (Shape::kRows + kJoinRows - 1) / kJoinRows), dim3(kJoinThreads), 0, s, a, pool.hd));
    return LC_OK;
}
template <int HD, int NG>
int32_t runs_full(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (a.typ == LC_TYPE_F32) return pool.hd == HD ? runs_as<HD, NG, true, true>(pool, seqs, a, blocks, s) : runs_as<HD, NG, true, false>(pool, seqs, a, blocks, s);
    return pool.hd == HD ? runs_as<HD, NG, false, true>(pool, seqs, a, blocks, s) : runs_as<HD, NG, false, false>(pool, seqs, a, blocks, s);
}
template <int HD>
int32_t runs_of(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const RunPlan& p, cudaStream_t s) {
    if constexpr (HD < 256)
        if (p.groups == 4) return runs_full<HD, 4>(pool, seqs, a, p.blocks, s);
    return p.groups == 2 ? runs_full<HD, 2>(pool, seqs, a, p.blocks, s) : runs_full<HD, 1>(pool, seqs, a, p.blocks, s);
}

int32_t check_heads(const char* call, const Kv8Pool& pool, const Kv8Seqs& seqs, int32_t n_heads) {
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    const int group = n_heads / pool.n_kv;
    // a sequence outside its table may have all rows: what a call's rows are in the kernels' 32 bits
    LC_CHECK((int64_t)seqs.n_rows * group < (int64_t)0x7fffffff - kTileRows2, LC_ERR_INVALID, "%s: %d rows of %d heads are too many for one call", call, seqs.n_rows, n_heads);
    LC_CHECK(line_fits(pool, seqs, group, 8 * most_groups(pool)) || tiles_fit(pool, seqs, group), LC_ERR_INVALID, "%s: %d rows of %d heads over tables of %d pages are too many for one call",
             call, seqs.n_rows, n_heads, seqs.width);
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
    if (n_rows == 0 || seqs.n_seqs == 0) {  // nothing to do, as for the call itself
        *out_bytes = 16;
        return LC_OK;
    }
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_attention_kv8_workspace: cache"));
    *out_bytes = most_bytes(pool, seqs, typ, n_heads / pool.n_kv, rows->max_rows);
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
    LC_CHECK(scale >= 0.0f && scale <= 2.0e38f, LC_ERR_INVALID, "lc_attention_kv8_dev: scale=%g", scale);
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(q_dev && out_dev, LC_ERR_INVALID, "lc_attention_kv8_dev: null queries or output");
    LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && out_stride >= (int64_t)n_heads * pool.hd, LC_ERR_INVALID, "lc_attention_kv8_dev: rows overlap");
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_attention_kv8_dev: cache"));
    const int group = n_heads / pool.n_kv;
    const Plan plan = plan_call(pool, seqs, typ, group, rows->max_rows);
    const size_t need = plan.bytes();
    LC_CHECK(workspace_dev && workspace_bytes >= need && (uintptr_t)workspace_dev % 16 == 0, LC_ERR_INVALID,
             "lc_attention_kv8_dev: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", need, workspace_bytes);
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    window = std::min(window, 1 << 30);  // the kernels' differences of positions stay in 32 bits
    const size_t elem = typ == LC_TYPE_F32 ? 4 : 2;
    AttnArgs a{q_dev, out_dev, q_stride, out_stride, (int)typ, group, window, rows_aligned(q_dev, q_stride, elem, 16), rows_aligned(out_dev, out_stride, elem, 16),
               scale * 1.44269504088896f, nullptr, (UnitRecord*)workspace_dev};
    a.part = plan.by_tiles ? (float*)workspace_dev : (float*)((char*)workspace_dev + (size_t)plan.runs.blocks * kRunWarps * sizeof(UnitRecord));
    cudaStream_t s = stream_or_own(stream_);
    if (plan.by_tiles) return launch_kv8_tiles(pool, seqs, a, plan.tiles, s);
    if (plan.runs.hd == 64) return runs_of<64>(pool, seqs, a, plan.runs, s);
    if (plan.runs.hd == 128) return runs_of<128>(pool, seqs, a, plan.runs, s);
    return runs_of<256>(pool, seqs, a, plan.runs, s);
}

}  // extern "C"
