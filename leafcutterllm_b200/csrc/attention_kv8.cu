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
#include <algorithm>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

constexpr int kRunWarps = 4;

// ------------------------------------------------------------------------------------------------------------------------------------
// Runs: few rows per sequence.  A unit is (sequence, kv head, row block of RB rows = tokens x heads of the group); its keys are cut into
// steps of 16.  All steps of all units stand in one line, which is cut into equal runs, one per WARP, so that contexts of any lengths
// keep all warps equally long at work and none waits for another.  A unit that lies in several runs leaves partial results, which the next kernel
// joins.  Keys and values come through a ring of the warp's own in shared memory (cp.async).
//
// Operand layouts, so that nothing is transposed: the dims of a score and the keys of a weighted sum are sums' indexes and may stand in any
// order, so a thread takes 16 neighbouring dims of its key (one 16-byte read) for four steps of the scores, and its columns of
// the weighted sum are 16 neighbouring dims of its four keys.  What it ends with is 32 neighbouring dims (HD 64: 16) of its row.
// ------------------------------------------------------------------------------------------------------------------------------------

// The line of `total` steps in equal runs, none of them empty, and none shorter than kLeast where that leaves warps without one.
constexpr uint32_t kLeast = 2;
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

// Where a place of the line lies.
struct Place {
    int seq, kvh, rb, step;        // step: index within the unit
    SeqWork w;
    uint32_t unit_start;           // place of the unit's first step
};
template <int RB>
__device__ __forceinline__ void place_at(Place& at, const Kv8Seqs& s, const Kv8Pool& p, const AttnArgs& a, const uint32_t* cum, uint32_t t) {
    at.seq = seq_at(cum, s.n_seqs, t);
    at.w = seq_work<RB>(s, p, a, at.seq);
    const uint32_t in = t - cum[at.seq], unit = in / at.w.steps;
    at.step = in - unit * at.w.steps;
    at.unit_start = t - at.step;
    at.kvh = unit / at.w.blocks;
    at.rb = unit - at.kvh * at.w.blocks;
}

// MT tiles of 16 rows: 8 MT rows in the split form, 16 MT in the plain one
template <int HD, int MT, bool SPLIT> struct RunShape {
    static constexpr int kRows = MT * (SPLIT ? 8 : 16);
    static constexpr int kStageBytes = 2 * kStep * HD + 16;   // keys, values; scales of the first 16 keys, of the others, of the values likewise
    static constexpr int kStages = HD == 64 ? 3 : 2;
    static constexpr bool kQueriesShared = HD == 256 || MT > 1;  // operand fragments of the queries in shared memory, not in registers
    static constexpr int kQueries = kQueriesShared ? MT * (HD / 16) * 512 : 0;
    static constexpr int kWarp = kStages * kStageBytes + kQueries;
    static constexpr int kBlocks = HD == 256 ? 1 : MT > 1 ? 2 : 3;
};

template <int HD, int MT, bool SPLIT, bool FULL>
__global__ void __launch_bounds__(kRunWarps * 32, RunShape<HD, MT, SPLIT>::kBlocks)
kv8_runs_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a) {
    using Shape = RunShape<HD, MT, SPLIT>;
    constexpr int RB = Shape::kRows;
    constexpr int NT = HD / 8;              // tiles of 8 dims of the output; a thread's values of a key are NT in a row
    constexpr int KS = HD / 16;             // k steps of the scores
    constexpr int HF = SPLIT ? 1 : 2;       // rows of a tile that a thread has a part in
    constexpr int OC = 2 * HF;
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
        const int s0 = at.step, s1 = min(w.steps, s0 + (int)(t_end - t));
        const int32_t* table = seqs.table + (size_t)at.seq * seqs.width;
        const int row_lo = at.rb * RB, row_n = min(RB, w.n * a.group - row_lo), key_end = w.ctx + w.n;

        // pages of 16 steps on, one per lane and 16 keys
        int pages_at = s0, pages = -1;
        auto look_up = [&]() {
            const int st = pages_at + (lane >> 1), key = (w.step0 + st) * kStep + (lane & 1) * 16;
            pages = w.inside && st < s1 && key < key_end ? table[key >> pool.page_shift] : -1;
        };
        look_up();
        bool poisoned = !w.inside;
        auto fetch = [&](int st) {
            if (st - pages_at == 16) { pages_at += 16; look_up(); }
            if (st < s1 && w.inside) {
                const uint32_t dst = ring + (uint32_t)(st % S) * Shape::kStageBytes;
                float* const scales = reinterpret_cast<float*>(mine + (st % S) * Shape::kStageBytes + 2 * kStep * HD);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int number = __shfl_sync(0xffffffffu, pages, 2 * (st - pages_at) + x), key = (w.step0 + st) * kStep + 16 * x;
                    if (key >= key_end || number < 0 || number >= pool.n_pages) {
                        if (key < key_end) {
                            poisoned = true;
                            if (lane == 0) kv8_raise(seqs, at.seq);
                        }
                        if (lane < 2) scales[2 * lane + x] = 0.0f;  // nothing of what lies there has a weight
                        continue;
                    }
                    const size_t ph = (size_t)number * pool.n_kv + at.kvh;
                    const size_t off = ((ph << pool.page_shift) + (key & page_mask)) * hd + lsrc;
                    const int8_t* ks = pool.k + off;
                    const int8_t* vs = pool.v + off;
#pragma unroll
                    for (int i = 0; i < 16 / kRowsPer; i++) {
                        const int row = lrow + i * kRowsPer;
                        cp_async16(dst + (16 * x + row) * HD + ((lch ^ ((row & 1) << 2)) & (kChunks - 1)) * 16, ks + i * kRowsPer * hd);
                        cp_async16(dst + (kStep + 16 * x + row) * HD + ((lch ^ (row & 6)) & (kChunks - 1)) * 16, vs + i * kRowsPer * hd);
                    }
                    if (lane < 2) cp_async4(dst + 2 * kStep * HD + (2 * lane + x) * 4, (lane ? pool.v_scale : pool.k_scale) + ph);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int k = 0; k < S - 1; k++) fetch(s0 + k);

        // the queries as operand fragments: step ks = 4 j + wd of the scores takes dims 64 j + 16 c + 4 wd .. + 3
        uint32_t qf[Shape::kQueriesShared ? 1 : KS][4];
        float rf[MT][HF];
        int limit[MT][HF];                   // last position that the row sees (-1: no row)
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            uint32_t f[KS][4];
#pragma unroll
            for (int hf = 0; hf < HF; hf++) {
                const int r = (SPLIT ? 8 : 16) * mt + g + 8 * hf;
                const bool has = r < row_n;
                const int tok = has ? (row_lo + r) / a.group : 0, hq = has ? (row_lo + r) - tok * a.group : 0;
                const int64_t src = (int64_t)(w.first + tok) * a.q_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                limit[mt][hf] = has ? w.ctx + tok : -1;
                float v[KS][4], top = 0.0f;
#pragma unroll
                for (int j = 0; j < KS / 4; j++) {
                    const int d = 64 * j + 16 * c;
                    if (has && (FULL || d < hd)) load16(a.q, src + d, a.typ, a.q_vec, &v[4 * j][0]);
                    else
#pragma unroll
                        for (int e = 0; e < 16; e++) v[4 * j + (e >> 2)][e & 3] = 0.0f;
                }
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(v[ks][e]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float up, down;
                row_scale(top, up, down);
                rf[mt][hf] = a.scale_log2 * down;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    if (SPLIT) {
                        h2_split(v[ks][0] * up, v[ks][1] * up, f[ks][0], f[ks][1]);
                        h2_split(v[ks][2] * up, v[ks][3] * up, f[ks][2], f[ks][3]);
                    } else {
                        f[ks][hf] = h2_pack(v[ks][0] * up, v[ks][1] * up);
                        f[ks][2 + hf] = h2_pack(v[ks][2] * up, v[ks][3] * up);
                    }
                }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (Shape::kQueriesShared) qs[(mt * KS + ks) * 32 + lane] = make_uint4(f[ks][0], f[ks][1], f[ks][2], f[ks][3]);
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) qf[Shape::kQueriesShared ? 0 : ks][e] = f[ks][e];
            }
        }

        float o[MT][NT][OC], m[MT][HF], l[MT][HF];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < OC; e++) o[mt][n][e] = 0.0f;
#pragma unroll
            for (int hf = 0; hf < HF; hf++) { m[mt][hf] = kNegInf; l[mt][hf] = 0.0f; }
        }

        // rows see all keys up to the first row's position (with a window, from the last row's on)
        const int sees = w.ctx + row_lo / a.group, from = a.window > 0 ? w.ctx + (row_lo + row_n - 1) / a.group - a.window : -1;
        for (int st = s0; st < s1; st++) {
            cp_async_wait<S - 2>();
            __syncwarp();
            fetch(st + S - 1);  // into the place of the step before
            const int key0 = (w.step0 + st) * kStep;
            const bool plain = key0 + kStep - 1 <= sees && key0 > from;
            const unsigned char* kp = mine + (st % S) * Shape::kStageBytes;
            const float4 scales = *reinterpret_cast<const float4*>(kp + 2 * kStep * HD);
            const float ksc[2] = {scales.x, scales.y};
            // the values' scales over the larger of them go to the weights, that one to their sums
            const float vmax = fmaxf(fabsf(scales.z), fabsf(scales.w)), vinv = vmax > 0.0f ? 1.0f / vmax : 0.0f;
            const float vr[2] = {scales.z * vinv, scales.w * vinv};
            float s[MT][4][4];
#pragma unroll
            for (int j = 0; j < HD / 64; j++) {
                uint32_t kw[4][4];
#pragma unroll
                for (int tl = 0; tl < 4; tl++) {
                    const int row = 8 * tl + g, ch = 4 * j + c;
                    const uint4 u = *reinterpret_cast<const uint4*>(kp + row * HD + ((ch ^ ((row & 1) << 2)) & (kChunks - 1)) * 16);
                    kw[tl][0] = u.x ^ 0x80808080u; kw[tl][1] = u.y ^ 0x80808080u; kw[tl][2] = u.z ^ 0x80808080u; kw[tl][3] = u.w ^ 0x80808080u;
                }
#pragma unroll
                for (int wd = 0; wd < 4; wd++) {
                    const int ks = 4 * j + wd;
                    uint32_t f[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (Shape::kQueriesShared) {
                            const uint4 u = qs[(mt * KS + ks) * 32 + lane];
                            f[mt][0] = u.x; f[mt][1] = u.y; f[mt][2] = u.z; f[mt][3] = u.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++) f[mt][e] = qf[Shape::kQueriesShared ? 0 : ks][e];
                        }
                    }
#pragma unroll
                    for (int tl = 0; tl < 4; tl++) {
                        const uint32_t b0 = ints01(kw[tl][wd]), b1 = ints23(kw[tl][wd]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            if (ks == 0) mma_f16_first(s[mt][tl], f[mt], b0, b1);
                            else mma_f16(s[mt][tl], f[mt], b0, b1);
                        }
                    }
                }
            }
            uint32_t pf[MT][2][4];           // weights of the first 16 keys, of the others
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < HF; hf++) {
                    float v[8];
                    const float f[2] = {rf[mt][hf] * ksc[0], rf[mt][hf] * ksc[1]};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int tl = e >> 1, k = e & 1;
                        v[e] = (SPLIT ? s[mt][tl][k] + s[mt][tl][2 + k] : s[mt][tl][2 * hf + k]) * f[tl >> 1];
                    }
                    if (!plain) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int key = key0 + 8 * (e >> 1) + 2 * c + (e & 1);
                            if (key > limit[mt][hf] || (a.window > 0 && key <= limit[mt][hf] - a.window)) v[e] = kNegInf;
                        }
                    }
                    float mx = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    mx = fmaxf(mx, m[mt][hf]);
                    const float ref = mx == kNegInf ? 0.0f : mx;
                    if (__any_sync(0xffffffffu, mx > m[mt][hf])) {
                        const float corr = exp2_fast(m[mt][hf] - ref);
                        l[mt][hf] *= corr;
#pragma unroll
                        for (int n = 0; n < NT; n++) { o[mt][n][2 * hf] *= corr; o[mt][n][2 * hf + 1] *= corr; }
                        m[mt][hf] = mx;
                    }
                    const float less = 8.0f - ref;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = exp2_fast(v[e] + less);
                    l[mt][hf] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float p0 = v[4 * x] * vr[x], p1 = v[4 * x + 1] * vr[x], p2 = v[4 * x + 2] * vr[x], p3 = v[4 * x + 3] * vr[x];
                        if (SPLIT) {
                            h2_split(p0, p1, pf[mt][x][0], pf[mt][x][1]);
                            h2_split(p2, p3, pf[mt][x][2], pf[mt][x][3]);
                        } else {
                            pf[mt][x][hf] = h2_pack(p0, p1);
                            pf[mt][x][2 + hf] = h2_pack(p2, p3);
                        }
                    }
                }
            // values: of each 16 keys a thread's are 2c, 2c + 1, 8 + 2c, 9 + 2c; its dims NT in a row (HD 256: 16 and 16 more 128 further)
            const unsigned char* vp = kp + kStep * HD;
            constexpr int WORDS = HD == 64 ? 2 : 4;
#pragma unroll
            for (int gr = 0; gr < (HD == 256 ? 2 : 1); gr++) {
                const int ch = HD == 64 ? g >> 1 : 8 * gr + g;
                uint32_t kv[2][4][WORDS];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int row = (x >> 2) * 16 + ((x >> 1) & 1) * 8 + 2 * c + (x & 1);
                    const unsigned char* at16 = vp + row * HD + ((ch ^ (row & 6)) & (kChunks - 1)) * 16;
                    uint32_t(&k4)[WORDS] = kv[x >> 2][x & 3];
                    if (HD == 64) {
                        const uint2 u = *reinterpret_cast<const uint2*>(at16 + (g & 1) * 8);
                        k4[0] = u.x ^ 0x80808080u; k4[1] = u.y ^ 0x80808080u;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(at16);
                        k4[0] = u.x ^ 0x80808080u; k4[1] = u.y ^ 0x80808080u;
                        k4[WORDS - 2] = u.z ^ 0x80808080u; k4[WORDS - 1] = u.w ^ 0x80808080u;
                    }
                }
#pragma unroll
                for (int wd = 0; wd < WORDS; wd++) {
                    uint32_t a01[2], a23[2], b01[2], b23[2];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        a01[x] = __byte_perm(kv[x][0][wd], kv[x][1][wd], 0x5140);
                        a23[x] = __byte_perm(kv[x][0][wd], kv[x][1][wd], 0x7362);
                        b01[x] = __byte_perm(kv[x][2][wd], kv[x][3][wd], 0x5140);
                        b23[x] = __byte_perm(kv[x][2][wd], kv[x][3][wd], 0x7362);
                    }
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        uint32_t v0[2], v1[2];
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t va = b < 2 ? a01[x] : a23[x], vb = b < 2 ? b01[x] : b23[x];
                            v0[x] = b & 1 ? ints23(va) : ints01(va);
                            v1[x] = b & 1 ? ints23(vb) : ints01(vb);
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            float acc[4];
                            mma_f16_first(acc, pf[mt][0], v0[0], v1[0]);
                            mma_f16(acc, pf[mt][1], v0[1], v1[1]);
                            float(&oo)[OC] = o[mt][16 * gr + 4 * wd + b];
                            if (SPLIT) {
                                oo[0] = fmaf(acc[0] + acc[2], vmax, oo[0]);
                                oo[1] = fmaf(acc[1] + acc[3], vmax, oo[1]);
                            } else {
#pragma unroll
                                for (int e = 0; e < OC; e++) oo[e] = fmaf(acc[e], vmax, oo[e]);
                            }
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();

        const bool starts = s0 == 0, ends = s1 == w.steps;
        float* part = a.part + (size_t)(2 * run + (starts ? 1 : 0)) * part_floats<HD, RB>();
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < HF; hf++) {
                float sum = l[mt][hf];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (poisoned) sum = __int_as_float(0x7fffffff);
                const int r = (SPLIT ? 8 : 16) * mt + g + 8 * hf;
                if (r >= row_n) continue;
                const bool whole = starts && ends;
                // a NaN sum makes all of the row NaN
                const float inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
                const int tok = (row_lo + r) / a.group, hq = (row_lo + r) - tok * a.group;
                const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                if (!whole && c == 0) { part[r] = m[mt][hf]; part[RB + r] = sum; }
                constexpr int GR = HD == 256 ? 2 : 1, W = HD == 64 ? 1 : 2;  // W runs of 16 dims
#pragma unroll
                for (int gr = 0; gr < GR; gr++)
#pragma unroll
                    for (int x = 0; x < W; x++) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            // HD 64: dims 8 (2c) + e of the first column, then of the second
                            const int tile = HD == 64 ? e & 7 : 16 * gr + e, col = HD == 64 ? e >> 3 : x;
                            v[e] = o[mt][tile][2 * hf + col] * inv;
                        }
                        const int d = HD == 64 ? 16 * c : 128 * gr + 32 * c + 16 * x;
                        if (!whole) store16(part + 2 * RB + r * HD + d, true, v);
                        else if (FULL || d < hd) store16(a.out, dst + d, a.typ, a.out_vec, v);
                    }
            }
        __syncwarp();
        t += (uint32_t)(s1 - s0);
    }
}

// Joins the partial results of units that lie in several runs.  grid: (units, slices of `per` groups of four dims of a unit's rows); what threads are
// left over take shares of the partial results.
constexpr int kJoinThreads = 128;
template <int HD, int RB>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a, int warps, int per) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint2 warp_sums[kJoinThreads / 32];
    __shared__ float4 s_val[kJoinThreads];
    __shared__ float s_m[kJoinThreads], s_sum[kJoinThreads];
    uint32_t* cum = reinterpret_cast<uint32_t*>(smem);
    uint32_t* units = cum + seqs.n_seqs + 1;
    const uint32_t total = line_up<RB>(seqs, pool, a, cum, units, warp_sums);
    pdl_wait();  // every block: this kernel's end then means that of the one before
    const Runs runs(total, warps);
    constexpr int P = part_floats<HD, RB>(), Q = HD / 4;
    const int shares = kJoinThreads / per, share = threadIdx.x / per, e = blockIdx.y * per + threadIdx.x - share * per;
    const int r = e / Q, d = (e - r * Q) * 4;
    for (uint32_t u = blockIdx.x; u < units[seqs.n_seqs]; u += gridDim.x) {
        const int i = seq_at(units, seqs.n_seqs, u);
        const SeqWork w = seq_work<RB>(seqs, pool, a, i);
        const uint32_t in = u - units[i], u0 = cum[i] + in * w.steps;
        const uint32_t b = runs.run_of(u0), last = runs.run_of(u0 + w.steps - 1);
        if (b == last) continue;                         // that run has written the rows
        const int kvh = in / w.blocks, row_lo = (in - kvh * w.blocks) * RB, row_n = min(RB, w.n * a.group - row_lo);
        const bool here = r < row_n;
        float mx = kNegInf, sum = 0.0f;
        float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (here) {
#pragma unroll 4
            for (uint32_t x = b + share; x <= last; x += shares) {
                const float* p = a.part + (size_t)(2 * x + (x == b ? 1 : 0)) * P;
                const float pm = p[r], ps = p[RB + r];
                const float4 v = *reinterpret_cast<const float4*>(p + 2 * RB + r * HD + d);
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
        if (share == 0 && here && d < pool.hd) {
            const int tok = (row_lo + r) / a.group, hq = (row_lo + r) - tok * a.group;
            const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + (int64_t)(kvh * a.group + hq) * pool.hd + d;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            store1(a.out, dst, a.typ, val.x * inv);
            store1(a.out, dst + 1, a.typ, val.y * inv);
            store1(a.out, dst + 2, a.typ, val.z * inv);
            store1(a.out, dst + 3, a.typ, val.w * inv);
        }
    }
}

struct RunPlan {
    int hd, mt, blocks;
    bool split;
    size_t bytes;
    int rows() const { return mt * (split ? 8 : 16); }
};
// f32 is always in the split form, for its 22 bits; 16-bit types where a unit has 8 rows at most, since it costs no more products there.  Two
// tiles share a step's keys and values where a unit has rows for them (heads of 256: their sums have no room in registers).
RunPlan plan_runs(const Kv8Pool& pool, uint32_t typ, int group, int max_rows) {
    RunPlan p;
    p.hd = pool.hd <= 64 ? 64 : pool.hd <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)group * (max_rows < 1 ? 1 : max_rows);
    p.split = typ == LC_TYPE_F32 || rows <= 8;
    p.mt = rows > (p.split ? 8 : 16) && p.hd < 256 ? 2 : 1;
    p.blocks = sm_count() * (p.hd == 256 ? 1 : p.mt > 1 ? 2 : 3);
    p.bytes = (size_t)2 * p.blocks * kRunWarps * p.rows() * (p.hd + 2) * sizeof(float);
    return p;
}

template <int HD, int MT, bool SPLIT, bool FULL>
int32_t runs_as(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int max_rows, int blocks, cudaStream_t s) {
    using Shape = RunShape<HD, MT, SPLIT>;
    const size_t cum = (size_t)(seqs.n_seqs + 1) * 4, smem = kRunWarps * Shape::kWarp + cum;
    LC_CUDA(ensure_smem_limit((const void*)kv8_runs_kernel<HD, MT, SPLIT, FULL>, smem));
    kv8_runs_kernel<HD, MT, SPLIT, FULL><<<blocks, kRunWarps * 32, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    // units by what max_rows says (the kernel goes on to more); few of them are cut into thinner slices, with more shares
    const int64_t rows = std::min<int64_t>(Shape::kRows, (int64_t)a.group * std::max(1, max_rows));
    const int64_t units = std::min<int64_t>(4096, ((int64_t)seqs.n_rows * a.group / Shape::kRows + seqs.n_seqs) * pool.n_kv);
    int per = kJoinThreads;
    while (per > 32 && units * ((rows * HD / 4 + per - 1) / per) < 2 * sm_count()) per /= 2;
    const unsigned slices = (unsigned)((Shape::kRows * HD / 4 + per - 1) / per);
    LC_CUDA(launch_pdl(kv8_join_kernel<HD, Shape::kRows>, dim3((unsigned)units, slices), dim3(kJoinThreads), 2 * cum, s, pool, seqs, a, blocks * kRunWarps, per));
    return LC_OK;
}
template <int HD, int MT, bool SPLIT>
int32_t runs_full(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int max_rows, int blocks, cudaStream_t s) {
    return pool.hd == HD ? runs_as<HD, MT, SPLIT, true>(pool, seqs, a, max_rows, blocks, s) : runs_as<HD, MT, SPLIT, false>(pool, seqs, a, max_rows, blocks, s);
}
template <int HD>
int32_t runs_of(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int max_rows, const RunPlan& p, cudaStream_t s) {
    if constexpr (HD < 256)
        if (p.mt == 2) return p.split ? runs_full<HD, 2, true>(pool, seqs, a, max_rows, p.blocks, s) : runs_full<HD, 2, false>(pool, seqs, a, max_rows, p.blocks, s);
    return p.split ? runs_full<HD, 1, true>(pool, seqs, a, max_rows, p.blocks, s) : runs_full<HD, 1, false>(pool, seqs, a, max_rows, p.blocks, s);
}

int32_t check_heads(const char* call, const Kv8Pool& pool, const Kv8Seqs& seqs, int32_t n_heads) {
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    // places of the line, row blocks of 8 at worst, in 31 bits
    const double chunks = (double)((int64_t)seqs.width << pool.page_shift) / kStep + 2, blocks = (double)seqs.n_rows * (n_heads / pool.n_kv) / 8 + seqs.n_seqs;
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
    TilePlan tiles;
    const int group = n_heads / pool.n_kv;
    *out_bytes = kv8_tiles_apply(pool, seqs, typ, group, rows->max_rows, &tiles) ? tiles.bytes : plan_runs(pool, typ, group, rows->max_rows).bytes;
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
    TilePlan tiles;
    const bool by_tiles = kv8_tiles_apply(pool, seqs, typ, group, rows->max_rows, &tiles);
    const size_t need = by_tiles ? tiles.bytes : plan.bytes;
    LC_CHECK(workspace_dev && workspace_bytes >= need && (uintptr_t)workspace_dev % 16 == 0, LC_ERR_INVALID,
             "lc_attention_kv8_dev: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", need, workspace_bytes);
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    window = std::min(window, 1 << 30);  // the kernels' differences of positions stay in 32 bits
    const size_t elem = typ == LC_TYPE_F32 ? 4 : 2;
    AttnArgs a{q_dev, out_dev, q_stride, out_stride, (int)typ, n_heads, group, window, rows_aligned(q_dev, q_stride, elem, 16), rows_aligned(out_dev, out_stride, elem, 16),
               scale * 1.44269504088896f, (float*)workspace_dev};
    cudaStream_t s = stream_or_own(stream_);
    if (by_tiles) return launch_kv8_tiles(pool, seqs, a, tiles, s);
    if (plan.hd == 64) return runs_of<64>(pool, seqs, a, rows->max_rows, plan, s);
    if (plan.hd == 128) return runs_of<128>(pool, seqs, a, rows->max_rows, plan, s);
    return runs_of<256>(pool, seqs, a, rows->max_rows, plan, s);
}

}  // extern "C"
