// Attention over the key/value cache in 4 bits: out = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the slots j up to the row's own.
//
// Here: few rows per sequence, by runs.  A unit is (sequence, kv head, row block of 8 NG rows = tokens x heads of the group); the units' steps of 16 keys stand in one line, which is cut into equal
// runs, one per warp, so that contexts of any lengths keep all warps equally long at work; what lies in several runs is joined by the next kernel.  Bytes come through a ring of the warp's
// own in shared memory (cp.async) and become f16 values, exact, in registers, on the way into the matrix unit (mma.sync m16n8k16, f32 sums):
//   Scores  queries are the operand of 16 rows, keys that of 8 columns.  Queries are f16 after a power of two for each row (16-bit types: exact down to 2^-24 of the row's largest element), f32 ones a
//           high and a low part, 22 bits; where a unit has 8 rows the low parts are the operand's other 8 rows and cost nothing.
//   Values  are the operand of 16 rows (dims), weights that of 8 columns (rows of queries), which the scores' layout already is.  Weights are 2^(s - max + 10) in f16; f32: and what that rounding lost, in a second
//           product, a step's sums added in f32, so that what the matrix unit cuts off when it adds stays within 16 keys.
// Dims of a score and keys of a sum may stand in any order, so a thread takes neighbouring dims of its key, whose scale they share, and two keys' dims become pairs by one byte permutation for eight of them.
//
// Why 11 bits are enough for 16-bit types' weights: each is off by up to 2^-11 of itself, either way, and an output is a mean over many keys.  Against 64 bits, and with weights of 32 bits: bf16 1.7e-3 and 1.7e-3,
// f16 2.7e-4 and 2.1e-4, most of it the outputs' own rounding.  A second product for the low parts, as f32 has it, would double the products with the values.
//
// 64 sequences of 128 to 4,096 slots, 32 heads over 8 of 128 in bf16: 37 us with the join, 87 MB (a floor of 13).  What bounds it are instructions: 360 a step of 16 keys, of which the matrix unit's are 16; 50 % of the
// issue slots at 12 warps an SM (153 registers), the rest is the beginning and the end of runs of 20 steps.  Three blocks an SM for up to 8 rows; four (128 registers) take longer, 38.5 us, 42.7 instead of 41.1 in f32, 98 instead of 94 with
// 16 sequences of 8,000 to 32,000, and five spill.  Two sequences of 60,001 and 131,000 slots, four tokens, 64 heads over 8 in f16: 123 us with the join, 220 MB (34): 32 rows share a step's unpacking, and 8 warps of
// 235 registers wait for one another's results (two groups of rows instead of four: 172).
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

constexpr float kWeightUp = 10.0f;   // weights are 2^this too large, and up to 2^4 more before the reference is raised: 2^14 at most, and f16's smallest is 2^-34 of the largest

template <int HD, int NG, bool F32> struct Run4Shape {
    static constexpr int kRows = 8 * NG;
    static constexpr int kTiles = NG == 1 ? 1 : NG / 2 * (F32 ? 2 : 1);   // operand tiles of 16 rows of queries
    static constexpr int kStages = HD == 256 && NG > 1 ? 2 : 4;
    static constexpr int kRing = kStages * Ring4<HD, true, true, kStages>::kPlace;
    static constexpr bool kQueriesShared = HD == 256 || kTiles > 1;       // operand fragments of the queries in shared memory, not in registers
    static constexpr int kQueries = kQueriesShared ? kTiles * (HD / 16) * 512 : 0;
    static constexpr int kWarp = kRing + kQueries;
    static constexpr int kByRegisters = HD == 256 ? 2 : NG <= 2 ? 3 : 2;   // with 8 rows four take 1 to 8 % longer, see above
    static constexpr int kByMemory = (220 << 10) / (kRunWarps * kWarp + 2048);
    static constexpr int kBlocks = kByRegisters < kByMemory ? kByRegisters : kByMemory;
};

template <int HD, int NG, bool F32, bool FULL>
__global__ void __launch_bounds__(kRunWarps * 32, Run4Shape<HD, NG, F32>::kBlocks)
kv4_runs_kernel(Kv4Pool pool, Kv8Seqs seqs, AttnArgs a) {
    using Shape = Run4Shape<HD, NG, F32>;
    constexpr int RB = Shape::kRows, S = Shape::kStages, TILES = Shape::kTiles;
    constexpr int KS = HD / 16;             // k steps of the scores
    constexpr int NT = HD / 16;             // tiles of 16 dims of the output
    constexpr int KW = HD / 32;             // words of a key that a thread has
    constexpr int VW = HD / 64;             // words of a value
    constexpr bool LOW_ROWS = F32 && NG == 1;   // the low parts are rows 8 .. 15 of the tile
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
    uint4* const qs = reinterpret_cast<uint4*>(mine + Shape::kRing);
    const int hd = FULL ? HD : pool.hd;

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
        const int row_lo = at.rb * RB, row_n = min(RB, w.n * a.group - row_lo);
        using Ring = Ring4<HD, FULL, true, S>;
        Ring keys(pool, hd, seqs.table + (size_t)at.seq * seqs.width, at.kvh, w.step0, ring, lane);
        bool bad = keys.begin(s0, w.inside ? s1 : s0);
#pragma unroll
        for (int k = 0; k < S - 1; k++) bad = keys.fetch(s0 + k, k == 0) || bad;

        // The queries as operand fragments.  A thread's dims are HD / 4 in a row, eight of which make two k steps: (0, 4), (1, 5) and (2, 6), (3, 7), as the keys' words give them.
        uint32_t qf[Shape::kQueriesShared ? 1 : KS][4];
        float rf[NG];                        // what a row's scores are multiplied by
        int limit[NG];                       // last slot that the row sees (-1: no row)
        {
            const float head = kUnit4 * pool.k_scale[at.kvh];
#pragma unroll
            for (int pair = 0; pair < (NG + 1) / 2; pair++) {
                float v[2][HD / 4], up[2];
#pragma unroll
                for (int x = 0; x < (NG == 1 ? 1 : 2); x++) {
                    const int gr = 2 * pair + x, r = 8 * gr + g;
                    const bool has = r < row_n;
                    const int tok = has ? (row_lo + r) / a.group : 0, hq = has ? (row_lo + r) - tok * a.group : 0;
                    const int64_t src = (int64_t)(w.first + tok) * a.q_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                    limit[gr] = has ? w.ctx + tok : -1;
                    float top = 0.0f;
#pragma unroll
                    for (int j = 0; j < HD / 64; j++) {
                        const int d = c * (HD / 4) + 16 * j;
                        float* u = v[x] + 16 * j;
                        if (has && (FULL || d < hd)) load16(a.q, src + d, a.typ, a.q_vec, u);
                        else
#pragma unroll
                            for (int e = 0; e < 16; e++) u[e] = 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; e++) top = max_nan(top, fabsf(u[e]));
                    }
                    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    float down;
                    row_scale(top, up[x], down);
                    // not finite: the row is NaN
                    rf[gr] = top < INFINITY ? score_factor(a.scale_log2, down, head) : __int_as_float(0x7fffffff);
                }
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t hi[2][2] = {}, lo[2][2] = {};
#pragma unroll
                    for (int x = 0; x < (NG == 1 ? 1 : 2); x++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const int e = 8 * (ks >> 1) + 2 * (ks & 1) + y;
                            const float p = v[x][e] * up[x], q = v[x][e + 4] * up[x];
                            if (F32) h2_split(p, q, hi[x][y], lo[x][y]);
                            else hi[x][y] = h2_pack(p, q);
                        }
                    // (row g, row g + 8) of the first two dims, then of the others
                    const uint4 f = LOW_ROWS ? make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]) : make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
                    if (Shape::kQueriesShared) {
                        qs[((F32 && NG > 1 ? 2 * pair : pair) * KS + ks) * 32 + lane] = f;
                        if (F32 && NG > 1) qs[((2 * pair + 1) * KS + ks) * 32 + lane] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
                    } else {
                        uint32_t(&q4)[4] = qf[Shape::kQueriesShared ? 0 : ks];
                        q4[0] = f.x; q4[1] = f.y; q4[2] = f.z; q4[3] = f.w;
                    }
                }
            }
        }

        // o: dims 2 t (places 0, 1) and 2 t + 1 (places 2, 3) of the thread's, of rows 2c, 2c + 1 of the group; m, l: of row g
        float o[NG][NT][4], m[NG], l[NG], off[NG];
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[gr][t][e] = 0.0f;
            m[gr] = kNegInf;
            l[gr] = 0.0f;
            off[gr] = kWeightUp;
        }
        auto is_far = [](float top) { return fabsf(top) > 65536.0f && top != kNegInf; };  // so far from 0 that a reference has no bits left for what is added to it
        bool far = false;                    // some row of the warp's has such a reference
        // rows see all keys up to the first row's slot (with a window, from the last row's on)
        const int sees = w.ctx + row_lo / a.group, from = a.window > 0 ? w.ctx + (row_lo + row_n - 1) / a.group - a.window : -1;
        const int plain0 = from < 0 ? 0 : from / kStep + 1 - w.step0, plain1 = (sees + 1) / kStep - w.step0;   // steps whose keys all rows see
        for (int st = s0; st < s1; st++) {
            cp_async_wait<S - 2>();
            __syncwarp();
            bad = keys.fetch(st + S - 1) || bad;  // into the place of the step before
            const bool plain = st >= plain0 && st < plain1;
            const unsigned char* kp = mine + (st & (S - 1)) * Ring::kPlace;
            const unsigned char* scales = kp + Ring::kScales;
            float s[NG][2][2];               // [group][tile of 8 keys][two keys]
            {
                float dot[TILES][2][4];
#pragma unroll
                for (int tl = 0; tl < 2; tl++) {
                    const int row = 8 * tl + g;
                    uint32_t kw[KW];
                    if (FULL) lds_words<KW>(kp + row * (HD / 2) + c * (HD / 8), kw);
                    else lds_words8<KW>(kp + row * (hd >> 1) + c * (HD / 8), kw);
                    const unsigned char* sc = scales + row * (hd >> 4) + c * (HD / 64);
                    uint32_t bytes = 0;
                    if (HD == 64) bytes = *sc;
                    else if (FULL) bytes = HD == 128 ? *reinterpret_cast<const uint16_t*>(sc) : *reinterpret_cast<const uint32_t*>(sc);
                    else
#pragma unroll
                        for (int j = 0; j < HD / 64; j++) bytes |= (uint32_t)sc[j] << (8 * j);
                    bytes &= 0x7f7f7f7fu;
#pragma unroll
                    for (int j = 0; j < HD / 64; j++) {   // 16 dims: two words, four k steps
                        const Scale4 k4 = scale4_both(bytes, j);
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            uint32_t kv[4];
                            values8(kw[2 * j + x], k4, kv);
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                const int ks = 4 * j + 2 * x + y;
#pragma unroll
                                for (int tile = 0; tile < TILES; tile++) {
                                    uint4 f;
                                    if (Shape::kQueriesShared) f = qs[(tile * KS + ks) * 32 + lane];
                                    else {
                                        const uint32_t(&q4)[4] = qf[Shape::kQueriesShared ? 0 : ks];
                                        f = make_uint4(q4[0], q4[1], q4[2], q4[3]);
                                    }
                                    const uint32_t fa[4] = {f.x, f.y, f.z, f.w};
                                    if (ks == 0) mma_f16_first(dot[tile][tl], fa, kv[2 * y], kv[2 * y + 1]);
                                    else mma_f16(dot[tile][tl], fa, kv[2 * y], kv[2 * y + 1]);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
#pragma unroll
                    for (int tl = 0; tl < 2; tl++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            if (LOW_ROWS) s[gr][tl][k] = dot[0][tl][k] + dot[0][tl][2 + k];
                            else if (F32) s[gr][tl][k] = dot[gr / 2 * 2][tl][2 * (gr & 1) + k] + dot[TILES > 1 ? gr / 2 * 2 + 1 : 0][tl][2 * (gr & 1) + k];
                            else s[gr][tl][k] = dot[gr / 2][tl][2 * (gr & 1) + k];
                        }
            }
            if (keys.any_bad && keys.outside(st)) {  // the rows that see its keys are NaN
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[gr][e >> 1][e & 1] = __int_as_float(0x7fffffff);
            }
            if (!plain) {
                const int key0 = (w.step0 + st) * kStep;
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = key0 + 8 * (e >> 1) + 2 * c + (e & 1);
                        if (key > limit[gr] || (a.window > 0 && key <= limit[gr] - a.window)) s[gr][e >> 1][e & 1] = kNegInf;
                    }
            }
            float mx[NG];
            bool raise = false;
#pragma unroll
            for (int gr = 0; gr < NG; gr++) mx[gr] = fmaxf(fmaxf(s[gr][0][0], s[gr][0][1]), fmaxf(s[gr][1][0], s[gr][1][1]));
#pragma unroll
            for (int gr = 0; gr < NG; gr++) mx[gr] = fmaxf(mx[gr], __shfl_xor_sync(0xffffffffu, mx[gr], 1));
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                mx[gr] = __fmul_rn(fmaxf(mx[gr], __shfl_xor_sync(0xffffffffu, mx[gr], 2)), rf[gr]);
                raise = raise || mx[gr] - m[gr] > 4.0f;   // the difference: far from 0, m + 4 may be rounded up to the next number, which mx may be
            }
            // the references are raised when a row's maximum has grown by more than 2^4; one vote for all groups, whose chains of instructions then run side by side
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const float top = fmaxf(mx[gr], m[gr]), corr = top == kNegInf ? 1.0f : exp2_fast(m[gr] - top);
                    l[gr] *= corr;
                    m[gr] = top;
                    off[gr] = top == kNegInf ? kWeightUp : kWeightUp - top;
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
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = fmaf(s[gr][e >> 1][e & 1], rf[gr], off[gr]);
                if (far) {  // products rounded by themselves, as the reference is: their difference is exact near it
                    const bool mine = is_far(m[gr]);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = mine ? __fadd_rn(__fsub_rn(__fmul_rn(s[gr][e >> 1][e & 1], rf[gr]), m[gr]), kWeightUp) : v[e];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = exp2_fast(v[e]);
                l[gr] += (v[0] + v[1]) + (v[2] + v[3]);
                if (F32) {
                    h2_split(v[0], v[1], ph[gr][0], pl[gr][0]);
                    h2_split(v[2], v[3], ph[gr][1], pl[gr][1]);
                } else {
                    ph[gr][0] = h2_pack(v[0], v[1]);
                    ph[gr][1] = h2_pack(v[2], v[3]);
                }
            }
            // values: a thread's keys are 2c, 2c + 1, 8 + 2c, 9 + 2c, its dims HD / 8 in a row
            const unsigned char* vp = kp + Ring::kHalf;
            uint32_t vw[4][VW], vb[4][HD == 256 ? 2 : 1];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int row = (x >> 1) * 8 + 2 * c + (x & 1);
                if (FULL) lds_words<VW>(vp + Ring::value_chunk(row, HD == 256 ? g : HD == 128 ? g >> 1 : g >> 2) * 16 + (HD == 256 ? 0 : HD == 128 ? (g & 1) * 8 : (g & 3) * 4), vw[x]);
                else lds_words8<VW>(vp + row * (hd >> 1) + g * (HD / 16), vw[x]);
                const unsigned char* sc = scales + HD + row * (hd >> 4) + (HD == 256 ? 2 * g : HD == 128 ? g : g >> 1);
                vb[x][0] = sc[0];
                if (HD == 256) vb[x][HD == 256 ? 1 : 0] = sc[1];
            }
#pragma unroll
            for (int half = 0; half < (HD == 256 ? 2 : 1); half++) {
                const Scale4 sa = scale4_pair(vb[0][half], vb[1][half]), sb = scale4_pair(vb[2][half], vb[3][half]);
#pragma unroll
                for (int wd = 0; wd < (VW < 2 ? 1 : 2); wd++) {
                    const int word = 2 * half + wd;
#pragma unroll
                    for (int q = 0; q < 2; q++) {   // four dims
                        const uint32_t xa = __byte_perm(vw[0][word], vw[1][word], q ? 0x7632 : 0x5410), xb = __byte_perm(vw[2][word], vw[3][word], q ? 0x7632 : 0x5410);
#pragma unroll
                        for (int b = 0; b < 2; b++) {   // two dims: a tile
                            const uint32_t ya = b ? xa >> 8 : xa, yb = b ? xb >> 8 : xb;
                            const uint32_t vf[4] = {value_lo(ya, sa), value_hi(ya, sa), value_lo(yb, sb), value_hi(yb, sb)};
#pragma unroll
                            for (int gr = 0; gr < NG; gr++) {
                                float(&oo)[4] = o[gr][4 * word + 2 * q + b];
                                if (F32) {
                                    float acc[4];
                                    mma_f16_first(acc, vf, pl[gr][0], pl[gr][1]);
                                    mma_f16(acc, vf, ph[gr][0], ph[gr][1]);
#pragma unroll
                                    for (int e = 0; e < 4; e++) oo[e] += acc[e];
                                } else {
                                    mma_f16(oo, vf, ph[gr][0], ph[gr][1]);
                                }
                            }
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();
        if (bad && lane == 0) kv8_raise(seqs, at.seq);

        const bool starts = s0 == 0, ends = s1 == w.steps, whole = starts && ends;
        const float unit = kUnit4 * pool.v_scale[at.kvh];
        float* part = a.part + (size_t)(2 * run + (starts ? 1 : 0)) * part_floats<HD, RB>();
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
            float sum = l[gr];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (!w.inside) sum = __int_as_float(0x7fffffff);
            if (c == 0 && 8 * gr + g < row_n) {
                const int r = 8 * gr + g;
                if (!whole) { part[r] = m[gr]; part[RB + r] = sum; }
                else if (a.lse) {
                    const int tok = (row_lo + r) / a.group;
                    a.lse[(int64_t)(w.first + tok) * a.lse_stride + at.kvh * a.group + row_lo + r - tok * a.group] = (m[gr] + (log2f(sum) - kWeightUp)) * 0.693147180559945f;
                }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int r = 8 * gr + 2 * c + x;
                const float total = __shfl_sync(0xffffffffu, sum, 8 * c + 4 * x);
                if (r >= row_n) continue;
                const float by = whole ? unit / total : unit;   // a NaN sum makes all of the row NaN
                const int tok = (row_lo + r) / a.group, hq = (row_lo + r) - tok * a.group;
                const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + (int64_t)(at.kvh * a.group + hq) * hd;
                constexpr int N = HD == 64 ? 8 : 16;  // dims stored at a time
#pragma unroll
                for (int half = 0; half < (HD == 256 ? 2 : 1); half++) {
                    float v[N];
#pragma unroll
                    for (int e = 0; e < N; e++) v[e] = o[gr][8 * half + (e >> 1)][2 * (e & 1) + x] * by;
                    const int d = HD == 64 ? 8 * g : HD == 128 ? 16 * g : 32 * g + 16 * half;
                    if (!whole) store_run<N>(part + 2 * RB + r * HD + d, true, v);
                    else if (FULL || d < hd) store_run<N>(a.out, dst + d, a.typ, a.out_vec, v);
                }
            }
        }
        __syncwarp();
    }
}

// Joins the partial results of units that lie in several runs.  A run's record says which unit begins in it; a block looks through those of kJoinRuns runs, a slice of kJoinRows
// rows of each.  Threads have four dims of a row each, and shares of the partial results.  (A block per run and four rows: 12 us more after two sequences of 131,000 keys, 137 instead of 125 with the runs.)
constexpr int kJoinThreads = 256, kJoinRuns = 8, kJoinRows = 2;
template <int HD, int RB>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(AttnArgs a, int hd, int runs) {
    constexpr int P = part_floats<HD, RB>(), Q = HD / 4, CELLS = kJoinRows * Q, SHARES = kJoinThreads / CELLS;
    __shared__ float4 s_val[kJoinThreads];
    __shared__ float2 s_sum[kJoinThreads];
    pdl_wait();  // every block: this kernel's end then means that of the one before
    const int b0 = blockIdx.x * kJoinRuns, row0 = blockIdx.y * kJoinRows, cell = threadIdx.x % CELLS, share = threadIdx.x / CELLS;
    const int r = row0 + cell / Q, d = (cell % Q) * 4;
    // the runs' records, one per lane
    const int lane = threadIdx.x & 31;
    UnitRecord mine;
    mine.row_n = 0;
    if (lane < kJoinRuns && b0 + lane < runs) {
        *reinterpret_cast<int4*>(&mine) = *reinterpret_cast<const int4*>(&a.records[b0 + lane]);
        mine.last = a.records[b0 + lane].last;
    }
    for (uint32_t which = __ballot_sync(0xffffffffu, mine.row_n > row0); which; which &= which - 1) {
        const int k = __ffs(which) - 1, b = b0 + k, last = __shfl_sync(0xffffffffu, mine.last, k), n = __shfl_sync(0xffffffffu, mine.row_n, k);
        const int4 at = make_int4(__shfl_sync(0xffffffffu, mine.first, k), __shfl_sync(0xffffffffu, mine.kvh, k), __shfl_sync(0xffffffffu, mine.row_lo, k), n);
        float mx = kNegInf, sum = 0.0f;
        float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](float pm, float ps, const float4& v) {
            const float m2 = fmaxf(mx, pm), ref = m2 == kNegInf ? 0.0f : m2;
            const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(pm - ref);
            sum = f0 * sum + (isnan(ps) ? ps : f1 * ps);
            val.x = fmaf(f0, val.x, f1 * v.x); val.y = fmaf(f0, val.y, f1 * v.y);
            val.z = fmaf(f0, val.z, f1 * v.z); val.w = fmaf(f0, val.w, f1 * v.w);
            mx = m2;
        };
        if (r < n) {
#pragma unroll 4
            for (int x = b + share; x <= last; x += SHARES) {
                const float* q = a.part + (size_t)(2 * x + (x == b ? 1 : 0)) * P;  // of the run itself the second place, of the later ones the first
                add(q[r], q[RB + r], *reinterpret_cast<const float4*>(q + 2 * RB + r * HD + d));
            }
        }
        s_val[threadIdx.x] = val;
        s_sum[threadIdx.x] = make_float2(mx, sum);
        __syncthreads();
        if (share == 0 && r < n) {
#pragma unroll
            for (int x = 1; x < SHARES; x++) {
                const float2 ms = s_sum[x * CELLS + cell];
                add(ms.x, ms.y, s_val[x * CELLS + cell]);
            }
            if (d < hd) {
                const int tok = (at.z + r) / a.group, hq = (at.z + r) - tok * a.group;
                const int64_t dst = (int64_t)(at.x + tok) * a.out_stride + (int64_t)(at.y * a.group + hq) * hd + d;
                const float inv = 1.0f / sum;
                store1(a.out, dst, a.typ, val.x * inv);
                store1(a.out, dst + 1, a.typ, val.y * inv);
                store1(a.out, dst + 2, a.typ, val.z * inv);
                store1(a.out, dst + 3, a.typ, val.w * inv);
                if (a.lse && d == 0) a.lse[(int64_t)(at.x + tok) * a.lse_stride + at.y * a.group + hq] = (mx + (log2f(sum) - kWeightUp)) * 0.693147180559945f;
            }
        }
        __syncthreads();
    }
}

struct Run4Plan {
    int hd, groups, blocks;
    size_t bytes;
};
template <int HD, bool F32> int run_blocks(int groups) {
    if (HD < 256 && groups == 4) return Run4Shape<HD, HD < 256 ? 4 : 1, F32>::kBlocks;
    return groups == 2 ? Run4Shape<HD, 2, F32>::kBlocks : Run4Shape<HD, 1, F32>::kBlocks;
}
// As many groups of 8 rows share a step's keys and values as a unit has rows for: four at most, whose sums are 128 registers (two for heads of 256).
int run_groups(const Kv4Pool& pool, int group, int max_rows) {
    const int64_t rows = (int64_t)group * (max_rows < 1 ? 1 : max_rows);
    return rows <= 8 ? 1 : rows <= 16 || pool.hd > 128 ? 2 : 4;
}
int most_groups(const Kv4Pool& pool) { return pool.hd > 128 ? 2 : 4; }
Run4Plan plan_runs(const Kv4Pool& pool, uint32_t typ, int groups) {
    Run4Plan p;
    p.hd = pool.hd <= 64 ? 64 : pool.hd <= 128 ? 128 : 256;
    p.groups = groups;
    const bool f32 = typ == LC_TYPE_F32;
    p.blocks = sm_count() * (p.hd == 64    ? (f32 ? run_blocks<64, true>(p.groups) : run_blocks<64, false>(p.groups))
                             : p.hd == 128 ? (f32 ? run_blocks<128, true>(p.groups) : run_blocks<128, false>(p.groups))
                                           : (f32 ? run_blocks<256, true>(p.groups) : run_blocks<256, false>(p.groups)));
    p.bytes = (size_t)p.blocks * kRunWarps * (sizeof(UnitRecord) + (size_t)2 * 8 * p.groups * (p.hd + 2) * sizeof(float));
    return p;
}
bool tiles_fit(const Kv4Pool& pool, const Kv8Seqs& seqs, int group) {
    TilePlan tiles;
    return line_fits(pool, seqs, group, kTileRows2) && kv8_tiles_plan(pool, seqs, group, &tiles);
}
// Whether tiles are faster than runs, us in runs / in tiles.  128 rows (tokens x heads of a group) of a sequence and kv head: bf16, 32 heads over 8 of 128, one sequence behind 1,000 tokens 20.9 / 24.8, behind
// 4,000 28.1 / 28.5, behind 16,000 52.3 / 40.6 (how long contexts are is not known here), 4 behind 2,000 36.7 / 32.9, 16 95.5 / 46.1, 64 behind 1,000 197 / 135; f32 one behind 4,000 34.7 / 36.5, 16 135 / 73,
// 64 275 / 203; heads of 64 one 21.7 / 21.9, 16 69.7 / 40.6.  64 rows, a block for each sequence and kv head, 16-bit types: 8 blocks 17.8 / 23.1, 25.8 / 26.4 and 38.4 / 38.6 (behind 1,000, 4,000, 16,000), 32
// blocks 27.9 / 29.3 and 36.0 / 34.0, 128 56.4 / 45.6 and 57.4 / 48.0, 144 61.1 / 45.6, but 152, more than SMs, 64.0 / 87.1 and 512 112 / 114; f32 77 / 71 with 128 and 88 / 137 with 152; heads of 64 41.0 / 40.3
// with 128.  32 rows: 39 / 48.
bool tiles_pay(const Kv4Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows) {
    const int64_t blocks = (int64_t)seqs.n_seqs * pool.n_kv;
    const bool one_wave = blocks <= sm_count() && 2 * blocks >= sm_count();
    return (int64_t)group * max_rows >= (typ != LC_TYPE_F32 && pool.hd > 64 && one_wave ? 64 : 128);
}
struct Plan {
    bool by_tiles;
    TilePlan tiles;
    Run4Plan runs;
    size_t bytes() const { return by_tiles ? tiles.bytes : runs.bytes; }
};
// The faster kernel, unless its line does not fit: a call with many more rows than its max_rows says goes by tiles then, or by as many groups as it takes.
Plan plan_call(const Kv4Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows) {
    Plan p;
    int groups = run_groups(pool, group, max_rows);
    p.by_tiles = kv8_tiles_plan(pool, seqs, group, &p.tiles) && line_fits(pool, seqs, group, kTileRows2) &&
                 (tiles_pay(pool, seqs, typ, group, max_rows) || !line_fits(pool, seqs, group, 8 * groups));
    while (!p.by_tiles && groups < most_groups(pool) && !line_fits(pool, seqs, group, 8 * groups)) groups *= 2;
    p.runs = plan_runs(pool, typ, groups);
    return p;
}
// The most that a call with at most these arguments needs: fewer rows, sequences or pages may go by runs instead of tiles, take fewer groups (whose
// runs are more), or have their keys cut where larger ones are not, so the answer goes by none of them.
size_t most_bytes(const Kv4Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows) {
    const bool any = !line_fits(pool, seqs, group, 8);  // then a smaller max_rows may lead to every kernel
    size_t most = kv8_tiles_most_bytes(pool, any ? 1 << 30 : (int64_t)group * max_rows);
    for (int groups = any ? most_groups(pool) : run_groups(pool, group, max_rows); groups >= 1; groups /= 2) most = std::max(most, plan_runs(pool, typ, groups).bytes);
    return most;
}

template <int HD, int NG, bool F32, bool FULL>
int32_t runs_as(const Kv4Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int blocks, cudaStream_t s) {
    using Shape = Run4Shape<HD, NG, F32>;
    const size_t cum = (size_t)(seqs.n_seqs + 1) * 4, smem = kRunWarps * Shape::kWarp + cum;
    LC_CUDA(ensure_smem_limit((const void*)kv4_runs_kernel<HD, NG, F32, FULL>, smem));
    kv4_runs_kernel<HD, NG, F32, FULL><<<blocks, kRunWarps * 32, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    LC_CUDA(launch_pdl(kv4_join_kernel<HD, Shape::kRows>, dim3((unsigned)(blocks * kRunWarps + kJoinRuns - 1) / kJoinRuns, Shape::kRows / kJoinRows), dim3(kJoinThreads), 0, s, a, pool.hd, blocks * kRunWarps));
    return LC_OK;
}
template <int HD, int NG>
int32_t runs_full(const Kv4Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (a.typ == LC_TYPE_F32) return pool.hd == HD ? runs_as<HD, NG, true, true>(pool, seqs, a, blocks, s) : runs_as<HD, NG, true, false>(pool, seqs, a, blocks, s);
    return pool.hd == HD ? runs_as<HD, NG, false, true>(pool, seqs, a, blocks, s) : runs_as<HD, NG, false, false>(pool, seqs, a, blocks, s);
}
template <int HD>
int32_t runs_of(const Kv4Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const Run4Plan& p, cudaStream_t s) {
    if constexpr (HD < 256)
        if (p.groups == 4) return runs_full<HD, 4>(pool, seqs, a, p.blocks, s);
    return p.groups == 2 ? runs_full<HD, 2>(pool, seqs, a, p.blocks, s) : runs_full<HD, 1>(pool, seqs, a, p.blocks, s);
}

int32_t check_heads(const char* call, const Kv4Pool& pool, const Kv8Seqs& seqs, int32_t n_heads) {
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    const int group = n_heads / pool.n_kv;
    // a sequence outside its table may have all rows: what a call's rows are in the kernels' 32 bits
    LC_CHECK((int64_t)seqs.n_rows * group < (int64_t)0x7fffffff - kTileRows2, LC_ERR_INVALID, "%s: %d rows of %d heads are too many for one call", call, seqs.n_rows, n_heads);
    LC_CHECK(line_fits(pool, seqs, group, 8 * most_groups(pool)) || tiles_fit(pool, seqs, group), LC_ERR_INVALID, "%s: %d rows of %d heads over tables of %d pages are too many for one call", call, seqs.n_rows, n_heads, seqs.width);
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_attention_kv4_workspace(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, int32_t n_heads, size_t* out_bytes) {
    const char* call = "lc_attention_kv4_workspace";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_CHECK(out_bytes, LC_ERR_INVALID, "%s: null output", call);
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    LC_TRY(check_heads(call, pool, seqs, n_heads));
    if (n_rows == 0 || seqs.n_seqs == 0) {  // nothing to do, as for the call itself
        *out_bytes = 16;
        return LC_OK;
    }
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    *out_bytes = most_bytes(pool, seqs, typ, n_heads / pool.n_kv, rows->max_rows);
    return LC_OK;
}

int32_t lc_attention_kv4_dev(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, const void* q_dev, int64_t q_stride, int32_t n_heads, float scale, int32_t window,
                             void* out_dev, int64_t out_stride, float* lse_dev, int64_t lse_stride, void* workspace_dev, size_t workspace_bytes, void* stream_) {
    const char* call = "lc_attention_kv4_dev";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    LC_TRY(check_heads(call, pool, seqs, n_heads));
    LC_CHECK(window >= 0, LC_ERR_INVALID, "%s: window=%d", call, window);
    LC_CHECK(scale >= 0.0f && scale <= 2.0e38f, LC_ERR_INVALID, "%s: scale=%g", call, scale);
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(q_dev && out_dev, LC_ERR_INVALID, "%s: null queries or output", call);
    LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && out_stride >= (int64_t)n_heads * pool.hd && (!lse_dev || lse_stride >= n_heads), LC_ERR_INVALID, "%s: rows overlap", call);
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    const int group = n_heads / pool.n_kv;
    const Plan plan = plan_call(pool, seqs, typ, group, rows->max_rows);
    const size_t need = plan.bytes();
    LC_CHECK(workspace_dev && workspace_bytes >= need && (uintptr_t)workspace_dev % 16 == 0, LC_ERR_INVALID, "%s: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", call, need, workspace_bytes);
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    window = std::min(window, 1 << 30);  // the kernels' differences of slots stay in 32 bits
    const size_t elem = typ == LC_TYPE_F32 ? 4 : 2;
    AttnArgs a{q_dev, out_dev, q_stride, out_stride, (int)typ, group, window, rows_aligned(q_dev, q_stride, elem, 16), rows_aligned(out_dev, out_stride, elem, 16), scale * 1.44269504088896f,
               (float*)workspace_dev, (UnitRecord*)workspace_dev, lse_dev, lse_stride, kWeightUp};
    cudaStream_t s = stream_or_own(stream_);
    if (plan.by_tiles) return launch_kv4_tiles(pool, seqs, a, plan.tiles, s);
    a.part = (float*)((char*)workspace_dev + (size_t)plan.runs.blocks * kRunWarps * sizeof(UnitRecord));
    if (plan.runs.hd == 64) return runs_of<64>(pool, seqs, a, plan.runs, s);
    if (plan.runs.hd == 128) return runs_of<128>(pool, seqs, a, plan.runs, s);
    return runs_of<256>(pool, seqs, a, plan.runs, s);
}

}  // extern "C"
