// What weight a call's rows gave the cached keys: mass[sequence][kv head][slot] += sum over rows and heads of the group of exp(scale q . k - lse).
//
// By runs, as attention of few rows: the steps of 16 keys of all sequences and kv heads stand in one line, which is cut into equal runs, one per warp.  A step's keys are the operand of 16 rows and
// queries, 8 at a time, that of 8 columns (mma.sync m16n8k16 in f16, as there); a key's sum over the rows then lies in four threads of a row of the result.  The warp goes over
// its steps once for every block of 8 NG rows and adds to the sums itself, so that every sum is added to by one warp, in the order of the rows.
//
// 64 sequences of 128 to 4,096 slots, one row of 32 heads over 8 of 128 in bf16: 22.6 us, 48 MB (a floor of 7.3).  What bounds it are instructions, 270 to 400 a step of 16 keys: 60 % of the issue slots at 20 warps an SM.  A first,
// simple kernel: 86.
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_kv4_weights.cuh"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

template <int HD, int NG, bool F32> struct WeightShape {
    static constexpr int kRows = 8 * NG;
    static constexpr int kTerms = F32 ? 2 : 1;
    static constexpr int kStages = HD == 64 ? 8 : 4;
    static constexpr int kRing = kStages * Ring4<HD, true, false, kStages>::kPlace;
    static constexpr bool kQueriesShared = HD == 256 || NG > 1;           // operand fragments of the queries in shared memory, not in registers
    static constexpr int kQueries = kQueriesShared ? NG * kTerms * (HD / 32) * 512 : 0;
    static constexpr int kWarp = kRing + kQueries;
    static constexpr int kByRegisters = HD == 256 ? 2 : F32 ? 4 : 5;
    static constexpr int kByMemory = (220 << 10) / (kRunWarps * kWarp + 2048);
    static constexpr int kBlocks = kByRegisters < kByMemory ? kByRegisters : kByMemory;
};

// A sequence's part of the line: of each kv head kUnitCost places and `blocks` for each step.
struct WeightWork {
    int first, n, ctx, blocks, step0, steps;
};
template <int RB>
__device__ __forceinline__ WeightWork weight_work(const Kv8Seqs& s, const Kv8Pool& p, const WeightArgs& a, int i) {
    WeightWork w;
    w.blocks = w.step0 = w.steps = 0;
    w.ctx = s.ctx[i];
    if (!kv8_span(s, i, w.first, w.n) || w.n == 0 || !kv8_in_table(s, p, w.ctx, w.n) || w.ctx + w.n > a.capacity) return w;
    w.blocks = (w.n * a.group + RB - 1) / RB;
    const int lo = a.window > 0 ? max(0, w.ctx - a.window + 1) : 0;
    w.step0 = lo / kStep;
    w.steps = (w.ctx + w.n + kStep - 1) / kStep - w.step0;
    return w;
}
// cum[i] = places before sequence i; by one block, returns the total
template <int RB>
__device__ __forceinline__ uint32_t weight_line(const Kv8Seqs& s, const Kv8Pool& p, const WeightArgs& a, uint32_t* cum, uint32_t* warp_sums) {
    const int per = (s.n_seqs + blockDim.x - 1) / blockDim.x, i0 = min((int)threadIdx.x * per, s.n_seqs), i1 = min(i0 + per, s.n_seqs);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t sum = 0;
    for (int i = i0; i < i1; i++) {
        const WeightWork w = weight_work<RB>(s, p, a, i);
        cum[i] = sum;
        if (w.steps) sum = add_places(sum, (uint32_t)min((unsigned long long)0x7fffffff, (unsigned long long)p.n_kv * ((unsigned long long)w.steps * w.blocks + kUnitCost)));
    }
    uint32_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl = add_places(incl, v);
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    uint32_t before = __shfl_up_sync(0xffffffffu, incl, 1), total = 0;
    if (lane == 0) before = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        if (w < warp) before = add_places(before, warp_sums[w]);
        total = add_places(total, warp_sums[w]);
    }
    for (int i = i0; i < i1; i++) cum[i] = add_places(cum[i], before);
    if (threadIdx.x == 0) cum[s.n_seqs] = total;
    __syncthreads();
    return total;
}

template <int HD, int NG, bool F32, bool FULL>
__global__ void __launch_bounds__(kRunWarps * 32, WeightShape<HD, NG, F32>::kBlocks)
kv4_weights_kernel(Kv4Pool pool, Kv8Seqs seqs, WeightArgs a) {
    using Shape = WeightShape<HD, NG, F32>;
    constexpr int RB = Shape::kRows, S = Shape::kStages, TERMS = Shape::kTerms;
    constexpr int KS = HD / 16, KW = HD / 32;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t warp_sums[kRunWarps];
    uint32_t* cum = reinterpret_cast<uint32_t*>(smem + kRunWarps * Shape::kWarp);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (blockIdx.x == 0) weights_check_seqs(pool, seqs, a);
    const uint32_t total = weight_line<RB>(seqs, pool, a, cum, warp_sums);
    const Runs runs(total, gridDim.x * kRunWarps);
    const uint32_t run = blockIdx.x * kRunWarps + warp;
    if (run >= runs.n) return;
    uint32_t t = runs.start(run);
    const uint32_t t_end = runs.start(run + 1);
    unsigned char* const mine = smem + warp * Shape::kWarp;
    const uint32_t ring = smem_u32(mine);
    uint4* const qs = reinterpret_cast<uint4*>(mine + Shape::kRing);
    const int hd = FULL ? HD : pool.hd;
    using Ring = Ring4<HD, FULL, false, S>;

    while (t < t_end) {
        // a segment: this run's steps of one sequence and kv head.  A step is the run's that has its first place.
        const int seq = seq_at(cum, seqs.n_seqs, t);
        const WeightWork w = weight_work<RB>(seqs, pool, a, seq);
        const uint32_t places = (uint32_t)w.steps * w.blocks + kUnitCost, in_seq = t - cum[seq], kvh = in_seq / places, in = in_seq - kvh * places, end = min(places, in + (t_end - t));
        t += end - in;
        auto step_from = [&](uint32_t place) { return place <= (uint32_t)kUnitCost ? 0 : (int)((place - kUnitCost + w.blocks - 1) / w.blocks); };
        const int s0 = step_from(in), s1 = step_from(end);
        if (s1 <= s0) continue;
        const int32_t* table = seqs.table + (size_t)seq * seqs.width;
        float* const mass = a.mass + (int64_t)seq * a.mass_stride + (int64_t)kvh * a.mass_head_stride;
        const float head = kUnit4 * pool.k_scale[kvh];

        for (int rb = 0; rb < w.blocks; rb++) {
            const int row_lo = rb * RB, row_n = min(RB, w.n * a.group - row_lo);
            const int tok_first = row_lo / a.group, tok_last = (row_lo + row_n - 1) / a.group;
            // the block's steps: from its first row's window to its last row's slot
            const int b0 = max(s0, (a.window > 0 ? max(0, w.ctx + tok_first - a.window + 1) : 0) / kStep - w.step0), b1 = min(s1, (w.ctx + tok_last) / kStep + 1 - w.step0);
            if (b0 >= b1) continue;
            Ring keys(pool, hd, table, kvh, w.step0, ring, lane);
            bool bad = keys.begin(b0, b1);
#pragma unroll
            for (int k = 0; k < S - 1; k++) bad = keys.fetch(b0 + k, k == 0) || bad;

            // The queries as operand fragments.  A thread's dims are HD / 4 in a row, eight of which make two k steps: (0, 4), (1, 5) and (2, 6), (3, 7), as the keys' words give them.
            uint32_t qf[Shape::kQueriesShared ? 1 : TERMS * KS][2];
            float f[NG][2], less[NG][2];         // of rows 2c, 2c + 1 of a group: what scores are multiplied by, and lse, in powers of two
            int limit[NG][2];                    // last slot that the row sees (-1: no row, or one that adds nothing)
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                const int r = 8 * gr + g;
                const bool has = r < row_n;
                const int tok = has ? (row_lo + r) / a.group : 0, hq = has ? (row_lo + r) - tok * a.group : 0;
                const int64_t src = (int64_t)(w.first + tok) * a.q_stride + (int64_t)((int)kvh * a.group + hq) * hd;
                const float lse = has ? a.lse[(int64_t)(w.first + tok) * a.lse_stride + (int)kvh * a.group + hq] : 0.0f;
                float v[HD / 4], top = 0.0f, up, down;
#pragma unroll
                for (int j = 0; j < HD / 64; j++) {
                    const int d = c * (HD / 4) + 16 * j;
                    float* u = v + 16 * j;
                    if (has && (FULL || d < hd)) load16(a.q, src + d, a.typ, a.q_vec, u);
                    else
#pragma unroll
                        for (int e = 0; e < 16; e++) u[e] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) top = max_nan(top, fabsf(u[e]));
                }
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                row_scale(top, up, down);
                const float rf = score_factor(a.scale_log2, down, head);
                const int rl = has && fabsf(lse) < INFINITY && top < INFINITY ? w.ctx + tok : -1;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int from = 8 * c + 4 * x;  // a thread that has row 2c + x
                    f[gr][x] = __shfl_sync(0xffffffffu, rf, from);
                    less[gr][x] = __shfl_sync(0xffffffffu, lse * 1.44269504088896f, from);
                    limit[gr][x] = __shfl_sync(0xffffffffu, rl, from);
                }
                if (rl < 0) up = 0.0f;  // products of a row that adds nothing are 0, or NaN, and masked
#pragma unroll
                for (int k2 = 0; k2 < KS / 2; k2++) {  // eight dims: two k steps
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float p = v[8 * k2 + e] * up, q = v[8 * k2 + e + 4] * up;
                        if (F32) h2_split(p, q, hi[e], lo[e]);
                        else hi[e] = h2_pack(p, q);
                    }
                    if (Shape::kQueriesShared) {
                        qs[((gr * TERMS) * (KS / 2) + k2) * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if (F32) qs[((gr * TERMS + TERMS - 1) * (KS / 2) + k2) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int ks = 2 * k2 + (e >> 1);
                            qf[Shape::kQueriesShared ? 0 : ks][e & 1] = hi[e];
                            if (F32) qf[Shape::kQueriesShared ? 0 : (TERMS - 1) * KS + ks][e & 1] = lo[e];
                        }
                    }
                }
            }
            __syncwarp();

            const int sees = w.ctx + tok_first, from = a.window > 0 ? w.ctx + tok_last - a.window : -1;
            bool all_rows = true;  // every row of the block is there and counts
#pragma unroll
            for (int gr = 0; gr < NG; gr++) all_rows = all_rows && limit[gr][0] >= 0 && limit[gr][1] >= 0;
            all_rows = __all_sync(0xffffffffu, all_rows);
            const int plain0 = !all_rows ? b1 : from < 0 ? 0 : from / kStep + 1 - w.step0, plain1 = (sees + 1) / kStep - w.step0;   // steps whose keys all rows see
            for (int st = b0; st < b1; st++) {
                cp_async_wait<S - 2>();
                __syncwarp();
                bad = keys.fetch(st + S - 1) || bad;  // into the place of the step before
                if (keys.any_bad && keys.outside(st)) continue;
                const int key0 = (w.step0 + st) * kStep, key = key0 + g + 8 * (c & 1);
                const bool plain = st >= plain0 && st < plain1;
                // the sums' own threads: c = 0 has key g, c = 1 key g + 8
                const bool writes = c < 2 && key < w.ctx + w.n;
                float* const to = mass + key;
                const float before = writes ? *to : 0.0f;
                const unsigned char* kp = mine + (st & (S - 1)) * Ring::kPlace;
                uint32_t kf[KS][4];
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int row = 8 * half + g;
                    uint32_t kw[KW];
                    if (FULL) lds_words<KW>(kp + row * (HD / 2) + c * (HD / 8), kw);
                    else lds_words8<KW>(kp + row * (hd >> 1) + c * (HD / 8), kw);
                    const unsigned char* sc = kp + Ring::kScales + row * (hd >> 4) + c * (HD / 64);
                    uint32_t bytes = 0;
                    if (HD == 64) bytes = *sc;
                    else if (FULL) bytes = HD == 128 ? *reinterpret_cast<const uint16_t*>(sc) : *reinterpret_cast<const uint32_t*>(sc);
                    else
#pragma unroll
                        for (int j = 0; j < HD / 64; j++) bytes |= (uint32_t)sc[j] << (8 * j);
                    bytes &= 0x7f7f7f7fu;
#pragma unroll
                    for (int j = 0; j < HD / 64; j++) {
                        const Scale4 k4 = scale4_both(bytes, j);
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            uint32_t kv[4];
                            values8(kw[2 * j + x], k4, kv);
#pragma unroll
                            for (int e = 0; e < 4; e++) kf[4 * j + 2 * x + (e >> 1)][2 * (e & 1) + half] = kv[e];
                        }
                    }
                }
                float sum[2] = {0.0f, 0.0f};     // of keys g, g + 8
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    float dot[2][4];             // two halves of the dims: their products need not wait for one another
#pragma unroll
                    for (int term = TERMS - 1; term >= 0; term--)  // low parts first
#pragma unroll
                        for (int k2 = 0; k2 < KS / 2; k2++) {
                            uint4 b;
                            if (Shape::kQueriesShared) b = qs[((gr * TERMS + term) * (KS / 2) + k2) * 32 + lane];
                            else {
                                const int at = Shape::kQueriesShared ? 0 : term * KS + 2 * k2, at1 = Shape::kQueriesShared ? 0 : at + 1;
                                b = make_uint4(qf[at][0], qf[at][1], qf[at1][0], qf[at1][1]);
                            }
                            if (term == TERMS - 1 && k2 == 0) {
                                mma_f16_first(dot[0], kf[0], b.x, b.y);
                                mma_f16_first(dot[1], kf[1], b.z, b.w);
                            } else {
                                mma_f16(dot[0], kf[2 * k2], b.x, b.y);
                                mma_f16(dot[1], kf[2 * k2 + 1], b.z, b.w);
                            }
                        }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float y = fmaf(dot[0][e] + dot[1][e], f[gr][e & 1], -less[gr][e & 1]);
                        if (!plain) {
                            const int k = key0 + g + 8 * (e >> 1);
                            if (k > limit[gr][e & 1] || (a.window > 0 && k <= limit[gr][e & 1] - a.window)) y = kNegInf;
                        }
                        sum[e >> 1] += exp2_fast(y);
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
                    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
                }
                if (writes) *to = before + (c ? sum[1] : sum[0]);
            }
            cp_async_wait<0>();
            __syncwarp();
            if (bad && lane == 0) kv8_raise(seqs, seq);
        }
    }
}

template <int HD, int NG, bool F32, bool FULL>
int32_t weights_as(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s) {
    using Shape = WeightShape<HD, NG, F32>;
    const size_t smem = kRunWarps * Shape::kWarp + (size_t)(seqs.n_seqs + 1) * 4;
    LC_CUDA(ensure_smem_limit((const void*)kv4_weights_kernel<HD, NG, F32, FULL>, smem));
    kv4_weights_kernel<HD, NG, F32, FULL><<<sm_count() * Shape::kBlocks, kRunWarps * 32, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
template <int HD, int NG>
int32_t weights_full(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s) {
    if (a.typ == LC_TYPE_F32) return pool.hd == HD ? weights_as<HD, NG, true, true>(pool, seqs, a, s) : weights_as<HD, NG, true, false>(pool, seqs, a, s);
    return pool.hd == HD ? weights_as<HD, NG, false, true>(pool, seqs, a, s) : weights_as<HD, NG, false, false>(pool, seqs, a, s);
}
// Whether tiles are faster than runs, us in runs / in tiles, with so many stretches of 256 keys (as long as the tables are).  256 rows (tokens x heads of a group) of a sequence and kv head: always, bf16 41 / 17 with
// 72 stretches, 211 / 122 with 2,048, 686 / 528 with 8,192, f32 62 / 20, 328 / 218, 1,120 / 1,028 and 2,131 / 2,008 with 16,384.  128 rows: bf16 28 / 12 with 128, 114 / 99 with 2,048, 388 / 450 with 8,192; f32
// 108 / 73 with 1,024, 312 / 396 with 4,096.  64 rows: bf16 17 / 12 with 128, 39 / 42 with 1,024, 59 / 85 with 2,048; f32 23 / 14 and 56 / 68.  32 rows: bf16 12 / 12 and 21 / 41.
bool tiles_pay(const Kv4Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int64_t rows) {
    const int64_t stretches = (((int64_t)seqs.width << pool.page_shift) + 255) / 256 * seqs.n_seqs * pool.n_kv;
    const bool f32 = typ == LC_TYPE_F32;
    return pool.hd <= 128 && (rows >= 256 || (rows >= 128 && stretches <= (f32 ? 8 : 16) * sm_count()) || (rows >= 64 && stretches <= (f32 ? 2 : 7) * sm_count()));
}
// As many groups of 8 rows share a step's keys as a sequence and kv head has rows for, four at most.
template <int HD>
int32_t weights_of(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, int64_t rows, cudaStream_t s) {
    if (rows <= 8) return weights_full<HD, 1>(pool, seqs, a, s);
    if (rows <= 16) return weights_full<HD, 2>(pool, seqs, a, s);
    return weights_full<HD, 4>(pool, seqs, a, s);
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" int32_t lc_kv4_weights_dev(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, const void* q_dev, int64_t q_stride, int32_t n_heads, float scale, int32_t window,
                                      const float* lse_dev, int64_t lse_stride, float* mass_dev, int64_t mass_stride, int64_t mass_head_stride, int32_t capacity, void* stream_) {
    const char* call = "lc_kv4_weights_dev";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    LC_CHECK(window >= 0, LC_ERR_INVALID, "%s: window=%d", call, window);
    LC_CHECK(scale >= 0.0f && scale <= 2.0e38f, LC_ERR_INVALID, "%s: scale=%g", call, scale);
    LC_CHECK(capacity >= 0 && mass_head_stride >= capacity && mass_stride >= capacity, LC_ERR_INVALID, "%s: capacity=%d (the strides of the sums are %lld and %lld)", call, capacity,
             (long long)mass_stride, (long long)mass_head_stride);
    LC_CHECK(seqs.n_seqs <= 1 || pool.n_kv == 1 || mass_stride >= (int64_t)(pool.n_kv - 1) * mass_head_stride + capacity || mass_head_stride >= (int64_t)(seqs.n_seqs - 1) * mass_stride + capacity,
             LC_ERR_INVALID, "%s: the sums of sequences and heads overlap (strides %lld and %lld)", call, (long long)mass_stride, (long long)mass_head_stride);
    const int group = n_heads / pool.n_kv;
    // a sequence outside its table may have all rows: what a call's rows are in the kernels' 32 bits; and the places of the line
    LC_CHECK((int64_t)n_rows * group < (int64_t)0x7fffffff - 64 && line_fits(pool, seqs, group, 8), LC_ERR_INVALID, "%s: %d rows of %d heads over tables of %d pages are too many for one call", call, n_rows,
             n_heads, seqs.width);
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(q_dev && lse_dev && mass_dev, LC_ERR_INVALID, "%s: null queries, lse or sums", call);
    LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && lse_stride >= n_heads, LC_ERR_INVALID, "%s: rows overlap", call);
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    const size_t elem = typ == LC_TYPE_F32 ? 4 : 2;
    const WeightArgs a{q_dev, lse_dev, mass_dev, q_stride, lse_stride, mass_stride, mass_head_stride, (int)typ, group, std::min(window, 1 << 30), capacity, rows_aligned(q_dev, q_stride, elem, 16),
                       scale * 1.44269504088896f};
    cudaStream_t s = stream_or_own(stream_);
    const int64_t most = (int64_t)group * std::max(1, rows->max_rows);
    if (tiles_pay(pool, seqs, typ, most)) return launch_kv4_weights_tiles(pool, seqs, a, s);
    if (pool.hd <= 64) return weights_of<64>(pool, seqs, a, most, s);
    if (pool.hd <= 128) return weights_of<128>(pool, seqs, a, most, s);
    return weights_of<256>(pool, seqs, a, most, s);
}
