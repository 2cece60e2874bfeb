// Attention over the 8-bit key/value cache for many rows per sequence (prompts), on tcgen05.
//
// A block has a unit: 256 rows (tokens x heads of the group, so that grouped heads share a tile's keys) of a sequence and kv head, in two tiles of 128, which
// take turns on the matrix unit while the other's softmax runs.  It walks the keys in tiles of 128.
//   warps 0-3, 4-7   the softmax of row tile 0, 1: a row per thread, scores and sums in tensor memory;
//   warp 13          copies the next keys and values from the cache into shared memory (bulk copies of 16 keys);
//   warps 8-11, 14, 15   unpack them to f16 (K as [key][dim], V as [dim][key], 128-byte swizzle);
//   warp 12          one thread issues the products.  With the unpacking in the same warps an iteration took 9,500 cycles instead of 4,000: the issue waits
//                    for the matrix unit's queue.
// Scores: S = Q K^T, each row of queries times a power of two of its own; f32 queries as f16 high and low parts, two products.
// Weights: with f the score's factor (scale log2 e S_k over the row's power of two) and S_v of the key's page over a power of two (the first page's), P_j = 2^(s_j f_j + log2 S_v,j - M + 6), M the row's largest exponent so far: the
// value's scale is in the weight, so a page's scale costs an addition per 16 keys; the denominator is sum P_j / S_v,j, and the power of two multiplies what is written.  P goes back into the place of S, as f16
// (f32: high and low parts).  O = P V:
//   f32             a key tile's sums are added to the row's in registers: what the matrix unit cuts off when it adds stays within a tile of keys (2,048 keys in
//                   its own sums were off by 1e-5);
//   16-bit types    O stays in tensor memory for all keys (the same error is a hundredth of the outputs' rounding), and so that it rarely
//                   has to be scaled again, M is raised only when a row's largest exponent has grown by more than 8.
//
// What bounds it (a pair of row tiles x 128 keys, head dim 128): products 2,048 cycles (f32: 4,096), exponentials 2,048 on the special-function unit, and 320 KB through
// shared memory, 2,500 cycles (128 of queries and keys, 64 of values for the products, 128 of copies and unpacking); about 3,900 pass, as a row tile's softmax, its sums
// and its next scores wait for one another.  Steps of 64 keys, whose scores are under way while the 64 before are weighted, took 571 us instead of 412 (three chunks of 700 - 2,048 tokens behind 1,000 - 6,100, 32 heads over 8, bf16): products half
// as wide read the queries twice.
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv8_attn.cuh"
#include "lc_umma.cuh"

namespace lc {

namespace {

constexpr int kKeys = 128, kTileThreads = 512, kConvWarps = 6, kSlots = 4;
// registers a thread at the launch
constexpr int kLaunchRegs = 128;
constexpr int kGroups = kKeys / 16;

// what the softmax needs to know of 16 keys: their scale, log2 of the values' scale, its inverse; and what the unpacking does
enum : int { kHere = 0, kAbsent = 1, kOutside = 2, kZeroValues = 4 };  // not among the unit's keys: zeros; outside the pool: keys of NaN
struct GroupConst {
    float f, lv, inv;
    int state;
};
struct TileShared {
    uint64_t s_full[2], p_full[2], o_full[2];  // scores, weights, sums of a row tile
    uint64_t c_full[kSlots];                   // consts of a key tile
    uint64_t raw_full[2], raw_free[2];         // copied keys, values
    uint64_t k_full, v_full[2];                // unpacked keys, values (a barrier for each place: the next tile's values may be there before this one's are waited for);
    uint64_t v_free[2];                        // the keys' place is free when the last row tile's scores are done, the values' when its sums are
    GroupConst consts[kSlots][kGroups];
    uint2 sums[kTileThreads / 32];
    uint32_t tmem;
    float base;                                // what the values' scales of the unit are relative to
    uint8_t down[kTileRows2];                  // exponents of the factors that undo the rows' powers of two; 255: a row that is not finite
};

template <int HD, bool SPLIT> struct TileShape {
    static constexpr int kPart = HD * 256;                    // 128 rows of HD f16
    static constexpr int kQ = 2 * (SPLIT ? 2 : 1) * kPart;    // [row tile][high, low]
    static constexpr int kK = HD * 256, kV = HD * 256;
    static constexpr int kSoftRegs = SPLIT ? 176 : 184, kOtherRegs = 256 - kSoftRegs;  // of the softmax's 256 threads, of the other 256
    static_assert(256 * (kSoftRegs + kOtherRegs) <= kLaunchRegs * kTileThreads, "setmaxnreg waits for registers that the launch does not have");
    static constexpr int kVs = SPLIT ? 1 : 2;                 // places for unpacked values: f32 queries leave room for one
    static constexpr int kRaw = kKeys * HD;                   // keys, values as they are in the cache
    static constexpr int kBytes = kQ + kK + kVs * kV + 2 * kRaw + 1024;
};

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    tmem_ld16(taddr, r);
    tmem_ld16(taddr + 16, r + 16);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// products issued by the lane whose `by` is set, in a warp that goes through this together
__device__ __forceinline__ void mma_ss_by(uint32_t by, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(da), "l"(db),
                 "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
__device__ __forceinline__ void mma_ts_by(uint32_t by, uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(db),
                 "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
// 16-byte chunk `ch` (of 8) of a row of 128 bytes
__device__ __forceinline__ int sw128(int row, int ch) { return row * 128 + ((ch ^ (row & 7)) << 4); }

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kTileThreads, 1) kv8_tiles_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a, int splits) {
    using Shape = TileShape<HD, SPLIT>;
    constexpr int TERMS = SPLIT ? 2 : 1;
    extern __shared__ unsigned char raw_smem[];
    __shared__ TileShared sh;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);
    unsigned char* const sq = smem;
    unsigned char* const sk = sq + Shape::kQ;
    unsigned char* const sv = sk + Shape::kK;
    unsigned char* const raw[2] = {sv + Shape::kVs * Shape::kV, sv + Shape::kVs * Shape::kV + Shape::kRaw};
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (blockIdx.x == 0 && blockIdx.y == 0) kv8_check_seqs(seqs, pool);

    // the unit: sequences in order, the row blocks with most keys first
    uint32_t* units = reinterpret_cast<uint32_t*>(smem);
    uint32_t* cum = units + seqs.n_seqs + 1;
    line_up<kTileRows2>(seqs, pool, a, cum, units, sh.sums);
    if (blockIdx.x >= units[seqs.n_seqs]) return;
    const int seq = seq_at(units, seqs.n_seqs, blockIdx.x);
    const int in = blockIdx.x - units[seq];
    __syncthreads();  // the arrays' place is the queries'
    const SeqWork w = seq_work<kTileRows2>(seqs, pool, a, seq);
    const int kvh = in % pool.n_kv, rb = w.blocks - 1 - in / pool.n_kv;
    const int row_lo = rb * kTileRows2, row_n = min(kTileRows2, w.n * a.group - row_lo);
    const int n_tiles = row_n > 128 ? 2 : 1;
    const int hd = pool.hd;
    const int64_t head0 = (int64_t)kvh * a.group * hd;
    auto row_at = [&](int r, int64_t stride) {  // offset of the unit's row r
        const int tok = (row_lo + r) / a.group;
        return (int64_t)(w.first + tok) * stride + head0 + (int64_t)(row_lo + r - tok * a.group) * hd;
    };
    float* const part = a.part + (size_t)(blockIdx.x * gridDim.y + blockIdx.y) * (kTileRows2 * (HD + 2));
    if (!w.inside) {
        if (splits == 1) {
            for (int e = tid; e < row_n * hd; e += kTileThreads) store1(a.out, row_at(e / hd, a.out_stride) + e % hd, a.typ, __int_as_float(0x7fffffff));
        } else if (tid < kTileRows2) {
            part[tid] = 0.0f;
            part[kTileRows2 + tid] = __int_as_float(0x7fffffff);
            for (int d = 0; d < HD; d++) part[2 * kTileRows2 + tid * HD + d] = 0.0f;
        }
        return;
    }
    // keys: from the first row's window to the last row's position; this block's share of their tiles
    const int tok_first = row_lo / a.group, tok_last = (row_lo + row_n - 1) / a.group;
    const int key_lo = a.window > 0 ? max(0, w.ctx + tok_first - a.window + 1) : 0, key_end = w.ctx + tok_last + 1;
    const int tiles0 = key_lo / kKeys, all = (key_end + kKeys - 1) / kKeys - tiles0;
    const int i0 = (int)((long long)all * blockIdx.y / splits), n = (int)((long long)all * (blockIdx.y + 1) / splits) - i0;
    const int tile0 = tiles0 + i0;
    if (n == 0) {  // only where a unit is cut
        if (tid < kTileRows2) { part[tid] = kNegInf; part[kTileRows2 + tid] = 0.0f; }
        return;
    }

    if (tid == 0) {
        for (int t = 0; t < 2; t++) {
            mbar_init(&sh.s_full[t], 1);
            mbar_init(&sh.o_full[t], 1);
            mbar_init(&sh.v_free[t], 1);
            mbar_init(&sh.p_full[t], 128);
            mbar_init(&sh.raw_full[t], 1);
            mbar_init(&sh.raw_free[t], kConvWarps);
            mbar_init(&sh.v_full[t], kConvWarps);
        }
        mbar_init(&sh.k_full, kConvWarps);
        for (int t = 0; t < kSlots; t++) mbar_init(&sh.c_full[t], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
        sh.base = 1.0f;
    }
    if (warp == 0) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t col_s[2] = {tmem, tmem + 128}, col_o[2] = {tmem + 256, tmem + 384};

    // the queries as f16, each row times a power of two of its own: what a row gives does not depend on the others
    {
        constexpr int C = HD / 16;  // lanes of a row, neighbours in a warp
        const int chunks = n_tiles * 128 * C;
        for (int e = tid; e < chunks; e += kTileThreads) {
            const int r = e / C, ch = e % C;
            float v[16], top = 0.0f;
            if (r < row_n && ch * 16 < hd) load16(a.q, row_at(r, a.q_stride) + ch * 16, a.typ, a.q_vec, v);
            else
#pragma unroll
                for (int x = 0; x < 16; x++) v[x] = 0.0f;
#pragma unroll
            for (int x = 0; x < 16; x++) top = max_nan(top, fabsf(v[x]));
#pragma unroll
            for (int o = C / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            float up, down;
            row_scale(top, up, down);
            if (ch == 0) sh.down[r] = top < INFINITY ? (uint8_t)(__float_as_uint(down) >> 23) : 255;
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
                if (SPLIT) h2_split(v[2 * x] * up, v[2 * x + 1] * up, hi[x], lo[x]);
                else hi[x] = h2_pack(v[2 * x] * up, v[2 * x + 1] * up);
            }
            unsigned char* dst = sq + (r >> 7) * TERMS * Shape::kPart + (ch >> 2) * (128 * 128);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int at = sw128(r & 127, 2 * (ch & 3) + x);
                *reinterpret_cast<uint4*>(dst + at) = make_uint4(hi[4 * x], hi[4 * x + 1], hi[4 * x + 2], hi[4 * x + 3]);
                if (SPLIT) *reinterpret_cast<uint4*>(dst + Shape::kPart + at) = make_uint4(lo[4 * x], lo[4 * x + 1], lo[4 * x + 2], lo[4 * x + 3]);
            }
        }
    }
    fence_async();
    __syncthreads();

    const int last = n_tiles - 1;
    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kOtherRegs));
      if (warp == 12 || warp == 13) {
        if (warp == 12) {
            // ------------------------------------------------------------------------------------------------ products
            // All lanes go the same way and one of them issues: descriptors then are the warp's and not a thread's (2,048-token prompt in f32 127 -> 119 us).
            const uint32_t q_at = smem_u32(sq), k_at = smem_u32(sk), v_at = smem_u32(sv), base = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t one = lane == 0;
            auto scores = [&](int t) {
                const uint32_t d = base + 128 * t;
#pragma unroll
                for (int term = TERMS - 1; term >= 0; term--) {  // the low parts first: what is cut off then is small
                    const uint64_t dq = umma_desc_sw128(q_at + (t * TERMS + term) * Shape::kPart), dk = umma_desc_sw128(k_at);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ks++) {
                        const uint64_t off = ((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4;
                        mma_ss_by(one, d, dq + off, dk + off, idesc_f16(kKeys), term < TERMS - 1 || ks > 0);
                    }
                }
                if (one) umma_commit(&sh.s_full[t]);
                __syncwarp();
            };
            auto sums = [&](int t, int i) {
                const uint32_t d = base + 256 + 128 * t, p = base + 128 * t;
                const uint64_t dv = umma_desc_sw128(v_at + (i % Shape::kVs) * Shape::kV);
                const uint32_t on = !SPLIT && i > 0;
#pragma unroll
                for (int term = TERMS - 1; term >= 0; term--)
#pragma unroll
                    for (int ks = 0; ks < kKeys / 16; ks++)
                        mma_ts_by(one, d, p + 16 * ks + 8 * term, dv + (((ks >> 2) * (HD * 128) + (ks & 3) * 32) >> 4), idesc_f16(HD), term < TERMS - 1 || ks > 0 ? 1u : on);
                if (one) {
                    umma_commit(&sh.o_full[t]);
                    if (t == last) umma_commit(&sh.v_free[i % Shape::kVs]);
                }
                __syncwarp();
            };
            bool ok = __all_sync(0xffffffffu, mbar_wait(&sh.k_full, 0));
            tc_fence_after();
            for (int t = 0; t < n_tiles && ok; t++) scores(t);
            for (int i = 0; i < n && ok; i++) {
                const bool more = i + 1 < n;
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.v_full[i % Shape::kVs], (i / Shape::kVs) & 1));
                for (int t = 0; t < n_tiles && ok; t++) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.p_full[t], i & 1));
                    tc_fence_after();
                    if (!ok) break;
                    sums(t, i);
                    if (more) {
                        if (t == 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.k_full, (i + 1) & 1));
                        if (!ok) break;
                        tc_fence_after();
                        scores(t);
                    }
                }
            }
        } else {
            // -------------------------------------------------------------------------------------------------- copies
            const int32_t* table = seqs.table + (size_t)seq * seqs.width;
            const int page_mask = (1 << pool.page_shift) - 1;
            const uint32_t bytes = 16 * hd;
            auto page_of = [&](int i, int group) {  // -1 in front of every row's window and behind the end, -2 outside the pool
                const int key = (tile0 + i) * kKeys + group * 16;
                if (i >= n || key + 15 < key_lo || key >= key_end) return -1;
                const int p = table[key >> pool.page_shift];
                return p >= 0 && p < pool.n_pages ? p : -2;
            };
            auto look_up = [&](int i) { return lane < kGroups ? page_of(i, lane) : -1; };  // lane g < 8: the page of group g
            // log2 of a scale of values over `base`, which is the first that is not 0, as a power of two between 2^-56 and 2^56; minus infinity for pages that count as zeros: 2^-90 of it
            // and less.  All lanes take part; `low` is the smallest so far.
            float base = 0.0f, to_base = 1.0f, low = INFINITY;
            auto log_scale = [&](float vsc) {
                const uint32_t which = __ballot_sync(0xffffffffu, vsc != 0.0f);
                if (base == 0.0f && which) {
                    const uint32_t e = (__float_as_uint(__shfl_sync(0xffffffffu, vsc, __ffs(which) - 1)) >> 23) & 0xff;
                    const uint32_t at = min(max(e, 127u - 56u), 127u + 56u);
                    base = __uint_as_float(at << 23);
                    to_base = __uint_as_float((254u - at) << 23);
                    if (lane == 0) sh.base = base;
                }
                float lv = vsc != 0.0f ? log2f(vsc * to_base) : kNegInf;
                if (lv < -90.0f) lv = kNegInf;
                float least = lv == kNegInf ? INFINITY : lv;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
                low = fminf(low, least);
                return lv;
            };
            int page = look_up(0);
            bool ok = true;
            for (int i = 0; i < n && ok; i++) {
                const int next = look_up(i + 1);
                const size_t ph = (size_t)(page < 0 ? 0 : page) * pool.n_kv + kvh;
                const size_t off = ((ph << pool.page_shift) + (((tile0 + i) * kKeys + lane * 16) & page_mask)) * hd;
                const float ksc = page >= 0 ? pool.k_scale[ph] : 1.0f, vsc = page >= 0 ? pool.v_scale[ph] : 0.0f;
                const uint32_t all = bytes * __popc(__ballot_sync(0xffffffffu, page >= 0));
                for (int x = 0; x < 2; x++) {
                    if (i > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.raw_free[x], (i - 1) & 1));
                    if (!ok) break;
                    if (x == 0) {
                        float lv = log_scale(vsc);
                        const bool counts = lv != kNegInf;
                        // A page of zeros counts in the denominator alone: its weights take the smallest scale so far (where there is none, that of the first pages that have one), so that
                        // they do not lift the reference above what the other pages' weights need, and its values are zeros.
                        if (i == 0 && low == INFINITY)
                            for (int k = 1; k < n && low == INFINITY; k += 4) {
                                const int p = page_of(k + (lane >> 3), lane & 7);
                                (void)log_scale(p >= 0 ? pool.v_scale[(size_t)p * pool.n_kv + kvh] : 0.0f);
                            }
                        if (!counts) lv = low == INFINITY ? 0.0f : low;
                        if (lane < kGroups) {
                            GroupConst g;
                            g.f = page < 0 ? 1.0f : ksc;
                            g.lv = lv;
                            g.inv = exp2f(-lv);
                            g.state = page == -1 ? kAbsent : page == -2 ? kOutside : counts ? kHere : kZeroValues;
                            sh.consts[i % kSlots][lane] = g;
                            if (page == -2) kv8_raise(seqs, seq);
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.c_full[i % kSlots]);
                    }
                    if (lane == 0) mbar_expect_tx(&sh.raw_full[x], all);
                    __syncwarp();
                    if (page >= 0) bulk_load(raw[x] + lane * bytes, (x ? pool.v : pool.k) + off, bytes, &sh.raw_full[x]);
                }
                page = next;
            }
            if (!ok)  // whatever is under way lands before the block ends
                for (int x = 0; x < 2; x++) (void)mbar_wait(&sh.raw_full[x], 0), (void)mbar_wait(&sh.raw_full[x], 1);
        }
      } else {
        // ---------------------------------------------------------------------------------------------------- unpacking
        const int cw = warp < 12 ? warp - 8 : warp - 10, ct = cw * 32 + lane;
        constexpr int KC = HD / 16, LPK = HD / 4, OPW = 32 / LPK;     // K: pieces of a key; V: lanes of a key, octets of keys that a warp has at a time
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            const GroupConst* gc = sh.consts[i % kSlots];
            ok = mbar_wait(&sh.c_full[i % kSlots], (i / kSlots) & 1) && mbar_wait(&sh.raw_full[0], i & 1);
            if (i > 0) ok = ok && mbar_wait(&sh.s_full[last], (i - 1) & 1);  // the keys' place is free
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
#pragma unroll 2
            for (int e = ct; e < kKeys * KC; e += 32 * kConvWarps) {
                const int key = e / KC, ch = e % KC, state = gc[key >> 4].state;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (!(state & (kAbsent | kOutside)) && ch * 16 < hd) x = *reinterpret_cast<const uint4*>(raw[0] + key * hd + ch * 16);
                x.x ^= 0x80808080u; x.y ^= 0x80808080u; x.z ^= 0x80808080u; x.w ^= 0x80808080u;
                unsigned char* dst = sk + (ch >> 2) * (128 * 128);
                uint4 first = make_uint4(ints01(x.x), ints23(x.x), ints01(x.y), ints23(x.y));
                uint4 second = make_uint4(ints01(x.z), ints23(x.z), ints01(x.w), ints23(x.w));
                if (state == kOutside) first = second = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);  // NaN
                // the upper half of a row's chunks writes its second piece first: eight lanes then meet all banks
                const bool swap = ch >= 4;
                *reinterpret_cast<uint4*>(dst + sw128(key, 2 * (ch & 3) + (swap ? 1 : 0))) = swap ? second : first;
                *reinterpret_cast<uint4*>(dst + sw128(key, 2 * (ch & 3) + (swap ? 0 : 1))) = swap ? first : second;
            }
            fence_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&sh.k_full); mbar_arrive(&sh.raw_free[0]); }

            ok = mbar_wait(&sh.raw_full[1], i & 1);
            if (i >= Shape::kVs) ok = ok && mbar_wait(&sh.v_free[i % Shape::kVs], (i / Shape::kVs - 1) & 1);  // the values' place is free
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            unsigned char* const to = sv + (i % Shape::kVs) * Shape::kV;
#pragma unroll 1
            for (int u = cw; u < 16 / OPW; u += kConvWarps) {
                const int octet = u * OPW + lane / LPK, d = (lane % LPK) * 4;
                const bool none = gc[octet >> 1].state != kHere || d >= hd;
                uint32_t x[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[k] = none ? 0u : *reinterpret_cast<const uint32_t*>(raw[1] + (octet * 8 + k) * hd + d);
                    x[k] ^= 0x80808080u;
                }
                uint32_t pairs01[4], pairs23[4];  // (keys 2k, 2k + 1) of dims 0, 1 and 2, 3
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    pairs01[k] = __byte_perm(x[2 * k], x[2 * k + 1], 0x5140);
                    pairs23[k] = __byte_perm(x[2 * k], x[2 * k + 1], 0x7362);
                }
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const uint32_t* p = b < 2 ? pairs01 : pairs23;
                    uint4 out;
                    out.x = b & 1 ? ints23(p[0]) : ints01(p[0]);
                    out.y = b & 1 ? ints23(p[1]) : ints01(p[1]);
                    out.z = b & 1 ? ints23(p[2]) : ints01(p[2]);
                    out.w = b & 1 ? ints23(p[3]) : ints01(p[3]);
                    // row b LPK + l holds dim 4 l + b: eight lanes write eight rows
                    *reinterpret_cast<uint4*>(to + (octet >> 3) * (HD * 128) + sw128(b * LPK + lane % LPK, octet & 7)) = out;
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&sh.v_full[i % Shape::kVs]); mbar_arrive(&sh.raw_free[1]); }
        }
      }
    } else {
        // ------------------------------------------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kSoftRegs));
        const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_s = col_s[t] + lanes, my_o = col_o[t] + lanes;
        const int limit = w.ctx + (row_lo + min(r, row_n - 1)) / a.group;      // last position that the row sees
        const int least = __shfl_sync(0xffffffffu, limit, 0), most = __shfl_sync(0xffffffffu, limit, 31);
        // The row's part of a score's factor; the page's is its keys' scale.  A factor of 0 as 2^-100, so that a masked score of minus infinity stays one (what it
        // stands for is below 2^-69: a sum of products is below 2^31).  NaN for a row that is not finite, whose scores may all be minus infinity, as masked ones are.
        const float row_f = sh.down[r] == 255 ? __int_as_float(0x7fffffff) : a.scale_log2 * __uint_as_float((uint32_t)sh.down[r] << 23);
        auto factor = [&](float f) { return max_nan(f * row_f, 0x1p-100f); };
        float o[HD], m = kNegInf, l = 0.0f, corr = 1.0f;
        bool ok = true, far = false;
        // Rounded as the scores of a far reference are (below), so that the largest of these is no more than a rounding of S_v from it.
        auto exponent = [](float x, float f, float lv) { return __fadd_rn(__fmul_rn(x, f), lv); };
        // Far from 0 a reference has no bits left for what is added to it, and a product that is rounded with it may be off by more than f16's range
        // (scores of 1e8: 2^4).  There a score is rounded by itself, as the reference was, and what remains over it goes on; without loss in a neighbourhood of the reference.
        auto is_far = [](float mx) { return fabsf(mx) > 65536.0f && mx != kNegInf; };
        auto over = [](float x, float f, float ref, float lv) {
            const float y = __fsub_rn(__fmul_rn(x, f), ref);
            return y > 9.0f - lv ? 9.0f - lv : y;  // 2^15 at most; NaN stays
        };
        auto add_up = [&](int i) {  // o = o corr + the key tile's sums
            ok = mbar_wait(&sh.o_full[t], i & 1) && ok;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD; c += 16) {
                uint32_t x[16];
                tmem_ld16(my_o + c, x);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e++) o[c + e] = fmaf(o[c + e], corr, __uint_as_float(x[e]));
            }
        };
        if (t < n_tiles) {
            if (SPLIT)
#pragma unroll
                for (int d = 0; d < HD; d++) o[d] = 0.0f;
            for (int i = 0; i < n && ok; i++) {
                if (SPLIT && i > 0) add_up(i - 1);
                ok = mbar_wait(&sh.c_full[i % kSlots], (i / kSlots) & 1) && mbar_wait(&sh.s_full[t], i & 1) && ok;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const GroupConst* gc = sh.consts[i % kSlots];
                const int key0 = (tile0 + i) * kKeys;
                const bool plain = key0 + kKeys - 1 <= least && (a.window == 0 || key0 > most - a.window);
                // places of the tile that the row sees: [from, to]
                const int to = limit - key0, from = a.window > 0 ? limit - a.window + 1 - key0 : 0;
                float mx = m, sum = 0.0f;
                if constexpr (SPLIT) {
#pragma unroll 1
                    for (int c = 0; c < kKeys; c += 32) {
                        uint32_t x[32];
                        tmem_ld32(my_s + c, x);
                        tmem_wait_ld();
                        if (!plain)
#pragma unroll
                            for (int e = 0; e < 32; e++)
                                if (c + e > to || c + e < from) x[e] = __float_as_uint(kNegInf);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float g = __uint_as_float(x[16 * h]);
#pragma unroll
                            for (int e = 1; e < 16; e++) g = fmaxf(g, __uint_as_float(x[16 * h + e]));
                            const GroupConst k = gc[c / 16 + h];
                            mx = fmaxf(mx, exponent(g, factor(k.f), k.lv));
                        }
                    }
                    const float ref = mx == kNegInf ? 0.0f : mx;
                    far = is_far(mx);
                    const bool any_far = __any_sync(0xffffffffu, far);
                    const float less = far ? 6.0f : 6.0f - ref;
                    corr = exp2_fast(m - ref);
                    m = mx;
                    // 16 keys' weights take the first 8 columns of their scores' 16, their low parts the other 8
#pragma unroll 2
                    for (int c = 0; c < kKeys; c += 16) {
                        uint32_t x[16], p[8], q[8];
                        tmem_ld16(my_s + c, x);
                        tmem_wait_ld();
                        const GroupConst k = gc[c / 16];
                        const float off = k.lv + less, f = far ? 1.0f : factor(k.f);
                        if (!plain)
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                if (c + e > to || c + e < from) x[e] = __float_as_uint(kNegInf);
                        if (any_far)
#pragma unroll
                            for (int e = 0; e < 16; e++) x[e] = far ? __float_as_uint(over(__uint_as_float(x[e]), factor(k.f), ref, k.lv)) : x[e];
                        const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
                        float2 gs = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, off2), v = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            gs = add2(gs, v);
                            h2_split(v.x, v.y, p[e / 2], q[e / 2]);
                        }
                        sum = fmaf(gs.x + gs.y, k.inv, sum);
                        tmem_st8(my_s + c, p);
                        tmem_st8(my_s + c + 8, q);
                    }
                    l = fmaf(l, corr, sum);
                } else {
                    uint32_t x[kKeys];
#pragma unroll
                    for (int c = 0; c < kKeys; c += 16) tmem_ld16(my_s + c, x + c);
                    tmem_wait_ld();
                    if (!plain)
#pragma unroll
                        for (int e = 0; e < kKeys; e++)
                            if (e > to || e < from) x[e] = __float_as_uint(kNegInf);
#pragma unroll
                    for (int c = 0; c < kKeys; c += 16) {
                        float g = __uint_as_float(x[c]);
#pragma unroll
                        for (int e = 1; e < 16; e++) g = fmaxf(g, __uint_as_float(x[c + e]));
                        const GroupConst k = gc[c / 16];
                        mx = fmaxf(mx, exponent(g, factor(k.f), k.lv));
                    }
                    const bool raise = mx > m + 8.0f;  // also from minus infinity
                    if (__any_sync(0xffffffffu, raise)) {
                        const float f = raise ? exp2_fast(m - mx) : 1.0f;
                        if (raise) m = mx;
                        far = is_far(m);
                        l *= f;
                        if (i > 0) {
                            ok = mbar_wait(&sh.o_full[t], (i - 1) & 1);
                            ok = __all_sync(0xffffffffu, ok);
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < HD; c += 16) {
                                uint32_t y[16];
                                tmem_ld16(my_o + c, y);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
                                tmem_st16(my_o + c, y);
                            }
                        }
                    }
                    const float ref = m == kNegInf ? 0.0f : m;
                    const float less = far ? 6.0f : 6.0f - ref;
                    if (__any_sync(0xffffffffu, far))
#pragma unroll
                        for (int c = 0; c < kKeys; c += 16) {
                            const GroupConst k = gc[c / 16];
#pragma unroll
                            for (int e = 0; e < 16; e++) x[c + e] = far ? __float_as_uint(over(__uint_as_float(x[c + e]), factor(k.f), ref, k.lv)) : x[c + e];
                        }
#pragma unroll
                    for (int c = 0; c < kKeys; c += 16) {
                        uint32_t p[8];
                        const GroupConst k = gc[c / 16];
                        const float off = k.lv + less, f = far ? 1.0f : factor(k.f);
                        const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
                        float2 gs = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(__uint_as_float(x[c + e]), __uint_as_float(x[c + e + 1])), f2, off2), v = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            gs = add2(gs, v);
                            p[e / 2] = h2_pack(v.x, v.y);
                        }
                        sum = fmaf(gs.x + gs.y, k.inv, sum);
                        tmem_st8(my_s + c, p);
                    }
                    l += sum;
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sh.p_full[t]);
            }
            if constexpr (!SPLIT) {
#pragma unroll
                for (int d = 0; d < HD; d++) o[d] = 0.0f;
            }
            if (ok) add_up(n - 1);
            if (!ok || isnan(l)) l = __int_as_float(0x7fffffff);
            if (!ok && lane == 0) kv8_raise(seqs, seq);
            const float base = sh.base;  // behind the last tile's consts
            if (r < row_n) {
                if (splits == 1) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t dst = row_at(r, a.out_stride);
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = o[((d + e) >> 2) + ((d + e) & 3) * (HD / 4)] * inv * base;
                        if (d < hd) store16(a.out, dst + d, a.typ, a.out_vec, v);
                    }
                } else {
                    part[r] = m;
                    part[kTileRows2 + r] = l;
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = o[((d + e) >> 2) + ((d + e) & 3) * (HD / 4)] * base;
                        store16(part + 2 * kTileRows2 + (size_t)r * HD + d, true, v);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_free(tmem, 512);
}

// Joins the parts of units whose keys are cut: a warp per row.
template <int HD>
__global__ void __launch_bounds__(256) kv8_tiles_join_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a, int splits) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint2 sums[8];
    uint32_t* units = reinterpret_cast<uint32_t*>(smem);
    uint32_t* cum = units + seqs.n_seqs + 1;
    line_up<kTileRows2>(seqs, pool, a, cum, units, sums);
    pdl_wait();
    if (blockIdx.x >= units[seqs.n_seqs]) return;
    const int seq = seq_at(units, seqs.n_seqs, blockIdx.x), in = blockIdx.x - units[seq];
    const SeqWork w = seq_work<kTileRows2>(seqs, pool, a, seq);
    const int kvh = in % pool.n_kv, row_lo = (w.blocks - 1 - in / pool.n_kv) * kTileRows2, row_n = min(kTileRows2, w.n * a.group - row_lo);
    const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= row_n) return;
    constexpr int PER = HD / 32;
    float mx = kNegInf, sum = 0.0f, v[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) v[e] = 0.0f;
    for (int s = 0; s < splits; s++) {
        const float* p = a.part + (size_t)(blockIdx.x * splits + s) * (kTileRows2 * (HD + 2));
        const float pm = p[r], ps = p[kTileRows2 + r];
        if (pm == kNegInf && ps == 0.0f) continue;      // no keys: its sums are not there
        const float m2 = fmaxf(mx, pm), ref = m2 == kNegInf ? 0.0f : m2;
        const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(pm - ref);
        sum = f0 * sum + (isnan(ps) ? ps : f1 * ps);
#pragma unroll
        for (int e = 0; e < PER; e++) v[e] = fmaf(f0, v[e], f1 * p[2 * kTileRows2 + (size_t)r * HD + lane * PER + e]);
        mx = m2;
    }
    const int tok = (row_lo + r) / a.group;
    const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + ((int64_t)kvh * a.group + (row_lo + r - tok * a.group)) * pool.hd;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (lane * PER + e < pool.hd) store1(a.out, dst + lane * PER + e, a.typ, v[e] * inv);
}

template <int HD, bool SPLIT>
int32_t tiles_as(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const TilePlan& plan, cudaStream_t s) {
    using Shape = TileShape<HD, SPLIT>;
    const void* kern = (const void*)kv8_tiles_kernel<HD, SPLIT>;
    const size_t smem = std::max<size_t>(Shape::kBytes, (size_t)2 * (seqs.n_seqs + 1) * 4 + 1024);
    LC_CUDA(ensure_smem_limit(kern, smem));
    static const int regs = [&] {  // setmaxnreg counts on the launch's registers: a build that has fewer must not start it
        cudaFuncAttributes at;
        return cudaFuncGetAttributes(&at, kern) == cudaSuccess ? at.numRegs : 0;
    }();
    LC_CHECK(regs == kLaunchRegs, LC_ERR_UNSUPPORTED, "attention in tiles was built with %d registers a thread instead of %d", regs, kLaunchRegs);
    kv8_tiles_kernel<HD, SPLIT><<<dim3((unsigned)plan.units, (unsigned)plan.splits), kTileThreads, smem, s>>>(pool, seqs, a, plan.splits);
    LC_CUDA(cudaGetLastError());
    if (plan.splits > 1) {
        const size_t cum = (size_t)2 * (seqs.n_seqs + 1) * 4;
        LC_CUDA(launch_pdl(kv8_tiles_join_kernel<HD>, dim3((unsigned)plan.units, kTileRows2 / 8), dim3(256), cum, s, pool, seqs, a, plan.splits));
    }
    return LC_OK;
}

constexpr int kLeastRows = 32;  // of a sequence and kv head, below which no call goes by tiles
int64_t table_tiles(const Kv8Pool& pool, const Kv8Seqs& seqs) { return (((int64_t)seqs.width << pool.page_shift) + kKeys - 1) / kKeys; }  // of a sequence's keys, at most
size_t part_bytes(const Kv8Pool& pool) { return (size_t)kTileRows2 * ((pool.hd <= 64 ? 64 : 128) + 2) * sizeof(float); }

}  // namespace

bool kv8_tiles_plan(const Kv8Pool& pool, const Kv8Seqs& seqs, int group, TilePlan* plan) {
    const int64_t units = ((int64_t)seqs.n_rows * group / kTileRows2 + seqs.n_seqs) * pool.n_kv;
    if (pool.hd > 128 || units < 1 || units > 1 << 20) return false;
    // fewer units than SMs: their keys are cut, into parts of at least four tiles where contexts are as long as the table
    plan->units = (int)units;
    plan->splits = (int)std::max<int64_t>(1, std::min<int64_t>({sm_count() / units, (table_tiles(pool, seqs) + 3) / 4, 64}));
    plan->bytes = plan->splits > 1 ? (size_t)units * plan->splits * part_bytes(pool) : 16;
    return true;
}
bool kv8_tiles_pay(const Kv8Pool& pool, const Kv8Seqs& seqs, uint32_t typ, int group, int max_rows, const TilePlan& plan) {
    const int64_t rows = (int64_t)group * max_rows;
    // Runs or tiles, us in runs / in tiles (32 heads over 8 kv heads of 128 unless said).  16-bit types: one sequence behind 4,000 tokens with 8 rows (tokens x heads of a
    // group) 22.7 / 24.1, 32 rows 35 / 25, 256 rows 44 / 36; 16 sequences of 32 rows behind 2,000 43.6 / 47.7, 64 of 64 rows behind 1,000 116.5 / 119, of 128 rows (4 kv heads of
    // 64) 86 / 50.  f32: one of 64 rows 39.5 / 34, of 512 78 / 58, with one kv head of 512 rows 39 / 47; 64 sequences of 64 rows 154 / 176, of 128 rows 94 / 73.
    if (typ == LC_TYPE_F32) return plan.units >= 16 && rows >= (plan.units > sm_count() ? 128 : 64);
    return rows >= (seqs.n_seqs * pool.n_kv * table_tiles(pool, seqs) <= 4 * sm_count() ? kLeastRows : 64);  // fewer rows waste a tile: they only may where there is little to do
}
size_t kv8_tiles_most_bytes(const Kv8Pool& pool, int64_t rows) {
    // parts are no more than SMs
    return pool.hd <= 128 && rows >= kLeastRows ? sm_count() * part_bytes(pool) : 16;
}

int32_t launch_kv8_tiles(const Kv8Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const TilePlan& plan, cudaStream_t s) {
    if (pool.hd <= 64) return a.typ == LC_TYPE_F32 ? tiles_as<64, true>(pool, seqs, a, plan, s) : tiles_as<64, false>(pool, seqs, a, plan, s);
    return a.typ == LC_TYPE_F32 ? tiles_as<128, true>(pool, seqs, a, plan, s) : tiles_as<128, false>(pool, seqs, a, plan, s);
}

}  // namespace lc
