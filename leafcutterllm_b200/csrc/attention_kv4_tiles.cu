// Attention over the 4-bit key/value cache for many rows per sequence (prompts), on tcgen05.
//
// A block has a unit: 256 rows (tokens x heads of the group, so that grouped heads share a tile's keys) of a sequence and kv head, in two tiles of 128, which
// take turns on the matrix unit while the other's softmax runs.  It walks the keys in tiles of 128.
//   warps 0-3, 4-7   the softmax of row tile 0, 1: a row per thread, scores and sums in tensor memory;
//   warp 13          copies the next keys and values with their scales from the cache into shared memory (bulk copies of 16 keys);
//   warps 8-11, 14, 15   make f16 values of them (K as [key][dim], V as [dim][key], 128-byte swizzle), exactly;
//   warp 12          one thread issues the products.
// Scores: S = Q K^T, each row of queries times a power of two of its own; f32 queries as f16 high and low parts, two products.
// Weights: P_j = 2^(s_j f - M + 6), f the scale times log2 e over the row's power of two, M the row's largest exponent so far; P goes back into the place of S, as f16 (f32: high and low parts).
// O = P V:
//   f32             a key tile's sums are added to the row's in registers: what the matrix unit cuts off when it adds stays within a tile of keys;
//   16-bit types    O stays in tensor memory for all keys (that error is a hundredth of the outputs' rounding), and so that it rarely
//                   has to be scaled again, M is raised only when a row's largest exponent has grown by more than 8.
// Every byte of the cache is a finite number, so keys that no row sees may be anything: their weights are 0.
//
// Three sequences of 700 to 2,048 rows behind 1,000 to 6,100 slots, 32 heads over 8 of 128 in bf16: 366 us, 315 GFLOP at 860 TFLOP/s (192 us at the rate of library products).  What bounds it, for 256 rows x 128 keys in 4,440
// cycles: the unpacking warps work 3,600 of them; a row tile's softmax is 2,200 of its chain; issuing 32 products is 2,190 (68 each with their commits; the matrix unit runs one in 62), which waits 800 for keys and 1,080 for weights.
// An issue of 50 cycles a product matters (one elected lane, descriptors of 32 changing bits: 105 to 155 before, 410 us), as do two places for keys and work of unpacking that is even over its warps (379).
// Weights of 11 bits for 16-bit types: as in attention_kv4.cu, where the reason stands.
#include <algorithm>
#include "lc_attn_tiles.cuh"
#include "lc_kernels.h"
#include "lc_kv4.cuh"

namespace lc {

namespace {

constexpr int kKeys = 128, kTileThreads = 512, kConvWarps = 6, kSlots = 4;
// registers a thread at the launch
constexpr int kLaunchRegs = 128;
constexpr int kGroups = kKeys / 16;
constexpr float kTileUp = 6.0f;   // weights are 2^this too large, and up to 2^8 more before the reference is raised: 2^14 at most

struct TileShared {
    uint64_t s_full[2], p_full[2], o_full[2];  // scores, weights, sums of a row tile
    uint64_t c_full[kSlots];                   // `outside` of a key tile
    uint64_t raw_full[2][2], raw_free[2][2];   // copied keys, values, of a place
    uint64_t k_full[2], v_full[2];             // unpacked keys, values (a barrier for each place: the next tile's may be there before this one's are waited for);
    uint64_t k_free[2], v_free[2];             // a place of keys is free when the last row tile's scores are done, one of values when its sums are
    uint2 sums[kTileThreads / 32];
    uint32_t outside[kSlots];                  // bit g: the key tile's group g of 16 lies on a page outside the pool
    uint32_t tmem;
    uint8_t down[kTileRows2];                  // exponents of the factors that undo the rows' powers of two; 255: a row that is not finite
};

template <int HD, bool SPLIT> struct TileShape {
    static constexpr int kPart = HD * 256;                    // 128 rows of HD f16
    static constexpr int kQ = 2 * (SPLIT ? 2 : 1) * kPart;    // [row tile][high, low]
    static constexpr int kK = HD * 256, kV = HD * 256;
    static constexpr int kSoftRegs = SPLIT ? 176 : 184, kOtherRegs = 256 - kSoftRegs;  // of the softmax's 256 threads, of the other 256
    static_assert(256 * (kSoftRegs + kOtherRegs) <= kLaunchRegs * kTileThreads, "setmaxnreg waits for registers that the launch does not have");
    static constexpr int kVs = SPLIT ? 1 : 2;                 // places for unpacked keys, values: f32 queries leave room for one
    static constexpr int kRawKs = SPLIT ? 1 : 2, kRawVs = 1;  // and for copied ones: two of values would not fit
    static constexpr int kRawHalf = kKeys * HD / 2 + kKeys * HD / 16;  // integers and scales of a tile's keys or values
    static constexpr int kBytes = kQ + kVs * (kK + kV) + (kRawKs + kRawVs) * kRawHalf + 1024;
    static_assert(kBytes + 1024 <= 227 * 1024, "shared memory of a block");
    // A slot of `outside` is written again when the values of the key tile before have been copied, whose place the unpacking of those kRawVs tiles earlier left; these wait for the sums of kVs tiles earlier,
    // and sums for the softmax that has read its slot.
    static_assert(kSlots >= 1 + kRawVs + kVs, "a slot that the softmax may still read");
};

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kTileThreads, 1) kv4_tiles_kernel(Kv4Pool pool, Kv8Seqs seqs, AttnArgs a, int splits) {
    using Shape = TileShape<HD, SPLIT>;
    constexpr int TERMS = SPLIT ? 2 : 1, RK = Shape::kRawKs, RV = Shape::kRawVs;
    extern __shared__ unsigned char raw_smem[];
    __shared__ TileShared sh;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);
    unsigned char* const sq = smem;
    unsigned char* const sk = sq + Shape::kQ;
    unsigned char* const sv = sk + Shape::kVs * Shape::kK;
    unsigned char* const raws = sv + Shape::kVs * Shape::kV;   // [places of keys, of values][integers, then scales]
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
    auto lse_at = [&](int r) {
        const int tok = (row_lo + r) / a.group;
        return (int64_t)(w.first + tok) * a.lse_stride + kvh * a.group + row_lo + r - tok * a.group;
    };
    float* const part = a.part + (size_t)(blockIdx.x * gridDim.y + blockIdx.y) * (kTileRows2 * (HD + 2));
    if (!w.inside) {
        if (splits == 1) {
            for (int e = tid; e < row_n * hd; e += kTileThreads) store1(a.out, row_at(e / hd, a.out_stride) + e % hd, a.typ, __int_as_float(0x7fffffff));
            if (a.lse && tid < row_n) a.lse[lse_at(tid)] = __int_as_float(0x7fffffff);
        } else if (tid < kTileRows2) {
            part[tid] = 0.0f;
            part[kTileRows2 + tid] = __int_as_float(0x7fffffff);
            for (int d = 0; d < HD; d++) part[2 * kTileRows2 + tid * HD + d] = 0.0f;
        }
        return;
    }
    // keys: from the first row's window to the last row's slot; this block's share of their tiles
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
            mbar_init(&sh.k_free[t], 1);
            mbar_init(&sh.v_free[t], 1);
            mbar_init(&sh.p_full[t], 128);
            for (int x = 0; x < 2; x++) {
                mbar_init(&sh.raw_full[t][x], 1);
                mbar_init(&sh.raw_free[t][x], kConvWarps);
            }
            mbar_init(&sh.k_full[t], kConvWarps);
            mbar_init(&sh.v_full[t], kConvWarps);
        }
        for (int t = 0; t < kSlots; t++) mbar_init(&sh.c_full[t], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 0) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t col_s[2] = {tmem, tmem + 128}, col_o[2] = {tmem + 256, tmem + 384};

    // the queries as f16, each row times a power of two of its own: what a row gives does not depend on the others.  Eight dims stand in the order (0, 4), (1, 5), (2, 6), (3, 7), as the keys' words give them.
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
                const int d = 8 * (x >> 2) + (x & 3);
                if (SPLIT) h2_split(v[d] * up, v[d + 4] * up, hi[x], lo[x]);
                else hi[x] = h2_pack(v[d] * up, v[d + 4] * up);
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
            // All lanes go the same way and one of them issues.  The allocation is of all columns, so it begins at 0, and the places in shared memory are counted from its base: operands that are the warp's.
            const uint32_t q_at = (smem_u32(raw_smem) + 1023u) & ~1023u, k_at = q_at + Shape::kQ, v_at = k_at + Shape::kVs * Shape::kK;
            const uint32_t one = elect_lane();
            auto scores = [&](int t, int i) {
#pragma unroll
                for (int term = TERMS - 1; term >= 0; term--) {  // the low parts first: what is cut off then is small
                    const uint32_t dq = desc_low(q_at + (t * TERMS + term) * Shape::kPart), dk = desc_low(k_at + (i % Shape::kVs) * Shape::kK);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ks++) {
                        const uint32_t off = ((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4;
                        mma_ss_low(one, 128 * t, dq + off, dk + off, idesc_f16(kKeys), term < TERMS - 1 || ks > 0);
                    }
                }
                if (one) {
                    umma_commit(&sh.s_full[t]);
                    if (t == last) umma_commit(&sh.k_free[i % Shape::kVs]);
                }
                __syncwarp();
            };
            auto sums = [&](int t, int i) {
                const uint32_t dv = desc_low(v_at + (i % Shape::kVs) * Shape::kV), on = !SPLIT && i > 0;
#pragma unroll
                for (int term = TERMS - 1; term >= 0; term--)
#pragma unroll
                    for (int ks = 0; ks < kKeys / 16; ks++)
                        mma_ts_low(one, 256 + 128 * t, 128 * t + 16 * ks + 8 * term, dv + (((ks >> 2) * (HD * 128) + (ks & 3) * 32) >> 4), idesc_f16(HD), term < TERMS - 1 || ks > 0 ? 1u : on);
                if (one) {
                    umma_commit(&sh.o_full[t]);
                    if (t == last) umma_commit(&sh.v_free[i % Shape::kVs]);
                }
                __syncwarp();
            };
            bool ok = __all_sync(0xffffffffu, tmem == 0 && mbar_wait(&sh.k_full[0], 0));
            tc_fence_after();
            for (int t = 0; t < n_tiles && ok; t++) scores(t, 0);
            for (int i = 0; i < n && ok; i++) {
                const bool more = i + 1 < n;
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.v_full[i % Shape::kVs], (i / Shape::kVs) & 1));
                for (int t = 0; t < n_tiles && ok; t++) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.p_full[t], i & 1));
                    tc_fence_after();
                    if (!ok) break;
                    sums(t, i);
                    if (more) {
                        if (t == 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.k_full[(i + 1) % Shape::kVs], ((i + 1) / Shape::kVs) & 1));
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, i + 1);
                    }
                }
            }
        } else {
            // -------------------------------------------------------------------------------------------------- copies
            const int32_t* table = seqs.table + (size_t)seq * seqs.width;
            const int page_mask = (1 << pool.page_shift) - 1;
            const uint32_t ints = 8 * hd, scales = hd;      // bytes of 16 rows
            auto look_up = [&](int i) {  // lane g < 8: the page of group g; -1 in front of every row's window and behind the end, -2 outside the pool
                const int key = (tile0 + i) * kKeys + lane * 16;
                if (lane >= kGroups || i >= n || key + 15 < key_lo || key >= key_end) return -1;
                const int p = table[key >> pool.page_shift];
                return p >= 0 && p < pool.n_pages ? p : -2;
            };
            int page = look_up(0);
            bool ok = true;
            int issued[2] = {0, 0};
            for (int i = 0; i < n && ok; i++) {
                const int next = look_up(i + 1);
                const size_t row = ((((size_t)(page < 0 ? 0 : page) * pool.n_kv + kvh) << pool.page_shift) + (((tile0 + i) * kKeys + lane * 16) & page_mask));
                const uint32_t bytes = (ints + scales) * __popc(__ballot_sync(0xffffffffu, page >= 0));
                const uint32_t outside = __ballot_sync(0xffffffffu, page == -2);
                for (int x = 0; x < 2; x++) {
                    const int places = x ? RV : RK, st = i % places;
                    if (i >= places) ok = __all_sync(0xffffffffu, mbar_wait(&sh.raw_free[st][x], (i / places - 1) & 1));
                    if (!ok) break;
                    if (x == 0 && lane == 0) {
                        sh.outside[i % kSlots] = outside;
                        if (outside) kv8_raise(seqs, seq);
                        mbar_arrive(&sh.c_full[i % kSlots]);
                    }
                    if (lane == 0) mbar_expect_tx(&sh.raw_full[st][x], bytes);
                    __syncwarp();
                    if (page >= 0) {
                        unsigned char* const to = raws + (x ? RK + st : st) * Shape::kRawHalf;
                        bulk_load(to + lane * ints, (x ? pool.v : pool.k) + row * (hd >> 1), ints, &sh.raw_full[st][x]);
                        bulk_load(to + kKeys * HD / 2 + lane * scales, (x ? pool.v_block : pool.k_block) + row * (hd >> 4), scales, &sh.raw_full[st][x]);
                    }
                    issued[x] = i + 1;
                }
                page = next;
            }
            if (!ok)  // whatever is under way lands before the block ends
                for (int x = 0; x < 2; x++)
                    for (int places = x ? RV : RK, i = max(0, issued[x] - places); i < issued[x]; i++) (void)mbar_wait(&sh.raw_full[i % places][x], (i / places) & 1);
        }
      } else {
        // ---------------------------------------------------------------------------------------------------- unpacking
        const int cw = warp < 12 ? warp - 8 : warp - 10, ct = cw * 32 + lane;
        constexpr int KC = HD / 16, VC = HD / 8;     // K: pieces of 16 dims of a key; V: words of 8 dims of a key
        const int row_ints = hd >> 1, row_scales = hd >> 4;
        // Rounds of 32 pieces: the keys' are 32 or 16, the values', twice as long, 8 or 4.  Warps with more of the values' have fewer of the keys'.
        constexpr int K_MORE = HD == 128 ? 6 : 4, K_LESS = HD == 128 ? 4 : 2, LESS = HD == 128 ? 2 : 4;   // the first LESS warps have K_LESS rounds of keys
        static_assert(LESS * K_LESS + (kConvWarps - LESS) * K_MORE == kKeys * KC / 32, "every round has a warp");
        const int k_from = cw < LESS ? cw * K_LESS : LESS * K_LESS + (cw - LESS) * K_MORE, k_to = k_from + (cw < LESS ? K_LESS : K_MORE);
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            const unsigned char* const rk = raws + (i % RK) * Shape::kRawHalf;
            const unsigned char* const rv = raws + (RK + i % RV) * Shape::kRawHalf;
            ok = mbar_wait(&sh.raw_full[i % RK][0], (i / RK) & 1);
            if (i >= Shape::kVs) ok = ok && mbar_wait(&sh.k_free[i % Shape::kVs], (i / Shape::kVs - 1) & 1);  // the keys' place is free
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            unsigned char* const k_to_place = sk + (i % Shape::kVs) * Shape::kK;
            // Two rounds at once, reads first: the compiler cannot know that the writes are elsewhere.  (Three: 368 us instead of 365; the reads of all: 469, registers.)
            constexpr int AT_ONCE = 2;
#pragma unroll 1
            for (int round = k_from; round < k_to; round += AT_ONCE) {
                uint2 ints[AT_ONCE];
                uint32_t scales[AT_ONCE];
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    const int e = (round + x) * 32 + lane, key = e / KC, ch = e % KC;
                    ints[x] = make_uint2(0, 0);
                    scales[x] = 0;  // dims behind the head's: zeros
                    if (round + x < k_to && ch * 16 < hd) {
                        ints[x] = *reinterpret_cast<const uint2*>(rk + key * row_ints + ch * 8);
                        scales[x] = rk[kKeys * HD / 2 + key * row_scales + ch];
                    }
                }
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    if (round + x >= k_to) break;
                    const int e = (round + x) * 32 + lane, key = e / KC, ch = e % KC;
                    // the upper half of a row's chunks writes its second piece first: eight lanes then meet all banks
                    const int swap = ch >= 4;
                    const Scale4 s = scale4_both(scales[x] & 0x7fu, 0);
                    uint32_t first[4], second[4];
                    values8(swap ? ints[x].y : ints[x].x, s, first);
                    values8(swap ? ints[x].x : ints[x].y, s, second);
                    unsigned char* dst = k_to_place + (ch >> 2) * (128 * 128);
                    *reinterpret_cast<uint4*>(dst + sw128(key, 2 * (ch & 3) + swap)) = make_uint4(first[0], first[1], first[2], first[3]);
                    *reinterpret_cast<uint4*>(dst + sw128(key, 2 * (ch & 3) + 1 - swap)) = make_uint4(second[0], second[1], second[2], second[3]);
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&sh.k_full[i % Shape::kVs]); mbar_arrive(&sh.raw_free[i % RK][0]); }

            ok = mbar_wait(&sh.raw_full[i % RV][1], (i / RV) & 1);
            if (i >= Shape::kVs) ok = ok && mbar_wait(&sh.v_free[i % Shape::kVs], (i / Shape::kVs - 1) & 1);  // the values' place is free
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            unsigned char* const to = sv + (i % Shape::kVs) * Shape::kV;
#pragma unroll 1
            for (int e = ct; e < 16 * VC; e += 32 * kConvWarps) {
                // eight keys, eight dims; every other octet of keys reads its pairs the other way round: the two that a warp has at a time then meet other banks
                const int octet = e / VC, word = e % VC, odd = octet & 1;
                const bool none = 8 * word >= hd;
                const uint32_t pick0 = odd ? 0x1054u : 0x5410u, pick1 = odd ? 0x3276u : 0x7632u;
                uint32_t out[8][4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int key = octet * 8 + 2 * k;
                    uint32_t u = 0, v = 0, su = 0, sv2 = 0;
                    if (!none) {
                        u = *reinterpret_cast<const uint32_t*>(rv + (key + odd) * row_ints + word * 4);
                        v = *reinterpret_cast<const uint32_t*>(rv + (key + 1 - odd) * row_ints + word * 4);
                        su = rv[kKeys * HD / 2 + key * row_scales + (word >> 1)];
                        sv2 = rv[kKeys * HD / 2 + (key + 1) * row_scales + (word >> 1)];
                    }
                    const Scale4 s = scale4_pair(su, sv2);
                    const uint32_t x = __byte_perm(u, v, pick0), y = __byte_perm(u, v, pick1);  // (key, key + 1) of dims 0 - 3, of 4 - 7
                    out[0][k] = value_lo(x, s); out[1][k] = value_hi(x, s); out[2][k] = value_lo(x >> 8, s); out[3][k] = value_hi(x >> 8, s);
                    out[4][k] = value_lo(y, s); out[5][k] = value_hi(y, s); out[6][k] = value_lo(y >> 8, s); out[7][k] = value_hi(y >> 8, s);
                }
#pragma unroll
                for (int b = 0; b < 8; b++)  // row b VC + l holds dim 8 l + b: eight lanes write eight rows
                    *reinterpret_cast<uint4*>(to + (octet >> 3) * (HD * 128) + sw128(b * VC + word, octet & 7)) = make_uint4(out[b][0], out[b][1], out[b][2], out[b][3]);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&sh.v_full[i % Shape::kVs]); mbar_arrive(&sh.raw_free[i % RV][1]); }
        }
      }
    } else {
        // ------------------------------------------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kSoftRegs));
        const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_s = col_s[t] + lanes, my_o = col_o[t] + lanes;
        const int limit = w.ctx + (row_lo + min(r, row_n - 1)) / a.group;      // last slot that the row sees
        const int least = __shfl_sync(0xffffffffu, limit, 0), most = __shfl_sync(0xffffffffu, limit, 31);
        // NaN for a row that is not finite, whose scores may all be minus infinity, as masked ones are
        const float f = sh.down[r] == 255 ? __int_as_float(0x7fffffff) : score_factor(a.scale_log2, __uint_as_float((uint32_t)sh.down[r] << 23), kUnit4 * pool.k_scale[kvh]);
        float o[HD], m = kNegInf, l = 0.0f, corr = 1.0f;
        bool ok = true, far = false;
        // Far from 0 a reference has no bits left for what is added to it, and a product that is rounded with it may be off by more than f16's range
        // (scores of 1e8: 2^4).  There a score is rounded by itself, as the reference was, and what remains over it goes on; without loss in a neighbourhood of the reference.
        auto is_far = [](float mx) { return fabsf(mx) > 65536.0f && mx != kNegInf; };
        auto over = [&](float x, float ref) {
            const float y = __fsub_rn(__fmul_rn(x, f), ref);
            return y > 9.0f ? 9.0f : y;  // 2^15 at most; NaN stays
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
                const uint32_t outside = sh.outside[i % kSlots];
                const int key0 = (tile0 + i) * kKeys;
                const bool plain = key0 + kKeys - 1 <= least && (a.window == 0 || key0 > most - a.window) && outside == 0;
                // places of the tile that the row sees: [from, to]
                const int to = limit - key0, from = a.window > 0 ? limit - a.window + 1 - key0 : 0;
                auto mask = [&](uint32_t& x, int e) {
                    if (outside >> (e >> 4) & 1) x = 0x7fffffffu;
                    if (e > to || e < from) x = __float_as_uint(kNegInf);
                };
                float top = kNegInf, sum = 0.0f;
                if constexpr (SPLIT) {
#pragma unroll 1
                    for (int c = 0; c < kKeys; c += 32) {
                        uint32_t x[32];
                        tmem_ld32(my_s + c, x);
                        tmem_wait_ld();
                        if (!plain)
#pragma unroll
                            for (int e = 0; e < 32; e++) mask(x[e], c + e);
#pragma unroll
                        for (int e = 0; e < 32; e++) top = fmaxf(top, __uint_as_float(x[e]));
                    }
                    const float mx = fmaxf(m, __fmul_rn(top, f)), ref = mx == kNegInf ? 0.0f : mx;
                    far = is_far(mx);
                    const bool any_far = __any_sync(0xffffffffu, far);
                    const float off = far ? kTileUp : kTileUp - ref, by = far ? 1.0f : f;
                    corr = exp2_fast(m - ref);
                    m = mx;
                    // 16 keys' weights take the first 8 columns of their scores' 16, their low parts the other 8
#pragma unroll 2
                    for (int c = 0; c < kKeys; c += 16) {
                        uint32_t x[16], p[8], q[8];
                        tmem_ld16(my_s + c, x);
                        tmem_wait_ld();
                        if (!plain)
#pragma unroll
                            for (int e = 0; e < 16; e++) mask(x[e], c + e);
                        if (any_far)
#pragma unroll
                            for (int e = 0; e < 16; e++) x[e] = far ? __float_as_uint(over(__uint_as_float(x[e]), ref)) : x[e];
                        const float2 f2 = make_float2(by, by), off2 = make_float2(off, off);
                        float2 gs = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, off2), v = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            gs = add2(gs, v);
                            h2_split(v.x, v.y, p[e / 2], q[e / 2]);
                        }
                        sum += gs.x + gs.y;
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
                        for (int e = 0; e < kKeys; e++) mask(x[e], e);
                    float tops[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                    for (int e = 0; e < kKeys; e++) tops[e & 3] = fmaxf(tops[e & 3], __uint_as_float(x[e]));
                    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    const float mx = fmaxf(m, __fmul_rn(top, f));
                    const bool raise = mx - m > 8.0f;  // also from minus infinity; the difference, because far from 0 m + 8 may be rounded up to the next number, which mx may be
                    if (__any_sync(0xffffffffu, raise)) {
                        const float by = raise ? exp2_fast(m - mx) : 1.0f;
                        if (raise) m = mx;
                        far = is_far(m);
                        l *= by;
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
                                for (int e = 0; e < 16; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * by);
                                tmem_st16(my_o + c, y);
                            }
                        }
                    }
                    const float ref = m == kNegInf ? 0.0f : m;
                    const float off = far ? kTileUp : kTileUp - ref, by = far ? 1.0f : f;
                    if (__any_sync(0xffffffffu, far))
#pragma unroll
                        for (int e = 0; e < kKeys; e++) x[e] = far ? __float_as_uint(over(__uint_as_float(x[e]), ref)) : x[e];
                    const float2 f2 = make_float2(by, by), off2 = make_float2(off, off);
                    float2 gs = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int c = 0; c < kKeys; c += 16) {
                        uint32_t p[8];
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(__uint_as_float(x[c + e]), __uint_as_float(x[c + e + 1])), f2, off2), v = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            gs = add2(gs, v);
                            p[e / 2] = h2_pack(v.x, v.y);
                        }
                        tmem_st8(my_s + c, p);
                    }
                    l += gs.x + gs.y;
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
            const float unit = kUnit4 * pool.v_scale[kvh];
            if (r < row_n) {
                if (splits == 1) {
                    const float by = unit / l;
                    const int64_t dst = row_at(r, a.out_stride);
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = o[(e & 7) * (HD / 8) + ((d + e) >> 3)] * by;
                        if (d < hd) store16(a.out, dst + d, a.typ, a.out_vec, v);
                    }
                    if (a.lse) a.lse[lse_at(r)] = (m + (log2f(l) - kTileUp)) * 0.693147180559945f;
                } else {
                    part[r] = m;
                    part[kTileRows2 + r] = l;
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = o[(e & 7) * (HD / 8) + ((d + e) >> 3)] * unit;
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

template <int HD, bool SPLIT>
int32_t tiles_as(const Kv4Pool& pool, const Kv8Seqs& seqs, AttnArgs a, const TilePlan& plan, cudaStream_t s) {
    using Shape = TileShape<HD, SPLIT>;
    const void* kern = (const void*)kv4_tiles_kernel<HD, SPLIT>;
    const size_t smem = std::max<size_t>(Shape::kBytes, (size_t)2 * (seqs.n_seqs + 1) * 4 + 1024);
    a.lse_less = kTileUp;
    LC_CUDA(ensure_smem_limit(kern, smem));
    static const int regs = [&] {  // setmaxnreg counts on the launch's registers: a build that has fewer must not start it
        cudaFuncAttributes at;
        return cudaFuncGetAttributes(&at, kern) == cudaSuccess ? at.numRegs : 0;
    }();
    LC_CHECK(regs == kLaunchRegs, LC_ERR_UNSUPPORTED, "attention in tiles was built with %d registers a thread instead of %d", regs, kLaunchRegs);
    kv4_tiles_kernel<HD, SPLIT><<<dim3((unsigned)plan.units, (unsigned)plan.splits), kTileThreads, smem, s>>>(pool, seqs, a, plan.splits);
    LC_CUDA(cudaGetLastError());
    if (plan.splits > 1) {
        const size_t cum = (size_t)2 * (seqs.n_seqs + 1) * 4;
        LC_CUDA(launch_pdl(kv_tiles_join_kernel<HD>, dim3((unsigned)plan.units, kTileRows2 / 8), dim3(256), cum, s, (const Kv8Pool&)pool, seqs, a, plan.splits));
    }
    return LC_OK;
}

}  // namespace

int32_t launch_kv4_tiles(const Kv4Pool& pool, const Kv8Seqs& seqs, const AttnArgs& a, const TilePlan& plan, cudaStream_t s) {
    if (pool.hd <= 64) return a.typ == LC_TYPE_F32 ? tiles_as<64, true>(pool, seqs, a, plan, s) : tiles_as<64, false>(pool, seqs, a, plan, s);
    return a.typ == LC_TYPE_F32 ? tiles_as<128, true>(pool, seqs, a, plan, s) : tiles_as<128, false>(pool, seqs, a, plan, s);
}

}  // namespace lc
