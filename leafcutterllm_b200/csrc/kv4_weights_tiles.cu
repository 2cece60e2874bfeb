// What weight many rows gave the cached keys, on tcgen05: mass[sequence][kv head][slot] += sum over rows and heads of the group of 2^(f_r q_r . k - L_r).
//
// A block takes 256 keys of a sequence and kv head, makes f16 values of them in shared memory (exactly), once, and goes over the rows 128 at a time: queries as f16 (after a power of two of
// each row's own; f32: high and low parts), products with the KEYS as the operand of 128 rows, so that a key's scores of all rows come to one thread, which adds their weights up in registers: nothing is
// exchanged between threads, and a sum is in the order of the rows.  Two blocks on an SM take turns on the matrix unit.
//
// 64 rows of three sequences of 3,000 to 16,000 slots, 32 heads over 8 of 128 in f16: 51 us, 13.6 GFLOP (8.3 us at the rate of library products; by runs 123).  What bounds it are instructions, and a block's phases one
// after the other: keys to values 4,400 cycles once, then for 128 rows their conversion 3,000, the products 1,900 (of the unit, 990: 16 of 62) and 32,768 exponentials with their sums 2,300 to 2,700 (of the unit, 2,048).
// Bringing the next stretch into L2 early gained nothing.
#include <algorithm>
#include <type_traits>
#include "lc_attn_tiles.cuh"
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_kv4_weights.cuh"

namespace lc {

namespace {

constexpr int kUnitKeys = 256, kWeightRows = 128, kWeightThreads = 256;

struct WeightShared {
    uint64_t done[2];                  // scores of the two tiles of keys
    uint32_t tmem;
    uint32_t sums[kWeightThreads / 32];
    int64_t at[kUnitKeys];             // the keys' rows in the pool; -1: none
    // of two tiles of rows, in turn
    float4 row[2][kWeightRows / 2];    // (f, f, -L, -L) of two rows
    int64_t from[2][kWeightRows];      // of a row's queries; -1: none
    int limit[2][kWeightRows];         // last slot that the row sees; -1: none
};
template <int HD, bool SPLIT> struct WeightTiles {
    static constexpr int kPart = HD * 256;                      // 128 rows of HD f16
    static constexpr int kBytes = 2 * kPart + (SPLIT ? 2 : 1) * kPart + 1024;
};

// Units of a sequence: of each kv head its keys' stretches of 256.
__device__ __forceinline__ uint32_t weight_units(const Kv8Seqs& s, const Kv8Pool& p, const WeightArgs& a, int i, int& first, int& n, int& ctx, int& chunk0) {
    ctx = s.ctx[i];
    chunk0 = 0;
    if (!kv8_span(s, i, first, n) || n == 0 || !kv8_in_table(s, p, ctx, n) || ctx + n > a.capacity) return 0;
    if (a.window > 0) chunk0 = max(0, ctx - a.window + 1) / kUnitKeys;
    return (uint32_t)((ctx + n + kUnitKeys - 1) / kUnitKeys - chunk0) * (uint32_t)p.n_kv;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kWeightThreads, sizeof(T) == 4 ? 1 : 2) kv4_weights_tiles_kernel(Kv4Pool pool, Kv8Seqs seqs, WeightArgs a) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int TERMS = SPLIT ? 2 : 1, PART = WeightTiles<HD, SPLIT>::kPart;
    extern __shared__ unsigned char raw_smem[];
    __shared__ WeightShared sh;
    unsigned char* const sk = (unsigned char*)(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);   // [2 tiles of 128 keys]
    unsigned char* const sq = sk + 2 * PART;                                                       // [high, low]
    uint32_t* const cum = reinterpret_cast<uint32_t*>(sq + TERMS * PART);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hd = pool.hd;
    if (blockIdx.x == 0) weights_check_seqs(pool, seqs, a);
    // cum[i]: units before sequence i
    {
        const int per = (seqs.n_seqs + kWeightThreads - 1) / kWeightThreads, i0 = min(tid * per, seqs.n_seqs), i1 = min(i0 + per, seqs.n_seqs);
        uint32_t sum = 0;
        int first, n, ctx, chunk0;
        for (int i = i0; i < i1; i++) {
            cum[i] = sum;
            sum = add_places(sum, weight_units(seqs, pool, a, i, first, n, ctx, chunk0));
        }
        uint32_t incl = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl = add_places(incl, v);
        }
        if (lane == 31) sh.sums[warp] = incl;
        __syncthreads();
        uint32_t before = __shfl_up_sync(0xffffffffu, incl, 1), total = 0;
        if (lane == 0) before = 0;
        for (int w = 0; w < kWeightThreads / 32; w++) {
            if (w < warp) before = add_places(before, sh.sums[w]);
            total = add_places(total, sh.sums[w]);
        }
        for (int i = i0; i < i1; i++) cum[i] = add_places(cum[i], before);
        if (tid == 0) cum[seqs.n_seqs] = total;
    }
    if (tid == 0) {
        mbar_init(&sh.done[0], 1);
        mbar_init(&sh.done[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 0) tmem_alloc(&sh.tmem, 256);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t total = cum[seqs.n_seqs];
    const uint32_t tmem = sh.tmem;
    uint32_t phase = 0;
    bool ok = true;
    for (uint32_t unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
        const int seq = seq_at(cum, seqs.n_seqs, unit);
        int first, n, ctx, chunk0;
        const uint32_t of_seq = weight_units(seqs, pool, a, seq, first, n, ctx, chunk0), in = unit - cum[seq];
        const int chunks = of_seq / pool.n_kv, kvh = in / chunks, key0 = (chunk0 + (int)(in - (uint32_t)kvh * chunks)) * kUnitKeys;
        const int rows = n * a.group;

        // rows in front of the keys see none of them, and rows whose window begins behind them
        const int r_from = max(0, key0 - ctx) * a.group / kWeightRows * kWeightRows;
        const int r_end = a.window > 0 ? (int)min((int64_t)rows, ((int64_t)key0 + kUnitKeys - 1 + a.window - ctx) * a.group) : rows;
        // the rows' numbers, a thread each (of the half that does not issue the products): those behind the last row, and those without a finite lse, are zeros that add nothing
        auto numbers = [&](int r0, int to) {
            const int at = tid - (kWeightThreads - kWeightRows);
            if (at < 0 || r0 >= r_end) return;
            const int mine = min(kWeightRows, rows - r0), r = r0 + min(at, mine - 1), tok = r / a.group, hq = kvh * a.group + r - tok * a.group;
            const float lse = a.lse[(int64_t)(first + tok) * a.lse_stride + hq];
            const bool counts = at < mine && fabsf(lse) < INFINITY;
            sh.from[to][at] = counts ? (int64_t)(first + tok) * a.q_stride + (int64_t)hq * hd : -1;
            sh.limit[to][at] = counts ? ctx + tok : -1;
            float* const k = reinterpret_cast<float*>(&sh.row[to][at >> 1]) + (at & 1);
            k[0] = 0.0f;
            k[2] = counts ? -lse * 1.44269504088896f : kNegInf;
        };
        numbers(r_from, 0);

        // a key per thread
        const int key = key0 + tid;
        bool held = key < ctx + n;
        {
            const int number = held ? seqs.table[(size_t)seq * seqs.width + (key >> pool.page_shift)] : 0;
            // in front of every row's window: not looked at
            const bool seen = held && (a.window == 0 || key > ctx - a.window);
            if (seen && (number < 0 || number >= pool.n_pages)) kv8_raise(seqs, seq);
            held = seen && number >= 0 && number < pool.n_pages;
            sh.at[tid] = held ? (int64_t)((((size_t)number * pool.n_kv + kvh) << pool.page_shift) + (key & ((1 << pool.page_shift) - 1))) : -1;
        }
        __syncthreads();
        {
            // 16 dims of a key at a time: neighbours read neighbouring bytes
            constexpr int C = HD / 16;
#pragma unroll 8
            for (int e = tid; e < kUnitKeys * C; e += kWeightThreads) {
                const int r = e / C, ch = e % C;
                const int64_t row = sh.at[r];
                uint32_t u[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
                // the upper half of a row's chunks writes its second piece first: eight threads then meet all banks
                const int swap = ch >= 4;
                if (row >= 0 && ch * 16 < hd) {
                    const uint2 x = *reinterpret_cast<const uint2*>(pool.k + row * (hd >> 1) + ch * 8);
                    const Scale4 s = scale4_both(pool.k_block[row * (hd >> 4) + ch] & 0x7fu, 0);
                    values8(swap ? x.y : x.x, s, u);
                    values8(swap ? x.x : x.y, s, v);
                }
                unsigned char* const to = sk + (r >> 7) * PART + (ch >> 2) * (128 * 128);
                *reinterpret_cast<uint4*>(to + sw128(r & 127, 2 * (ch & 3) + swap)) = make_uint4(u[0], u[1], u[2], u[3]);
                *reinterpret_cast<uint4*>(to + sw128(r & 127, 2 * (ch & 3) + 1 - swap)) = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
        const float head = kUnit4 * pool.k_scale[kvh];
        float* const mass = a.mass + (int64_t)seq * a.mass_stride + (int64_t)kvh * a.mass_head_stride + key;
        const float before = held ? *mass : 0.0f;
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        for (int r0 = r_from, turn = 0; r0 < r_end && ok; r0 += kWeightRows, turn ^= 1) {
            const int mine = min(kWeightRows, rows - r0);
            // the queries: HD / 16 threads a row
            constexpr int C = HD / 16;
#pragma unroll(SPLIT ? 2 : 4)
            for (int e = tid; e < kWeightRows * C; e += kWeightThreads) {
                const int r = e / C, ch = e % C;
                const int64_t at_q = sh.from[turn][r];
                const bool here = at_q >= 0 && ch * 16 < hd;
                float* const k = reinterpret_cast<float*>(&sh.row[turn][r >> 1]) + (r & 1);
                const int at0 = (ch >> 2) * (128 * 128) + sw128(r, 2 * (ch & 3)), at1 = (ch >> 2) * (128 * 128) + sw128(r, 2 * (ch & 3) + 1);
                if constexpr (!SPLIT) {
                    // pairs of 16 bits: the largest magnitude of a row by pairs; f16 as it is, bf16 times a power of two
                    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
                    __align__(16) T x[16];
#pragma unroll
                    for (int y = 0; y < 2; y++) reinterpret_cast<uint4*>(x)[y] = make_uint4(0, 0, 0, 0);
                    if (here) {
                        if (a.q_vec)
#pragma unroll
                            for (int y = 0; y < 2; y++) reinterpret_cast<uint4*>(x)[y] = reinterpret_cast<const uint4*>((const T*)a.q + at_q + ch * 16)[y];
                        else
#pragma unroll
                            for (int y = 0; y < 16; y++) x[y] = ((const T*)a.q)[at_q + ch * 16 + y];
                    }
                    const Pair* const pairs = reinterpret_cast<const Pair*>(x);
                    Pair most = __habs2(pairs[0]);
#pragma unroll
                    for (int y = 1; y < 8; y++) most = __hmax2_nan(most, __habs2(pairs[y]));
                    float top = max_nan(elem_f(most.x), elem_f(most.y));
#pragma unroll
                    for (int o = C / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const bool finite = top < INFINITY;
                    float up = 1.0f, down = 1.0f;
                    if (!std::is_same<T, __half>::value) row_scale(top, up, down);
                    if (ch == 0) {
                        if (finite) k[0] = score_factor(a.scale_log2, down, head);
                        else { sh.limit[turn][r] = -1; k[2] = kNegInf; }   // a row that is not finite adds nothing either
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            if constexpr (std::is_same<T, __half>::value) {
                                const uint32_t lo = reinterpret_cast<const uint32_t*>(x)[4 * y + (z >> 1)], hi = reinterpret_cast<const uint32_t*>(x)[4 * y + 2 + (z >> 1)];
                                w[4 * y + z] = __byte_perm(lo, hi, z & 1 ? 0x7632 : 0x5410);
                            } else {
                                w[4 * y + z] = h2_pack(elem_f(x[8 * y + z]) * up, elem_f(x[8 * y + z + 4]) * up);
                            }
                        }
                    if (!finite)
#pragma unroll
                        for (int y = 0; y < 8; y++) w[y] = 0;
                    *reinterpret_cast<uint4*>(sq + at0) = make_uint4(w[0], w[1], w[2], w[3]);
                    *reinterpret_cast<uint4*>(sq + at1) = make_uint4(w[4], w[5], w[6], w[7]);
                } else {
                    float v[16], top = 0.0f;
                    if (here) load16((const T*)a.q + at_q + ch * 16, a.q_vec, v);
                    else
#pragma unroll
                        for (int x = 0; x < 16; x++) v[x] = 0.0f;
#pragma unroll
                    for (int x = 0; x < 16; x++) top = max_nan(top, fabsf(v[x]));
#pragma unroll
                    for (int o = C / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const bool finite = top < INFINITY;
                    float up, down;
                    row_scale(top, up, down);
                    if (ch == 0) {
                        if (finite) k[0] = score_factor(a.scale_log2, down, head);
                        else { sh.limit[turn][r] = -1; k[2] = kNegInf; }
                    }
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        const int d = 8 * (x >> 2) + (x & 3);
                        h2_split(finite ? v[d] * up : 0.0f, finite ? v[d + 4] * up : 0.0f, hi[x], lo[x]);
                    }
                    *reinterpret_cast<uint4*>(sq + at0) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(sq + at1) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                    *reinterpret_cast<uint4*>(sq + PART + at0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    *reinterpret_cast<uint4*>(sq + PART + at1) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                }
            }
            fence_async();
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            if (tid == 0) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
#pragma unroll
                    for (int term = TERMS - 1; term >= 0; term--) {  // the low parts first: what is cut off then is small
                        const uint64_t dk = umma_desc_sw128(smem_u32(sk + t * PART)), dq = umma_desc_sw128(smem_u32(sq + term * PART));
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ks++) {
                            const uint64_t off = ((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4;
                            umma_f16_ss(tmem + 128 * t, dk + off, dq + off, idesc_f16(kWeightRows), term < TERMS - 1 || ks > 0);
                        }
                    }
                    umma_commit(&sh.done[t]);
                }
            }
            numbers(r0 + kWeightRows, turn ^ 1);   // the next ones, while the products run
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.done[warp >> 2], phase));
            phase ^= 1;
            tc_fence_after();
            // rows see all keys of the block: with all of these rows there, and none of them in front of its last key or with a window behind its first
            const int tok_first = r0 / a.group, tok_last = (r0 + mine - 1) / a.group;
            const bool plain = ctx + tok_first >= key0 + kUnitKeys - 1 && (a.window == 0 || ctx + tok_last - a.window < key0);
            const uint32_t from = tmem + 128 * (warp >> 2) + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < kWeightRows; c += 32) {
                uint32_t x[32];
                tmem_ld32(from + c, x);
                tmem_wait_ld();
                if (!plain)
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int limit = sh.limit[turn][c + e];
                        if (key > limit || (a.window > 0 && key <= limit - a.window)) x[e] = __float_as_uint(kNegInf);
                    }
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float4 k = sh.row[turn][(c + e) / 2];
                    float2 y = fma2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), make_float2(k.x, k.y), make_float2(k.z, k.w));
                    if (!plain) {  // a masked score times a factor that is 0
                        if (x[e] == 0xff800000u) y.x = kNegInf;
                        if (x[e + 1] == 0xff800000u) y.y = kNegInf;
                    }
                    sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], make_float2(exp2_fast(y.x), exp2_fast(y.y)));
                }
            }
            tc_fence_before();
            ok = __syncthreads_and(ok);   // the queries' place, the rows' numbers and the scores' columns are free
            tc_fence_after();
        }
        if (!ok && tid == 0) kv8_raise(seqs, seq);
        if (held && ok) *mass = before + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
        __syncthreads();       // and the keys' place
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_free(tmem, 256);
}

template <int HD, typename T> int32_t tiles_as(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s) {
    constexpr bool split = sizeof(T) == 4;
    const size_t smem = WeightTiles<HD, split>::kBytes + (size_t)(seqs.n_seqs + 1) * 4;
    LC_CUDA(ensure_smem_limit((const void*)kv4_weights_tiles_kernel<HD, T>, smem));
    const int64_t chunks = (((int64_t)seqs.width << pool.page_shift) + kUnitKeys - 1) / kUnitKeys + 1;
    const int64_t blocks = std::min<int64_t>((int64_t)sm_count() * (split ? 1 : 2), chunks * seqs.n_seqs * pool.n_kv);
    kv4_weights_tiles_kernel<HD, T><<<(unsigned)blocks, kWeightThreads, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
template <int HD> int32_t tiles_of(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s) {
    return a.typ == LC_TYPE_F32 ? tiles_as<HD, float>(pool, seqs, a, s) : a.typ == LC_TYPE_F16 ? tiles_as<HD, __half>(pool, seqs, a, s) : tiles_as<HD, __nv_bfloat16>(pool, seqs, a, s);
}

}  // namespace

int32_t launch_kv4_weights_tiles(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s) {
    return pool.hd <= 64 ? tiles_of<64>(pool, seqs, a, s) : tiles_of<128>(pool, seqs, a, s);
}

}  // namespace lc
