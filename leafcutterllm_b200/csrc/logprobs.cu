// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits, in one pass over them.
//
// With m the row's maximum, d = x - m, S = sum e^d and T = sum e^d d:   log p(x) = d - log S,   entropy = log S - T / S.
// Every thread keeps a running S and T against its warp's m, sixteen logits at a time, whose f32 sums are added in 64 bits.  A later maximum m' turns
// (S, T) into (f S, f (T + (m - m') S)), f = e^(m - m').  m is the warp's and not the lane's: some lane finds a new maximum of its own in most steps, a warp in
// one of six (2,048 rows of 128,256, bf16: 255 us with maxima of lanes, 157 now: 3.3 TB/s, three quarters of the issue slots).
//
// The best `top`: a logit below the block's bound cannot be among them.  The bound is the top-th largest of the maxima of groups of
// four threads after 1, 2, 4, ... steps, and every logit that reaches it goes to a list of its warp's; a full list is cut to its best `top` by counting,
// for each, the larger ones.
//
// A row goes to a cluster of 1, 2, 4 or 8 blocks, which join over distributed shared memory: one launch, no workspace.
#include <cooperative_groups.h>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include <algorithm>

namespace lc {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, kChunkElems = 16, kMaxCluster = 8, kMaxTop = 32, kList = 128, kGroups = kThreads / 4;

// e^-200 is 0 in f32; a difference of logits may be minus infinity, and 0 times that is not 0
constexpr float kLeastExponent = -200.0f;

struct Sums {
    float m;
    double s, t;
};
// Of the sums in the lanes of a warp (m minus infinity: none), in all lanes.
__device__ __forceinline__ Sums join_lanes(Sums a) {
    const float m = warp_max(a.m), d = fmaxf(a.m - m, kLeastExponent);
    const double f = a.m == -INFINITY ? 0.0 : (double)expf(d);
    double s = f * a.s, t = a.m == -INFINITY ? 0.0 : f * (a.t + (double)d * a.s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    return Sums{m, s, t};
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Whole numbers in the order of the logits; -0 equals 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long key_of(float x, int index) { return ((unsigned long long)order_of(x) << 32) | (uint32_t)~index; }

struct LogprobArgs {
    const void* x;
    const int64_t* tokens;
    float* logprob;
    float* entropy;
    float* top_logprob;
    int64_t* top_id;
    int64_t stride;
    int vocab, top, vec;  // vec: rows are 16-byte aligned
    int size_shift;       // blocks of a row = 1 << size_shift
};

// what a block leaves for its cluster
struct BlockPart {
    Sums sums;
    int bad;
    unsigned long long keys[kMaxTop];
};

// Sixteen logits of a thread as they lie in memory: `U` pieces of 16 bytes, a block's width apart.  Places behind the end give minus infinity.
template <typename T> struct Chunk {
    static constexpr int E = 16 / sizeof(T), U = kChunkElems / E;
    uint4 w[U];
    __device__ __forceinline__ void load(const T* row, int piece0, int n, bool vec) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = (piece0 + u * kThreads) * E;
            if (vec && at + E <= n) {
                w[u] = __ldcs(reinterpret_cast<const uint4*>(row + at));
            } else {
                __align__(16) T t[E];
#pragma unroll
                for (int e = 0; e < E; e++) t[e] = at + e < n ? row[at + e] : to_elem<T>(-INFINITY);
                w[u] = *reinterpret_cast<const uint4*>(t);
            }
        }
    }
    __device__ __forceinline__ void values(float (&x)[kChunkElems]) const {
#pragma unroll
        for (int u = 0; u < U; u++) {
            __align__(16) T t[E];
            *reinterpret_cast<uint4*>(t) = w[u];
#pragma unroll
            for (int e = 0; e < E; e++) x[u * E + e] = elem_f(t[e]);
        }
    }
};
// By a whole warp: cuts its list to the best `top`; returns the last of them, or 0 where there are fewer.  Not inlined: one copy of it per place in the unrolled
// search made the code so long that a step's way through it took 13,000 cycles.
__device__ __noinline__ unsigned long long cut_list(unsigned long long* list, int listed, int top, uint32_t* bound) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    unsigned long long key[kList / 32];
    int above[kList / 32];
#pragma unroll
    for (int k = 0; k < kList / 32; k++) {
        key[k] = k * 32 + lane < listed ? list[k * 32 + lane] : 0ull;
        above[k] = 0;
    }
#pragma unroll 4
    for (int j = 0; j < listed; j++) {
        const unsigned long long other = list[j];
#pragma unroll
        for (int k = 0; k < kList / 32; k++) above[k] += other > key[k];
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kList / 32; k++)
        if (key[k] != 0ull && above[k] < top) list[above[k]] = key[k];
    __syncwarp();
    if (listed < top) return 0ull;
    const unsigned long long last = list[top - 1];
    if (lane == 0) atomicMax(bound, (uint32_t)(last >> 32));
    return last;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(LogprobArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ BlockPart part;
    __shared__ Sums warp_sums[kWarps];
    __shared__ int s_bad;
    __shared__ uint32_t s_bound;                       // order of a value that at least `top` logits reach
    __shared__ unsigned long long s_list[kWarps][kList];
    __shared__ int s_count[kWarps];
    __shared__ __align__(16) uint32_t s_seen[kWarps][kGroups];
    static_assert(kGroups == 64, "two maxima a lane");
    __shared__ uint32_t s_top[kGroups];                // maxima of four lanes each, in the order of whole numbers
    __shared__ unsigned long long s_keys[kThreads];
    static_assert(kMaxCluster * kMaxTop <= kThreads && kWarps * kMaxTop <= kThreads, "a thread for each of the keys that are joined");
    cg::cluster_group cluster = cg::this_cluster();
    const int size = 1 << a.size_shift, rank = blockIdx.x & (size - 1);
    const int64_t r = blockIdx.x >> a.size_shift;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* whole = (const T*)a.x + r * a.stride;
    // this block's slice, in pieces of 16 bytes
    const int pieces = (a.vocab + E - 1) / E;
    const int p0 = (int)(((long long)pieces * rank) >> a.size_shift), p1 = (int)(((long long)pieces * (rank + 1)) >> a.size_shift);
    const int first = p0 * E, n = max(0, min(a.vocab, p1 * E) - first);
    const T* row = whole + first;
    if (threadIdx.x == 0) { s_bad = 0; s_bound = 0; }
    __syncthreads();

    float m = -INFINITY;                               // the warp's
    double sum_s = 0.0, sum_t = 0.0;
    bool bad = false;
    float lane_top = -INFINITY;
    int steps = 0;
    unsigned long long* list = s_list[warp];           // the warp's candidates
    int listed = 0;
    unsigned long long last = 0;                       // what a candidate has to exceed: the top-th of the list when it was cut
    const int count = p1 - p0;                         // pieces
    constexpr int U = Chunk<T>::U;
    // what the row's last step needs is under way from here on
    float asked = __int_as_float(0x7fffffff);
    if (rank == 0 && threadIdx.x == 0 && a.logprob) {
        const int64_t tok = a.tokens[r];
        if (tok >= 0 && tok < a.vocab) asked = elem_f(whole[tok]);
    }
    Chunk<T> next;
    if (count > 0) next.load(row, (int)threadIdx.x, n, a.vec);
    for (int base = 0; base < count; base += kThreads * U) {
        float x[kChunkElems];
        const int piece0 = base + (int)threadIdx.x;
        next.values(x);
        if (base + kThreads * U < count) next.load(row, piece0 + kThreads * U, n, a.vec);
        float top = x[0];
#pragma unroll
        for (int e = 1; e < kChunkElems; e++) top = max_nan(top, x[e]);
        if (!(top < INFINITY)) bad = true;
        if (__any_sync(0xffffffffu, top > m)) {
            const float now = warp_max(fmaxf(top, m));
            if (m != -INFINITY) {
                const float dm = fmaxf(m - now, kLeastExponent);
                const double f = expf(dm);
                sum_t = f * (sum_t + (double)dm * sum_s);
                sum_s = f * sum_s;
            }
            m = now;
        }
        if (m != -INFINITY) {
            float2 s = make_float2(0.0f, 0.0f), t = s;
            const float2 less = make_float2(-m, -m), log2e = make_float2(1.44269504088896f, 1.44269504088896f);
#pragma unroll
            for (int e = 0; e < kChunkElems; e += 2) {
                float2 d = add2(make_float2(x[e], x[e + 1]), less);
                d.x = fmaxf(d.x, kLeastExponent);
                d.y = fmaxf(d.y, kLeastExponent);
                const float2 y = mul2(d, log2e);
                const float2 p = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                s = add2(s, p);
                t = fma2(p, d, t);
            }
            sum_s += (double)(s.x + s.y);
            sum_t += (double)(t.x + t.y);
        }
        if (TOP) {
            // after 1, 2, 4, ... steps the bound is the top-th largest of the maxima so far of groups of four lanes; a warp that is behind has smaller ones there
            lane_top = fmaxf(lane_top, top);
            if ((steps & (steps + 1)) == 0) {
                uint32_t o = order_of(lane_top);
                o = max(o, __shfl_xor_sync(0xffffffffu, o, 1));
                o = max(o, __shfl_xor_sync(0xffffffffu, o, 2));
                if ((lane & 3) == 0) s_top[threadIdx.x >> 2] = o;
                if (steps == 0) __syncthreads();
                else __syncwarp();
                // at first every warp finds it, for itself; then one of them, for all
                if (steps == 0 || warp == (__popc(steps) & (kWarps - 1))) {
                    // what the other warps go on writing is copied first: compared with later maxima, none of the earlier ones may be left
                    const uint32_t v0 = *(volatile uint32_t*)&s_top[lane], v1 = *(volatile uint32_t*)&s_top[32 + lane];
                    uint32_t* const seen = s_seen[warp];
                    seen[lane] = v0;
                    seen[32 + lane] = v1;
                    __syncwarp();
                    int above0 = 0, above1 = 0;
#pragma unroll
                    for (int k = 0; k < kGroups; k += 4) {
                        const uint4 u = *reinterpret_cast<const uint4*>(&seen[k]);
                        above0 += (u.x > v0) + (u.y > v0) + (u.z > v0) + (u.w > v0);
                        above1 += (u.x > v1) + (u.y > v1) + (u.z > v1) + (u.w > v1);
                    }
                    // equal ones have equal counts
                    const uint32_t kth = __reduce_min_sync(0xffffffffu, min(above0 < a.top ? v0 : 0xffffffffu, above1 < a.top ? v1 : 0xffffffffu));
                    if (lane == 0) atomicMax(&s_bound, kth);
                    __syncwarp();
                }
            }
            steps++;
            const float bound = value_of(*(volatile uint32_t*)&s_bound);
            if (__any_sync(0xffffffffu, top >= bound)) {
                int mine = 0;
#pragma unroll
                for (int e = 0; e < kChunkElems; e++) mine += x[e] >= bound && (piece0 + (e / E) * kThreads) * E + e % E < n;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                const int more = __shfl_sync(0xffffffffu, upto, 31);
                if (listed + more <= kList) {
                    int to = listed + upto - mine;
                    if (mine) {
#pragma unroll
                        for (int e = 0; e < kChunkElems; e++)
                            if (x[e] >= bound && (piece0 + (e / E) * kThreads) * E + e % E < n) list[to++] = key_of(x[e], first + (piece0 + (e / E) * kThreads) * E + e % E);
                    }
                    listed += more;
                } else {
                    // more than the list has room for (many equal logits): one logit of every lane at a time, and only what beats the list's last
#pragma unroll
                    for (int e = 0; e < kChunkElems; e++) {
                        const int at = (piece0 + (e / E) * kThreads) * E + e % E;
                        const unsigned long long key = x[e] >= bound && at < n ? key_of(x[e], first + at) : 0ull;
                        unsigned who = __ballot_sync(0xffffffffu, key > last);
                        if (who) {
                            if (listed > kList - 32) {
                                last = cut_list(list, listed, a.top, &s_bound);
                                listed = min(listed, a.top);
                                who = __ballot_sync(0xffffffffu, key > last);
                            }
                            if (key > last) list[listed + __popc(who & ((1u << lane) - 1))] = key;
                            listed += __popc(who);
                        }
                    }
                }
            }
        }
    }

    // the block's part
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum_s += __shfl_xor_sync(0xffffffffu, sum_s, o);
        sum_t += __shfl_xor_sync(0xffffffffu, sum_t, o);
    }
    const Sums mine{m, sum_s, sum_t};
    if (bad) s_bad = 1;
    if (lane == 0) warp_sums[warp] = mine;
    if (TOP) {
        __syncthreads();  // the bound is the block's last
        const uint32_t bound = s_bound;
        int kept = 0;
#pragma unroll
        for (int k = 0; k < kList; k += 32) {
            const unsigned long long key = k + lane < listed ? list[k + lane] : 0ull;
            const bool keep = key != 0ull && (uint32_t)(key >> 32) >= bound;
            const unsigned who = __ballot_sync(0xffffffffu, keep);
            if (keep) list[kept + __popc(who & ((1u << lane) - 1))] = key;
            kept += __popc(who);
            __syncwarp();
        }
        listed = kept;
        if (lane == 0) s_count[warp] = listed;
        __syncthreads();
        int all = 0, before = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) all += s_count[w];
        if (all > kThreads) {  // cut the lists first: `top` of each at most
            if (listed > a.top) {
                (void)cut_list(list, listed, a.top, &s_bound);
                listed = a.top;
            }
            __syncthreads();
            if (lane == 0) s_count[warp] = listed;
            __syncthreads();
            all = 0;
#pragma unroll
            for (int w = 0; w < kWarps; w++) all += s_count[w];
        }
#pragma unroll
        for (int w = 0; w < kWarps; w++) before += w < warp ? s_count[w] : 0;
        __syncwarp();
        for (int k = lane; k < listed; k += 32) s_keys[before + k] = list[k];
        if (threadIdx.x < a.top) part.keys[threadIdx.x] = 0ull;
        __syncthreads();
        if ((int)threadIdx.x < all) {
            const unsigned long long key = s_keys[threadIdx.x];
            int above = 0;
#pragma unroll 4
            for (int k = 0; k < all; k++) above += s_keys[k] > key;
            if (above < a.top) part.keys[above] = key;
        }
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        const Sums sums = join_lanes(lane < kWarps ? warp_sums[lane] : Sums{-INFINITY, 0.0, 0.0});
        if (lane == 0) {
            part.sums = sums;
            part.bad = s_bad;
        }
    }
    // the cluster's first block joins the parts
    cluster.sync();
    if (rank == 0 && (TOP || warp == 0)) {
        const BlockPart* p = cluster.map_shared_rank(&part, min(lane, size - 1));
        const Sums all = join_lanes(lane < size ? p->sums : Sums{-INFINITY, 0.0, 0.0});
        const bool any_bad = __any_sync(0xffffffffu, p->bad != 0);
        const float nan = __int_as_float(0x7fffffff);
        const bool empty = all.m == -INFINITY;
        // log S to f32: near 1 by way of S - 1
        const float ls = empty ? 0.0f : all.s < 1.5 ? log1pf((float)(all.s - 1.0)) : logf((float)all.s);
        if (threadIdx.x == 0) {
            if (a.entropy) a.entropy[r] = any_bad ? nan : empty ? 0.0f : ls - (float)all.t / (float)all.s;
            if (a.logprob) {
                a.logprob[r] = any_bad || isnan(asked) ? nan : empty ? -INFINITY : (asked - all.m) - ls;
            }
        }
        if (TOP) {
            const int c = size * a.top;
            if ((int)threadIdx.x < c) s_keys[threadIdx.x] = cluster.map_shared_rank(&part, threadIdx.x / a.top)->keys[threadIdx.x % a.top];
            __syncthreads();
            if ((int)threadIdx.x < c) {
                const unsigned long long key = s_keys[threadIdx.x];
                int above = 0;
#pragma unroll 4
                for (int k = 0; k < c; k++) above += s_keys[k] > key || (s_keys[k] == key && k < (int)threadIdx.x);  // empty places are equal
                if (above < a.top) {
                    a.top_logprob[r * a.top + above] = any_bad ? nan : empty ? -INFINITY : (value_of((uint32_t)(key >> 32)) - all.m) - ls;
                    a.top_id[r * a.top + above] = any_bad ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
                }
            }
        }
    }
    if (size > 1) cluster.sync();  // no block leaves while another reads its part
}

template <typename T>
int32_t logprobs_as(LogprobArgs a, int rows, cudaStream_t s) {
    a.vec = rows_aligned(a.x, rows > 1 ? a.stride : 0, sizeof(T), 16);
    // as few blocks to a row as give every SM one, since a block's beginning and end take about 5 us: 64 rows of 32,000, 20 alternatives: 17.3, 12.8, 11.9, 15.9 us with 1, 2, 4,
    // 8; 2,048 of 128,256, four: 157 with 1, 188 with 2; one row of 32,000, five: 12.7 with 1, 6.9 with 8
    int size = 1;
    while (size < kMaxCluster && (int64_t)rows * size < sm_count() && a.vocab >= size * kThreads * 8) size *= 2;
    while ((1 << a.size_shift) < size) a.size_shift++;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * size);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (a.top > 0) LC_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, a));
    else LC_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, a));
    return LC_OK;
}

int32_t check_logprobs(const char* call, int64_t rows, int64_t vocab, int64_t stride, const void* x, const void* tokens, int32_t top, const void* logprob,
                       const void* top_logprob, const void* top_id) {
    LC_CHECK(rows >= 0 && rows <= 1 << 26, LC_ERR_INVALID, "%s: rows=%lld (0 .. 2^26)", call, (long long)rows);
    LC_CHECK(vocab > 0 && vocab <= 1 << 30, LC_ERR_INVALID, "%s: vocab=%lld (1 .. 2^30)", call, (long long)vocab);
    LC_CHECK(stride >= vocab, LC_ERR_INVALID, "%s: rows overlap (stride %lld, vocab %lld)", call, (long long)stride, (long long)vocab);
    LC_CHECK(top >= 0 && top <= kMaxTop && top <= vocab, LC_ERR_INVALID, "%s: top=%d (0 .. %d, vocab at most)", call, top, kMaxTop);
    LC_CHECK(rows == 0 || x, LC_ERR_INVALID, "%s: null logits", call);
    LC_CHECK(rows == 0 || !logprob || tokens, LC_ERR_INVALID, "%s: log probabilities of no tokens", call);
    LC_CHECK(rows == 0 || top == 0 || (top_logprob && top_id), LC_ERR_INVALID, "%s: no place for the likeliest tokens", call);
    return LC_OK;
}

}  // namespace

int32_t launch_token_logprobs(uint32_t typ, const void* x, int32_t rows, int32_t vocab, int64_t stride, const int64_t* tokens, int32_t top,
                              float* logprob, float* entropy, float* top_logprob, int64_t* top_id, cudaStream_t s) {
    if (rows == 0) return LC_OK;
    LogprobArgs a{x, tokens, logprob, entropy, top_logprob, top_id, stride, vocab, top, 0, 0};
    if (typ == LC_TYPE_F32) return logprobs_as<float>(a, rows, s);
    if (typ == LC_TYPE_F16) return logprobs_as<__half>(a, rows, s);
    return logprobs_as<__nv_bfloat16>(a, rows, s);
}

int32_t check_token_logprobs(const char* call, size_t rows, size_t vocab, const float* logits, const int64_t* tokens, int32_t top, const float* logprob,
                             const float* top_logprob, const int64_t* top_id) {
    const int64_t v = (int64_t)std::min<size_t>(vocab, (size_t)1 << 40);
    return check_logprobs(call, (int64_t)std::min<size_t>(rows, (size_t)1 << 40), v, v, logits, tokens, top, logprob, top_logprob, top_id);
}

}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_token_logprobs_dev(uint32_t typ, const void* logits_dev, int32_t rows, int32_t vocab, int64_t stride, const int64_t* tokens_dev,
                              int32_t top, float* logprob_dev, float* entropy_dev, float* top_logprob_dev, int64_t* top_id_dev, void* stream_) {
    LC_CHECK(typ == LC_TYPE_F32 || typ == LC_TYPE_F16 || typ == LC_TYPE_BF16, LC_ERR_UNSUPPORTED, "lc_token_logprobs_dev: type %u (f32, f16 and bf16 are taken)", typ);
    LC_TRY(check_logprobs("lc_token_logprobs_dev", rows, vocab, stride, logits_dev, tokens_dev, top, logprob_dev, top_logprob_dev, top_id_dev));
    if (rows == 0) return LC_OK;
    DeviceScope dev;
    LC_TRY(dev.enter(logits_dev, "lc_token_logprobs_dev: logits"));
    return launch_token_logprobs(typ, logits_dev, rows, vocab, stride, tokens_dev, top, logprob_dev, entropy_dev, top_logprob_dev, top_id_dev, stream_or_own(stream_));
}

}  // extern "C"
