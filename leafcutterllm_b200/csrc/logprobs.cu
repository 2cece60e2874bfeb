// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits, in one pass over them.
//
// With m the row's maximum, d = x - m, S = sum e^d and T = sum e^d d:   log p(x) = d - log S,   entropy = log S - T / S.
// Every thread keeps a running m, S and T.  Sixteen logits at a time: their f32 sums are added to S and T in 64 bits, which a row of one
// near-certain token needs (log S ~ 1e-3 is then S - 1).  A later maximum m' turns (S, T) into (f S, f (T + (m - m') S)), f = e^(m - m').
//
// The best `top` are kept per warp, lane i holding the i-th as a key (logit in the order of whole numbers, then the lower index).  A logit below
// the block's bound cannot be among them; the bound is the largest of the warps' last keys, and to begin with the top-th largest of
// the lanes' maxima of the first sixteen.  Only logits above it take the way through the list.
//
// A row goes to a cluster of 1, 2, 4 or 8 blocks, which join over distributed shared memory: one launch, no workspace.
#include <cooperative_groups.h>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include <algorithm>

namespace lc {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, kChunkElems = 16, kMaxCluster = 8, kMaxTop = 32;

struct Sums {
    float m;
    double s, t;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    if (b.m == -INFINITY) return a;
    if (a.m == -INFINITY) return b;
    const float m = fmaxf(a.m, b.m);
    const float da = a.m - m, db = b.m - m;
    const double fa = expf(da), fb = expf(db);
    return Sums{m, fa * a.s + fb * b.s, fa * (a.t + (double)da * a.s) + fb * (b.t + (double)db * b.s)};
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
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
};

// what a block leaves for its cluster
struct BlockPart {
    Sums sums;
    int bad;
    unsigned long long keys[kMaxTop];
};

// Sixteen logits of a thread: `per` pieces of 16 bytes, blockDim apart.  Places behind the end give minus infinity.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int piece0, int n, bool vec, float (&x)[kChunkElems]) {
    constexpr int E = 16 / sizeof(T), U = kChunkElems / E;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int at = (piece0 + u * kThreads) * E;
        if (vec && at + E <= n) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(row + at));
            __align__(16) T t[E];
            *reinterpret_cast<uint4*>(t) = w;
#pragma unroll
            for (int e = 0; e < E; e++) x[u * E + e] = elem_f(t[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) x[u * E + e] = at + e < n ? elem_f(row[at + e]) : -INFINITY;
        }
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(LogprobArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ BlockPart part;
    __shared__ Sums warp_sums[kWarps];
    __shared__ int s_bad;
    __shared__ uint32_t s_bound;                       // order of a value that at least `top` logits reach
    __shared__ unsigned long long s_keys[kMaxCluster > kWarps ? kMaxCluster * kMaxTop : kWarps * kMaxTop];
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t r = blockIdx.x / size;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* whole = (const T*)a.x + r * a.stride;
    // this block's slice, in pieces of 16 bytes
    const int pieces = (a.vocab + E - 1) / E;
    const int p0 = (int)((long long)pieces * rank / size), p1 = (int)((long long)pieces * (rank + 1) / size);
    const int first = p0 * E, n = max(0, min(a.vocab, p1 * E) - first);
    const T* row = whole + first;
    if (threadIdx.x == 0) { s_bad = 0; s_bound = 0; }
    __syncthreads();

    Sums mine{-INFINITY, 0.0, 0.0};
    bool bad = false;
    unsigned long long best = 0;                       // lane i: the warp's i-th best key
    const int count = p1 - p0;                         // pieces
    constexpr int U = kChunkElems / E;
    for (int base = 0; base < count; base += kThreads * U) {
        float x[kChunkElems];
        const int piece0 = base + (int)threadIdx.x;
        load_chunk<T>(row, piece0, n, a.vec, x);
        float top = x[0];
#pragma unroll
        for (int e = 1; e < kChunkElems; e++) top = max_nan(top, x[e]);
        if (!(top < INFINITY)) bad = true;
        if (top > mine.m) {
            if (mine.m != -INFINITY) {
                const float dm = mine.m - top;
                const double f = expf(dm);
                mine.t = f * (mine.t + (double)dm * mine.s);
                mine.s = f * mine.s;
            }
            mine.m = top;
        }
        if (mine.m != -INFINITY) {
            float s = 0.0f, t = 0.0f;
#pragma unroll
            for (int e = 0; e < kChunkElems; e++) {
                const float d = fmaxf(x[e] - mine.m, -200.0f);  // e^-200 is 0 here; keeps 0 * -inf out
                const float p = exp2_fast(d * 1.44269504088896f);
                s += p;
                t = fmaf(p, d, t);
            }
            mine.s += (double)s;
            mine.t += (double)t;
        }
        if (TOP) {
            if (base == 0) {
                // a first bound: the top-th largest of the lanes' maxima
                uint32_t o = order_of(top);
                int above = 0;
#pragma unroll
                for (int k = 1; k < 32; k++) {
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, o, k);
                    above += other > o || (other == o && (lane ^ k) < lane);
                }
                if (above == a.top - 1) atomicMax(&s_bound, o);
                __syncthreads();
            }
            float bound = value_of(*(volatile uint32_t*)&s_bound);
            if (__any_sync(0xffffffffu, top >= bound)) {
                unsigned long long last = __shfl_sync(0xffffffffu, best, a.top - 1);
#pragma unroll
                for (int e = 0; e < kChunkElems; e++) {
                    const int at = (piece0 + (e / E) * kThreads) * E + e % E;
                    unsigned long long key = x[e] >= bound && at < n ? key_of(x[e], first + at) : 0ull;
                    unsigned who = __ballot_sync(0xffffffffu, key > last);
                    while (who) {
                        const int src = __ffs(who) - 1;
                        who &= who - 1;
                        const unsigned long long in = __shfl_sync(0xffffffffu, key, src);
                        if (in > last) {
                            const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
                            if (best < in) best = lane == 0 || up > in ? in : up;
                            last = __shfl_sync(0xffffffffu, best, a.top - 1);
                        }
                    }
                }
                if (last != 0 && lane == 0 && (uint32_t)(last >> 32) > *(volatile uint32_t*)&s_bound) atomicMax(&s_bound, (uint32_t)(last >> 32));
            }
        }
    }

    // the block's part
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums other;
        other.m = __shfl_xor_sync(0xffffffffu, mine.m, o);
        other.s = __shfl_xor_sync(0xffffffffu, mine.s, o);
        other.t = __shfl_xor_sync(0xffffffffu, mine.t, o);
        // the same order on both sides
        mine = (lane & o) == 0 ? join(mine, other) : join(other, mine);
    }
    if (bad) s_bad = 1;
    if (lane == 0) warp_sums[warp] = mine;
    if (TOP && lane < a.top) s_keys[warp * a.top + lane] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        Sums all = warp_sums[0];
        for (int w = 1; w < kWarps; w++) all = join(all, warp_sums[w]);
        part.sums = all;
        part.bad = s_bad;
    }
    if (TOP) {
        const int c = kWarps * a.top;
        if (threadIdx.x < c) {  // 8 warps x 32 at most: as many as threads
            const unsigned long long key = s_keys[threadIdx.x];
            int above = 0;
            for (int k = 0; k < c; k++) above += s_keys[k] > key || (s_keys[k] == key && k < (int)threadIdx.x);  // empty places are equal
            if (above < a.top) part.keys[above] = key;
        }
    }
    cluster.sync();
    if (rank == 0) {
        if (TOP) {
            for (int k = threadIdx.x; k < size * a.top; k += kThreads) s_keys[k] = cluster.map_shared_rank(&part, k / a.top)->keys[k % a.top];
        }
        Sums all = part.sums;
        int any_bad = part.bad;
        for (int b = 1; b < size; b++) {
            const BlockPart* p = cluster.map_shared_rank(&part, b);
            all = join(all, p->sums);
            any_bad |= p->bad;
        }
        __syncthreads();
        const float nan = __int_as_float(0x7fffffff);
        const bool empty = all.m == -INFINITY;
        const double ls = empty ? 0.0 : log(all.s);
        if (threadIdx.x == 0) {
            if (a.entropy) a.entropy[r] = any_bad ? nan : empty ? 0.0f : (float)(ls - all.t / all.s);
            if (a.logprob) {
                const int64_t tok = a.tokens[r];
                float y = nan;
                if (!any_bad && tok >= 0 && tok < a.vocab) y = empty ? -INFINITY : (float)((double)elem_f(whole[tok]) - (double)all.m - ls);
                a.logprob[r] = y;
            }
        }
        if (TOP) {
            const int c = size * a.top;
            if (threadIdx.x < c) {
                const unsigned long long key = s_keys[threadIdx.x];
                int above = 0;
                for (int k = 0; k < c; k++) above += s_keys[k] > key || (s_keys[k] == key && k < (int)threadIdx.x);
                if (above < a.top) {
                    const float v = value_of((uint32_t)(key >> 32));
                    a.top_logprob[r * a.top + above] = any_bad ? nan : empty ? -INFINITY : (float)((double)v - (double)all.m - ls);
                    a.top_id[r * a.top + above] = any_bad ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
                }
            }
        }
    }
    cluster.sync();  // no block leaves while another reads its part
}

template <typename T>
int32_t logprobs_as(LogprobArgs a, int rows, cudaStream_t s) {
    a.vec = rows_aligned(a.x, rows > 1 ? a.stride : 0, sizeof(T), 16);
    // a cluster is as large as leaves two blocks an SM, and its blocks a chunk each
    int size = 1;
    while (size < kMaxCluster && (int64_t)rows * size < 2 * sm_count() && a.vocab >= 2 * size * kThreads * kChunkElems / 4) size *= 2;
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
    LogprobArgs a{x, tokens, logprob, entropy, top_logprob, top_id, stride, vocab, top, 0};
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
