// What weight a call's rows gave the cached keys: mass[sequence][kv head][slot] += sum over rows and heads of the group of exp(scale q . k - lse).
//
// A thread per key: every sum is one thread's, in the order of rows and heads, so that nothing depends on timing.
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

struct WeightArgs {
    const void* q;
    const float* lse;
    float* mass;
    int64_t q_stride, lse_stride, mass_stride, mass_head_stride;
    int typ, group, window, capacity;
    float scale;
};
constexpr int kThreads = 128;

// grid: (chunks of 128 keys, sequences, kv heads)
__global__ void __launch_bounds__(kThreads) kv4_weights_kernel(Kv4Pool pool, Kv8Seqs seqs, WeightArgs a) {
    __shared__ float qs[256];
    const int i = blockIdx.y, kvh = blockIdx.z, hd = pool.hd, blocks = hd >> 4;
    int first, n;
    if (!kv8_span(seqs, i, first, n)) { if (threadIdx.x == 0) kv8_raise(seqs, i); return; }
    if (n == 0) return;
    const int ctx = seqs.ctx[i];
    if (!kv8_in_table(seqs, pool, ctx, n) || ctx + n > a.capacity) { if (threadIdx.x == 0) kv8_raise(seqs, i); return; }
    const int key = blockIdx.x * kThreads + threadIdx.x;
    if (blockIdx.x * kThreads >= ctx + n) return;
    const bool here = key < ctx + n && (a.window == 0 || key > ctx - a.window);
    const int number = here ? seqs.table[(size_t)i * seqs.width + (key >> pool.page_shift)] : -1;
    const bool held = number >= 0 && number < pool.n_pages;
    if (here && !held) kv8_raise(seqs, i);
    const size_t row = (((size_t)(held ? number : 0) * pool.n_kv + kvh) << pool.page_shift) + (key & ((1 << pool.page_shift) - 1));
    float sum = 0.0f;
    for (int j = 0; j < n; j++)
        for (int g = 0; g < a.group; g++) {
            const int h = kvh * a.group + g;
            __syncthreads();
            for (int d = threadIdx.x; d < hd; d += kThreads) {
                const int64_t src = (int64_t)(first + j) * a.q_stride + (int64_t)h * hd + d;
                qs[d] = a.typ == LC_TYPE_F32 ? ((const float*)a.q)[src] : a.typ == LC_TYPE_F16 ? elem_f(((const __half*)a.q)[src]) : elem_f(((const __nv_bfloat16*)a.q)[src]);
            }
            __syncthreads();
            const float lse = a.lse[(int64_t)(first + j) * a.lse_stride + h];
            if (!held || key > ctx + j || (a.window > 0 && key <= ctx + j - a.window) || !(fabsf(lse) < INFINITY)) continue;
            float s = 0.0f;
            for (int b = 0; b < blocks; b++) {
                const uint2 w = *reinterpret_cast<const uint2*>(pool.k + row * (hd >> 1) + 8 * b);
                float part = 0.0f;
                for (int e = 0; e < 16; e++) part = fmaf((float)(int)(((e < 8 ? w.x : w.y) >> (4 * (e & 7)) & 15u) - 8u), qs[16 * b + e], part);
                s = fmaf(part, scale4_f(pool.k_block[row * blocks + b]), s);
            }
            sum += expf(s * (a.scale * pool.k_scale[kvh]) - lse);
        }
    if (held) a.mass[(int64_t)i * a.mass_stride + (int64_t)kvh * a.mass_head_stride + key] += sum;
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
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(q_dev && lse_dev && mass_dev, LC_ERR_INVALID, "%s: null queries, lse or sums", call);
    LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && lse_stride >= n_heads, LC_ERR_INVALID, "%s: rows overlap", call);
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    const WeightArgs a{q_dev, lse_dev, mass_dev, q_stride, lse_stride, mass_stride, mass_head_stride, (int)typ, n_heads / pool.n_kv, std::min(window, 1 << 30), capacity, scale};
    const int64_t keys = std::min<int64_t>((int64_t)seqs.width << pool.page_shift, capacity);
    kv4_weights_kernel<<<dim3((unsigned)std::max<int64_t>(1, (keys + kThreads - 1) / kThreads), (unsigned)seqs.n_seqs, (unsigned)pool.n_kv), kThreads, 0, stream_or_own(stream_)>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
