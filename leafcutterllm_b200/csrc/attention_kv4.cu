// Attention over the key/value cache in 4 bits: out = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the slots j up to the row's own.
//
// A warp per row and head: a lane scores a key of 32 at a time, then all lanes add up the values' dims.
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_kv8_attn.cuh"

namespace lc {

namespace {

struct Attn4Args {
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride, lse_stride;
    int typ, heads, group, window;
    float scale;
};
constexpr int kWarps = 4;

__global__ void __launch_bounds__(kWarps * 32) kv4_attention_kernel(Kv4Pool pool, Kv8Seqs seqs, Attn4Args a) {
    __shared__ float qs[kWarps][256];
    if (blockIdx.x == 0) kv8_check_seqs(seqs, pool);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = pool.hd, blocks = hd >> 4;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + warp;
    const int r = (int)(unit / a.heads), h = (int)(unit % a.heads), kvh = h / a.group;
    if (r >= seqs.n_rows) return;
    const RowPlace at = row_place(seqs, pool, r);
    if (at.seq < 0) return;
    const int64_t dst = (int64_t)r * a.out_stride + (int64_t)h * hd;
    float l = 0.0f, m = kNegInf, o[8] = {};
    bool bad = at.slot < 0;
    if (!bad) {
        for (int d = lane; d < hd; d += 32) {
            const int64_t src = (int64_t)r * a.q_stride + (int64_t)h * hd + d;
            qs[warp][d] = a.typ == LC_TYPE_F32 ? ((const float*)a.q)[src] : a.typ == LC_TYPE_F16 ? elem_f(((const __half*)a.q)[src]) : elem_f(((const __nv_bfloat16*)a.q)[src]);
        }
        __syncwarp();
        const int limit = seqs.ctx[at.seq] + at.index, from = a.window > 0 ? max(0, limit - a.window + 1) : 0, mask = (1 << pool.page_shift) - 1;
        const int32_t* table = seqs.table + (size_t)at.seq * seqs.width;
        const float gk = pool.k_scale[kvh], gv = pool.v_scale[kvh];
        for (int key0 = from & ~31; key0 <= limit; key0 += 32) {
            const int key = key0 + lane;
            const bool sees = key >= from && key <= limit;
            const int number = sees ? table[key >> pool.page_shift] : 0;
            const bool held = number >= 0 && number < pool.n_pages;
            if (sees && !held) { bad = true; kv8_raise(seqs, at.seq); }
            const size_t row = (((size_t)(held ? number : 0) * pool.n_kv + kvh) << pool.page_shift) + (key & mask);
            float s = kNegInf;
            if (sees && held) {
                s = 0.0f;
                for (int b = 0; b < blocks; b++) {
                    const uint2 w = *reinterpret_cast<const uint2*>(pool.k + row * (hd >> 1) + 8 * b);
                    float part = 0.0f;
                    for (int e = 0; e < 16; e++) part = fmaf((float)(int)(((e < 8 ? w.x : w.y) >> (4 * (e & 7)) & 15u) - 8u), qs[warp][16 * b + e], part);
                    s = fmaf(part, scale4_f(pool.k_block[row * blocks + b]), s);
                }
                s *= a.scale * gk;
            }
            const float top = fmaxf(m, warp_max(s)), ref = top == kNegInf ? 0.0f : top, corr = expf(m - ref), p = expf(s - ref);
            m = top;
            l = l * corr + warp_sum(p);
            for (int i = 0; i < 8; i++) o[i] *= corr;
            for (int x = 0; x < 32; x++) {
                const float w = __shfl_sync(0xffffffffu, p, x);
                const size_t vrow = __shfl_sync(0xffffffffu, (unsigned long long)row, x);
                if (w == 0.0f) continue;
                for (int i = 0; i < 8; i++) {
                    const int d = lane + 32 * i;
                    if (d < hd) {
                        const int n = (int)((uint8_t)pool.v[vrow * (hd >> 1) + (d >> 1)] >> (4 * (d & 1)) & 15) - 8;
                        o[i] = fmaf(w, (float)n * scale4_f(pool.v_block[vrow * blocks + (d >> 4)]) * gv, o[i]);
                    }
                }
            }
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    if (bad) l = __int_as_float(0x7fffffff);
    for (int i = 0; i < 8; i++) {
        const int d = lane + 32 * i;
        if (d < hd) store1(a.out, dst + d, a.typ, o[i] / l);
    }
    if (a.lse && lane == 0) a.lse[(int64_t)r * a.lse_stride + h] = m + logf(l);
}

}  // namespace
}  // namespace lc

using namespace lc;

namespace {
int32_t check_heads(const char* call, const Kv4Pool& pool, const Kv8Seqs& seqs, int32_t n_heads) {
    LC_CHECK(n_heads > 0 && n_heads <= 65536 && n_heads % pool.n_kv == 0, LC_ERR_INVALID, "%s: %d heads over %d kv heads", call, n_heads, pool.n_kv);
    LC_CHECK((int64_t)seqs.n_rows * n_heads <= (int64_t)1 << 30, LC_ERR_INVALID, "%s: %d rows of %d heads are too many for one call", call, seqs.n_rows, n_heads);
    return LC_OK;
}
}  // namespace

extern "C" {

int32_t lc_attention_kv4_workspace(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, int32_t n_heads, size_t* out_bytes) {
    const char* call = "lc_attention_kv4_workspace";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_CHECK(out_bytes, LC_ERR_INVALID, "%s: null output", call);
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    LC_TRY(check_heads(call, pool, seqs, n_heads));
    *out_bytes = 16;
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
    LC_CHECK(workspace_dev && workspace_bytes >= 16 && (uintptr_t)workspace_dev % 16 == 0, LC_ERR_INVALID, "%s: needs a workspace of 16 bytes, 16-byte aligned (got %zu)", call, workspace_bytes);
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)pool.hd);
    const Attn4Args a{q_dev, out_dev, lse_dev, q_stride, out_stride, lse_stride, (int)typ, n_heads, n_heads / pool.n_kv, std::min(window, 1 << 30), scale};
    const int64_t units = (int64_t)n_rows * n_heads;
    kv4_attention_kernel<<<(unsigned)((units + kWarps - 1) / kWarps), kWarps * 32, 0, stream_or_own(stream_)>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}

}  // extern "C"
