// The key/value cache in 4 bits: appending rows (with the position rotation on the way), reading rows back.
//
// A row's 16 dims x have the block scale s = e4m3(max |x| / (7 g)) and the integers n = rint(x / (s g)), all as if in 64 bits, so that the cache's bytes depend on the definition alone.
// Rotations are in 64 bits (the GPU has half as many such units as of f32); quotients are in f32, 2^-22 off, and what lies too near a border between two integers or two scales
// is compared with the border in 64 bits, where both are exact.  A thread has the 16 dims of one block and loads the 16 that they are paired with, so rows pass once.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include "lc_kernels.h"
#include "lc_kv4.cuh"
#include "lc_rope.cuh"

namespace lc {

int32_t kv4_check(const char* call, const lc_kv4_cache* c, const lc_kv8_rows* r, uint32_t typ, int32_t n_rows, Kv4Pool* view, Kv8Seqs* seqs) {
    LC_CHECK(c && r, LC_ERR_INVALID, "%s: null cache or rows", call);
    LC_CHECK(c->k_block_dev && c->v_block_dev, LC_ERR_INVALID, "%s: null pointer in the cache", call);
    LC_CHECK(((uintptr_t)c->k_block_dev | (uintptr_t)c->v_block_dev) % 16 == 0, LC_ERR_INVALID, "%s: the block scales must be 16-byte aligned", call);
    const lc_kv8_cache as8{c->k_dev, c->v_dev, const_cast<float*>(c->k_scale_dev), const_cast<float*>(c->v_scale_dev), c->n_pages, c->n_kv_heads, c->page_tokens, c->head_dim};
    LC_TRY(kv8_check(call, &as8, r, typ, n_rows, view, seqs));
    view->k_block = c->k_block_dev;
    view->v_block = c->v_block_dev;
    return LC_OK;
}

namespace {

struct Append4Args {
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    int64_t k_stride, v_stride, q_stride, qo_stride;
    const int64_t* positions;     // per sequence, or null: the slots
    const uint64_t* turns;
    int n_heads, half;            // half = rot_dim / 2
    int rows, kv_slices;          // rows of a block; blocks of them for the keys and values, the others are the queries'
    bool interleaved;
    double magnitude;
};
constexpr int kAppendThreads = 256, kAppendRows = 8;

// Sixteen numbers of at most 4 bits each, and their scale's byte.
struct Block4 {
    uint2 words;
    uint32_t scale;
};
// y: the numbers in 64 bits (in f32 where these are all there is)
template <typename Y>
__device__ __forceinline__ Block4 quantised(const Y (&y)[16], float g) {
    float x[16], most = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        x[e] = (float)y[e];
        if (sizeof(Y) == 8 && isinf(x[e]) && !isinf(y[e])) x[e] = copysignf(FLT_MAX, x[e]);  // two large ones together
        const float a = fabsf(x[e]);
        most = a < INFINITY ? fmaxf(most, a) : most;
    }
    // s: k steps of the numbers of its size, 2^-9 at the least; k = 16 is the next size's 8
    const float want = most * (1.0f / (7.0f * g));
    const int size = min(max((__float_as_int(want) >> 23) - 127, -6), 9);
    const float r = want * __int_as_float((127 + 3 - size) << 23);
    float k = rintf(r);
    if (fabsf(fabsf(r - k) - 0.5f) < 0x1p-15f) {
        double top = 0.0;
#pragma unroll
        for (int e = 0; e < 16; e++) top = fabs((double)y[e]) < (double)INFINITY ? fmax(top, fabs((double)y[e])) : top;
        const float below = rintf(r - 0.5f);
        const double border = ((double)below + 0.5) * (double)__int_as_float((127 + size - 3) << 23) * (7.0 * (double)g);
        k = top > border ? below + 1.0f : top < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));
    }
    const float s = fminf(k * __int_as_float((127 + size - 3) << 23), 448.0f);
    Block4 out;
    out.scale = s >= 0x1p-6f ? (__float_as_uint(s) >> 20) - (120u << 3) : (uint32_t)(s * 512.0f);
    const float inv = s > 0.0f ? 1.0f / (s * g) : 0.0f;
    const double step = (double)s * (double)g;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float a = fabsf(x[e] * inv);
        float n = rintf(a);
        if (fabsf(fabsf(a - n) - 0.5f) < 1e-5f) {
            const float below = rintf(a - 0.5f);
            const double border = ((double)below + 0.5) * step, z = fabs((double)y[e]);
            n = z > border ? below + 1.0f : z < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));
        }
        const int m = a == a ? (int)fminf(n, 7.0f) : 0;
        w[e >> 3] |= (uint32_t)(x[e] < 0.0f ? 8 - m : 8 + m) << (4 * (e & 7));
    }
    out.words = make_uint2(w[0], w[1]);
    return out;
}

// Sixteen elements in a row as f32
template <typename T, bool VEC> __device__ __forceinline__ void load16f(const T* p, float (&v)[16]) {
    if (VEC) {
        __align__(16) T t[16];
#pragma unroll
        for (int u = 0; u < (int)sizeof(T); u++) reinterpret_cast<uint4*>(t)[u] = reinterpret_cast<const uint4*>(p)[u];
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = elem_f(t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = elem_f(p[e]);
    }
}

// Dims d0 .. d0 + 15 of a head of keys, turned.  VEC: they lie on one side of the middle and of the end of the rotated part, and 16-byte accesses are possible.
template <typename T, bool VEC>
__device__ __forceinline__ void turned16(const T* x, int d0, int half, bool interleaved, const double2* row, int n8, double (&y)[16]) {
    float v[16];
    load16f<T, VEC>(x + d0, v);
    if (VEC) {
        if (d0 >= 2 * half) {
#pragma unroll
            for (int e = 0; e < 16; e++) y[e] = v[e];
        } else if (interleaved) {
            const int p8 = d0 >> 4;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const double2 t = row[k * n8 + p8];
                const double a = v[2 * k], b = v[2 * k + 1];
                y[2 * k] = a * t.x - b * t.y;
                y[2 * k + 1] = a * t.y + b * t.x;
            }
        } else {
            const bool second = d0 >= half;
            float w[16];
            load16f<T, VEC>(x + (second ? d0 - half : d0 + half), w);
            const int p8 = (second ? d0 - half : d0) >> 3;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const double2 t = row[(e & 7) * n8 + p8 + (e >> 3)];
                const double own = v[e], other = w[e];
                y[e] = own * t.x + other * (second ? t.y : -t.y);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int d = d0 + e;
            y[e] = v[e];
            if (d < 2 * half) {
                const int p = interleaved ? d >> 1 : d < half ? d : d - half;
                const bool second = interleaved ? d & 1 : d >= half;
                const double other = elem_f(x[interleaved ? d ^ 1 : second ? d - half : d + half]);
                const double2 t = row[turn_place(p, n8)];
                y[e] = y[e] * t.x + other * (second ? t.y : -t.y);
            }
        }
    }
}

// grid: (groups of rows, slices of kv heads and then of query heads)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) kv4_append_kernel(Kv4Pool pool, Kv8Seqs seqs, Append4Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ RowPlace place[kAppendRows];
    if (blockIdx.x == 0 && blockIdx.y == 0) kv8_check_seqs(seqs, pool);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * a.rows, rows = min(a.rows, seqs.n_rows - row0);
    if (warp < rows) {
        const RowPlace at = row_place(seqs, pool, row0 + warp);
        if (lane == 0) {
            place[warp] = at;
            if (at.seq >= 0 && at.page < 0) kv8_raise(seqs, at.seq);
        }
    }
    __syncthreads();
    const bool kv = (int)blockIdx.y < a.kv_slices;
    const int slices = kv ? a.kv_slices : gridDim.y - a.kv_slices, sl = kv ? blockIdx.y : blockIdx.y - a.kv_slices, heads = kv ? pool.n_kv : a.n_heads;
    const int h0 = heads * sl / slices, mine = heads * (sl + 1) / slices - h0;
    const int hd = pool.hd, half = a.half, n8 = (half + 7) >> 3;
    for (int e = tid; e < rows * half; e += kAppendThreads) {
        const int j = e / half, p = e - j * half;
        const RowPlace& at = place[j];
        if (at.seq < 0) continue;
        double2 t = turn_of(a.turns[p], (a.positions ? a.positions[at.seq] : (int64_t)seqs.ctx[at.seq]) + at.index);
        t.x *= a.magnitude;
        t.y *= a.magnitude;
        const int to = j * 8 * n8 + turn_place(p, n8);
        if (kv) reinterpret_cast<double2*>(smem)[to] = t;
        else put_turn(reinterpret_cast<typename TurnEntry<T>::type*>(smem)[to], t);
    }
    __syncthreads();
    if (kv) {
        // blocks of 16 dims: of the rows' keys, then of their values
        const int blocks = hd >> 4, per_row = mine * blocks, all = rows * per_row;
        for (int e = tid; e < 2 * all; e += kAppendThreads) {
            const bool is_k = e < all;
            const int f = is_k ? e : e - all, j = f / per_row, g = f - j * per_row, h = h0 + g / blocks, b = g % blocks;
            const RowPlace& at = place[j];
            if (at.page < 0) continue;
            const T* x = (const T*)(is_k ? a.k : a.v) + (int64_t)(row0 + j) * (is_k ? a.k_stride : a.v_stride) + (int64_t)h * hd;
            Block4 out;
            if (is_k && half > 0) {
                double y[16];
                turned16<T, VEC>(x, 16 * b, half, a.interleaved, reinterpret_cast<const double2*>(smem) + j * 8 * n8, n8, y);
                out = quantised(y, pool.k_scale[h]);
            } else {
                float y[16];
                load16f<T, VEC>(x + 16 * b, y);
                out = quantised(y, (is_k ? pool.k_scale : pool.v_scale)[h]);
            }
            const size_t row = (((size_t)at.page * pool.n_kv + h) << pool.page_shift) + at.slot;
            *reinterpret_cast<uint2*>((is_k ? pool.k : pool.v) + row * (hd >> 1) + 8 * b) = out.words;
            (is_k ? pool.k_block : pool.v_block)[row * blocks + b] = (uint8_t)out.scale;
        }
    } else {
        using Entry = typename TurnEntry<T>::type;
        const int items = VEC ? turn_items(hd, half) : hd - half, per_row = mine * items;
        for (int e = tid; e < rows * per_row; e += kAppendThreads) {
            const int j = e / per_row, g = e - j * per_row, h = h0 + g / items, i = g % items;
            const RowPlace& at = place[j];
            if (at.seq < 0 || at.slot < 0) continue;
            const T* in = (const T*)a.q + (int64_t)(row0 + j) * a.q_stride + (int64_t)h * hd;
            T* out = (T*)a.q_out + (int64_t)(row0 + j) * a.qo_stride + (int64_t)h * hd;
            const Entry* row = reinterpret_cast<const Entry*>(smem) + j * 8 * n8;
            if constexpr (VEC) turn_item(in, out, i, half, a.interleaved, row, n8);
            else turn_item_plain(in, out, i, half, a.interleaved, row, n8);
        }
    }
}

struct Read4Args {
    void* k;
    void* v;
    int64_t k_stride, v_stride;
    int rows;
    bool vec;  // whether 16 elements are stored in 16-byte pieces
};
// A block takes a few rows, a thread 16 dims of them at a time: of the keys, then of the values.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv4_read_kernel(Kv4Pool pool, Kv8Seqs seqs, Read4Args a) {
    __shared__ RowPlace place[kAppendRows];
    if (blockIdx.x == 0 && blockIdx.y == 0) kv8_check_seqs(seqs, pool);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * a.rows, rows = min(a.rows, seqs.n_rows - row0);
    if (warp < rows) {
        const RowPlace at = row_place(seqs, pool, row0 + warp);
        if (lane == 0) {
            place[warp] = at;
            if (at.seq >= 0 && at.page < 0) kv8_raise(seqs, at.seq);
        }
    }
    __syncthreads();
    const int h0 = pool.n_kv * blockIdx.y / gridDim.y, mine = pool.n_kv * (blockIdx.y + 1) / gridDim.y - h0;
    const int blocks = pool.hd >> 4, per_row = mine * blocks, all = rows * per_row;
    for (int e = tid; e < 2 * all; e += kAppendThreads) {
        const bool is_k = e < all;
        T* out = (T*)(is_k ? a.k : a.v);
        const int f = is_k ? e : e - all, j = f / per_row, g = f - j * per_row, h = h0 + g / blocks, b = g % blocks;
        const RowPlace& at = place[j];
        if (at.seq < 0 || !out) continue;
        float scale = __int_as_float(0x7fffffff), head = 1.0f;
        uint2 w = make_uint2(0, 0);
        if (at.page >= 0) {
            const size_t row = (((size_t)at.page * pool.n_kv + h) << pool.page_shift) + at.slot;
            w = *reinterpret_cast<const uint2*>((is_k ? pool.k : pool.v) + row * (pool.hd >> 1) + 8 * b);
            scale = scale4_f((is_k ? pool.k_block : pool.v_block)[row * blocks + b]);
            head = (is_k ? pool.k_scale : pool.v_scale)[h];
        }
        __align__(16) T t[16];
#pragma unroll
        for (int x = 0; x < 16; x++) t[x] = to_elem<T>((float)(int)(((x < 8 ? w.x : w.y) >> (4 * (x & 7)) & 15u) - 8u) * scale * head);
        out += (int64_t)(row0 + j) * (is_k ? a.k_stride : a.v_stride) + (int64_t)h * pool.hd + 16 * b;
        if (a.vec) {
#pragma unroll
            for (int x = 0; x < (int)sizeof(T); x++) reinterpret_cast<uint4*>(out)[x] = reinterpret_cast<const uint4*>(t)[x];
        } else {
#pragma unroll
            for (int x = 0; x < 16; x++) out[x] = t[x];
        }
    }
}

// Rows of a block: as many as leave two blocks for each SM; few rows: their heads over several blocks, of at least `least` heads
struct RowGrid {
    int rows, groups;
};
RowGrid row_grid(int n_rows) {
    RowGrid g;
    g.rows = std::max(1, std::min(kAppendRows, n_rows / (2 * sm_count())));
    g.groups = (n_rows + g.rows - 1) / g.rows;
    return g;
}
int slices_of(int groups, int heads, int least) { return std::max(1, std::min({(2 * sm_count() + groups - 1) / groups, (heads + least - 1) / least, 64})); }

template <typename T>
int32_t append4_as(const Kv4Pool& pool, const Kv8Seqs& seqs, Append4Args a, cudaStream_t s) {
    const RowGrid grid = row_grid(seqs.n_rows);
    a.rows = grid.rows;
    a.kv_slices = slices_of(grid.groups, pool.n_kv, 4);
    const int slices = a.kv_slices + (a.q ? slices_of(grid.groups, a.n_heads, 4) : 0);
    const bool vec = a.half % (a.interleaved ? 8 : 16) == 0 && rows_aligned(a.k, a.k_stride, sizeof(T), 16) && rows_aligned(a.v, a.v_stride, sizeof(T), 16) &&
                     (!a.q || (rows_aligned(a.q, a.q_stride, sizeof(T), 16) && rows_aligned(a.q_out, a.qo_stride, sizeof(T), 16)));
    const size_t smem = (size_t)a.rows * ((a.half + 7) / 8 * 8) * sizeof(double2);
    const auto kern = vec ? kv4_append_kernel<T, true> : kv4_append_kernel<T, false>;
    kern<<<dim3((unsigned)grid.groups, (unsigned)slices), kAppendThreads, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
template <typename T>
int32_t read4_as(const Kv4Pool& pool, const Kv8Seqs& seqs, Read4Args a, cudaStream_t s) {
    a.vec = (!a.k || rows_aligned(a.k, a.k_stride, sizeof(T), 16)) && (!a.v || rows_aligned(a.v, a.v_stride, sizeof(T), 16));
    const RowGrid grid = row_grid(seqs.n_rows);
    a.rows = grid.rows;
    kv4_read_kernel<T><<<dim3((unsigned)grid.groups, (unsigned)slices_of(grid.groups, pool.n_kv, 4)), kAppendThreads, 0, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_kv4_append_dev(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, const int64_t* positions_dev, const void* k_dev, int64_t k_stride, const void* v_dev,
                          int64_t v_stride, const void* q_dev, int64_t q_stride, void* q_out_dev, int64_t q_out_stride, int32_t n_heads, const uint64_t* turns_dev, int32_t rot_dim, int32_t layout,
                          double magnitude, void* stream_) {
    const char* call = "lc_kv4_append_dev";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    LC_CHECK(rot_dim >= 0 && rot_dim <= pool.hd && rot_dim % 2 == 0, LC_ERR_INVALID, "%s: rot_dim=%d (even, head_dim %d at most)", call, rot_dim, pool.hd);
    LC_CHECK(rot_dim == 0 || turns_dev, LC_ERR_INVALID, "%s: a rotation needs its table", call);
    LC_CHECK(layout == LC_ROPE_HALF || layout == LC_ROPE_INTERLEAVED, LC_ERR_INVALID, "%s: layout=%d", call, layout);
    LC_CHECK(std::isfinite(magnitude) && std::fabs(magnitude) <= 1e30, LC_ERR_INVALID, "%s: magnitude=%g", call, magnitude);
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    const int64_t row = (int64_t)pool.n_kv * pool.hd;
    LC_CHECK(k_dev && v_dev, LC_ERR_INVALID, "%s: null keys or values", call);
    LC_CHECK(k_stride >= row && v_stride >= row, LC_ERR_INVALID, "%s: rows of keys or values overlap (strides %lld, %lld below %lld)", call, (long long)k_stride, (long long)v_stride, (long long)row);
    if (q_dev) {
        LC_CHECK(q_out_dev, LC_ERR_INVALID, "%s: queries without a place for them", call);
        LC_CHECK(n_heads > 0 && n_heads <= 65536, LC_ERR_INVALID, "%s: n_heads=%d", call, n_heads);
        LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && q_out_stride >= (int64_t)n_heads * pool.hd, LC_ERR_INVALID, "%s: rows of queries overlap", call);
        LC_CHECK(q_dev != q_out_dev || q_stride == q_out_stride || n_rows == 1, LC_ERR_INVALID, "%s: queries in place with another stride", call);
    }
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    Append4Args a{k_dev, v_dev, q_dev, q_out_dev, k_stride, v_stride, q_stride, q_out_stride, positions_dev, turns_dev, q_dev ? n_heads : 0, rot_dim / 2, 0, 0, layout == LC_ROPE_INTERLEAVED, magnitude};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return append4_as<float>(pool, seqs, a, s);
    if (typ == LC_TYPE_F16) return append4_as<__half>(pool, seqs, a, s);
    return append4_as<__nv_bfloat16>(pool, seqs, a, s);
}

int32_t lc_kv4_read_dev(const lc_kv4_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, void* k_out_dev, int64_t k_stride, void* v_out_dev, int64_t v_stride, void* stream_) {
    const char* call = "lc_kv4_read_dev";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv4_check(call, cache, rows, typ, n_rows, &pool, &seqs));
    const int64_t row = (int64_t)pool.n_kv * pool.hd;
    LC_CHECK((!k_out_dev || k_stride >= row) && (!v_out_dev || v_stride >= row), LC_ERR_INVALID, "%s: rows overlap", call);
    if (n_rows == 0 || seqs.n_seqs == 0 || (!k_out_dev && !v_out_dev)) return LC_OK;
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    Read4Args a{k_out_dev, v_out_dev, k_stride, v_stride, 0, false};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return read4_as<float>(pool, seqs, a, s);
    if (typ == LC_TYPE_F16) return read4_as<__half>(pool, seqs, a, s);
    return read4_as<__nv_bfloat16>(pool, seqs, a, s);
}

}  // extern "C"
