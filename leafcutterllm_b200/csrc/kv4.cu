// The key/value cache in 4 bits: appending rows (with the position rotation on the way), reading rows back.
//
// A row's 16 dims x have the block scale s = e4m3(max |x| / (7 g)) and the integers n = rint(x / (s g)), all as if in 64 bits, so that the cache's bytes depend on the definition alone.
// f32 decides them wherever its error bounds allow; a block with a number or a scale too near a border between two, with infinities, NaN or sizes beyond f32's relative errors is done again in 64 bits.
// A thread has the 16 dims of one block and loads the 16 that they are paired with, so rows pass once.
//
// 4,970 rows of five sequences, 32 heads over 8 of 128 in bf16: append 27 us (107 MB), read back 9.2 (26 MB); first kernels 57 together.  What bounds the append is its instructions, 3,500 a row: 60 % of
// the issue slots, three blocks on an SM for 80 registers, the last wave of blocks half full; keys and values are a block's own work beside the queries' blocks (one block for both: 45).  Read: latency, four blocks of 16 dims
// a thread under way.  64 sequences of one row, 32 kv heads in f32: 7.9 and 4.6 us, 12.4 together, in each the chain row range -> context -> table -> row.
// Blocks of zeros are answered at once (every eighth row of zeros took 184 us when they went the 64-bit way); a block beyond 448 x 7 times its head's scale still goes it.
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
// s is `k` steps of the numbers of its size, 2^size to 2^(size + 1): 2^(size - 3) each; k = 16 is the next size's 8
__device__ __forceinline__ float block_scale(float k, int size) { return fminf(k * __int_as_float((127 + size - 3) << 23), 448.0f); }
__device__ __forceinline__ int size_of(float want) { return min(max((__float_as_int(want) >> 23) - 127, -6), 9); }
__device__ __forceinline__ uint32_t scale_byte(float s) { return s >= 0x1p-6f ? (__float_as_uint(s) >> 20) - (120u << 3) : (uint32_t)(s * 512.0f); }

// Where a block's numbers come from: dims d0 .. d0 + 15 of a head at x, turned by the row of a table (cosines and sines, then what their f32 lost) where they are before 2 * half.
template <typename T> struct BlockFrom {
    const T* x;
    const float2* row;
    const float2* low;
    int d0, half, n8;
    bool interleaved;
    __device__ __forceinline__ double number(int e) const {
        const int d = d0 + e;
        const double own = elem_f(x[d]);
        if (d >= 2 * half) return own;
        const int p = interleaved ? d >> 1 : d < half ? d : d - half, at = turn_place(p, n8);
        const bool second = interleaved ? d & 1 : d >= half;
        const double other = elem_f(x[interleaved ? d ^ 1 : second ? d - half : d + half]);
        const double c = (double)row[at].x + (double)low[at].x, si = (double)row[at].y + (double)low[at].y;
        return own * c + other * (second ? si : -si);
    }
};
template <typename P> __device__ __forceinline__ P* from_lane(P* p, int lane) { return reinterpret_cast<P*>(__shfl_sync(0xffffffffu, (unsigned long long)p, lane)); }
// The definition, in 64 bits, for the block of one lane, by the whole warp: a number per lane, twice.  Its own lane gets the result.
template <typename T> __device__ __noinline__ Block4 quantised64(const T* x, int d0, int half, const float2* row, const float2* low, int n8, bool interleaved, float head, int whose, Block4 out) {
    const int lane = threadIdx.x & 31;
    const BlockFrom<T> f{from_lane(x, whose), row, low, __shfl_sync(0xffffffffu, d0, whose), __shfl_sync(0xffffffffu, half, whose), n8, interleaved};
    const float g = __shfl_sync(0xffffffffu, head, whose);
    const double y = f.number(lane & 15), z = fabs(y);
    double top = z < (double)INFINITY ? z : 0.0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    // f32 says which two scales and integers are near; the border between them, exact in 64 bits, says which it is
    const float want = (float)fmin(top, (double)FLT_MAX) * (1.0f / (7.0f * g));
    const int size = size_of(want);
    const float r = want * __int_as_float((127 + 3 - size) << 23);
    float k = rintf(r);
    if (fabsf(fabsf(r - k) - 0.5f) < 0x1p-15f) {
        const float below = rintf(r - 0.5f);
        const double border = ((double)below + 0.5) * (double)__int_as_float((127 + size - 3) << 23) * (7.0 * (double)g);
        k = top > border ? below + 1.0f : top < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));
    }
    const float s = block_scale(k, size);
    const double step = (double)s * (double)g;
    const float a = fminf((float)fmin(z, (double)FLT_MAX) * (s > 0.0f ? 1.0f / (s * g) : 0.0f), 8.0f);
    float n = rintf(a);
    if (fabsf(fabsf(a - n) - 0.5f) < 1e-5f) {
        const float below = rintf(a - 0.5f);
        const double border = ((double)below + 0.5) * step;
        n = z > border ? below + 1.0f : z < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));
    }
    const int m = step > 0.0 && !isnan(y) ? (int)fminf(n, 7.0f) : 0;
    uint32_t w = (uint32_t)(y < 0.0 ? 8 - m : 8 + m) << (4 * (lane & 7));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
    const uint32_t w0 = __shfl_sync(0xffffffffu, w, 0), w1 = __shfl_sync(0xffffffffu, w, 8);
    if (lane == whose) {
        out.words = make_uint2(w0, w1);
        out.scale = scale_byte(s);
    }
    return out;
}
// The same in f32, for numbers that are off by `off` at most: false where one, or their scale, lies too near a border, where one is not finite, and for sizes that f32's relative errors do not
// hold for (0 is one that they do).  Numbers that are exact (off 0) often lie on borders, bf16 under a scale that is a power of two; these are compared in 64 bits.
__device__ __forceinline__ bool quantised32(const float (&y)[16], float off, float g, Block4& out) {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e++) most = max_nan(most, fabsf(y[e]));
    const float want = most * (1.0f / (7.0f * g));
    const int size = size_of(want);
    const float up = __int_as_float((127 + 3 - size) << 23), r = want * up;
    float k = rintf(r);
    // r is off by 2^-21 of itself besides; quotients, up to 7.5, by 2^-19
    bool sure = fabsf(r - k) < 0.5f - (off * (1.0f / (7.0f * g)) * up + r * 0x1p-21f);
    if (!sure && off == 0.0f) {
        const float below = rintf(r - 0.5f);
        const double border = ((double)below + 0.5) * (double)__int_as_float((127 + size - 3) << 23) * (7.0 * (double)g);
        k = (double)most > border ? below + 1.0f : (double)most < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));
        sure = true;
    }
    const float s = block_scale(k, size), inv = 1.0f / (s * g);
    float least = 0.0f;
    uint32_t w[2] = {0, 0};
    // of eight sums' upper bits, 0x4b400000, what eight multiplications by 16 leave
    constexpr uint32_t kUpper = 0x3f400000u;
#pragma unroll
    for (int e = 15; e >= 0; e--) {
        // added to 1.5 2^23 + 8, a small number is rounded to a whole one, to the nearest even, and 8 more are in the sum's low bits
        const float q = y[e] * inv, t = q + 12582920.0f;
        least = fmaxf(least, fabsf(q - (t - 12582920.0f)));
        w[e >> 3] = w[e >> 3] * 16u + __float_as_uint(t);
    }
    sure = sure && most * inv < 7.49f && most > 1e-30f && s > 0.0f;
    if (!(least < 0.5f - (off * inv + 0x1p-19f)) && sure) {
        if (off != 0.0f) return false;
        const double step = (double)s * (double)g, middle = 0.5 * step;
        w[0] = w[1] = 0;
#pragma unroll
        for (int e = 15; e >= 0; e--) {
            const float n = (y[e] * inv + 12582912.0f) - 12582912.0f;
            const double rest = fma((double)-n, step, (double)y[e]);   // compared with what 64 bits hold, its one rounding does not matter
            const bool odd = ((int)n & 1) != 0;
            const float to = rest > middle || (rest == middle && odd) ? n + 1.0f : rest < -middle || (rest == -middle && odd) ? n - 1.0f : n;
            w[e >> 3] = w[e >> 3] * 16u + __float_as_uint(to + 12582920.0f);
        }
    }
    const bool zeros = most == 0.0f && off == 0.0f;   // nothing to decide: rows that fill up a batch, heads that are switched off
    out.words = zeros ? make_uint2(0x88888888u, 0x88888888u) : make_uint2(w[0] - kUpper, w[1] - kUpper);
    out.scale = zeros ? 0 : scale_byte(s);
    return sure || zeros;
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

// Dims d0 .. d0 + 15 of a head of keys, turned in f32; returns how far one may be off.  VEC: they lie on one side of the middle and of the end of the rotated part, and 16-byte accesses are possible.
template <typename T, bool VEC>
__device__ __forceinline__ float turned16(const T* x, int d0, int half, bool interleaved, const float2* row, int n8, float (&y)[16]) {
    float v[16], big = 0.0f, other_big = 0.0f;
    load16f<T, VEC>(x + d0, v);
#pragma unroll
    for (int e = 0; e < 16; e++) big = fmaxf(big, fabsf(v[e]));
    if (VEC) {
        if (d0 >= 2 * half) {
#pragma unroll
            for (int e = 0; e < 16; e++) y[e] = v[e];
            return 0.0f;
        }
        if (interleaved) {
            const int p8 = d0 >> 4;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float2 t = row[k * n8 + p8];
                y[2 * k] = v[2 * k] * t.x - v[2 * k + 1] * t.y;
                y[2 * k + 1] = v[2 * k] * t.y + v[2 * k + 1] * t.x;
            }
        } else {
            const bool second = d0 >= half;
            float w[16];
            load16f<T, VEC>(x + (second ? d0 - half : d0 + half), w);
            const int p8 = (second ? d0 - half : d0) >> 3;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float2 t = row[(e & 7) * n8 + p8 + (e >> 3)];
                y[e] = v[e] * t.x + w[e] * (second ? t.y : -t.y);
                other_big = fmaxf(other_big, fabsf(w[e]));
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
                const float other = elem_f(x[interleaved ? d ^ 1 : second ? d - half : d + half]);
                const float2 t = row[turn_place(p, n8)];
                y[e] = y[e] * t.x + other * (second ? t.y : -t.y);
                other_big = fmaxf(other_big, fabsf(other));
            }
        }
    }
    // sine and cosine are off by 2^-25 of themselves (magnitude 1), products and their sum by 2^-24 each, of the two numbers together
    return (big + fmaxf(big, other_big)) * 0x1p-22f;
}

// grid: (groups of rows, slices of kv heads and then of query heads)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads, 3) kv4_append_kernel(Kv4Pool pool, Kv8Seqs seqs, Append4Args a) {
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
    const bool kv = (int)blockIdx.y < a.kv_slices;
    const int slices = kv ? a.kv_slices : gridDim.y - a.kv_slices, sl = kv ? blockIdx.y : blockIdx.y - a.kv_slices, heads = kv ? pool.n_kv : a.n_heads;
    const int h0 = heads * sl / slices, h1 = heads * (sl + 1) / slices;
    const int hd = pool.hd, half = a.half, n8 = (half + 7) >> 3;
    float2* const tab = reinterpret_cast<float2*>(smem);       // cosines and sines of the rows' pairs, then what f32 lost of them
    float2* const low = tab + rows * 8 * n8;
    if (VEC && tid < rows) {
        const uint32_t head = (uint32_t)(hd * sizeof(T));
        if (kv) {
            prefetch_l2((const T*)a.k + (row0 + tid) * a.k_stride + (int64_t)h0 * hd, (h1 - h0) * head);
            prefetch_l2((const T*)a.v + (row0 + tid) * a.v_stride + (int64_t)h0 * hd, (h1 - h0) * head);
        } else {
            prefetch_l2((const T*)a.q + (row0 + tid) * a.q_stride + (int64_t)h0 * hd, (h1 - h0) * head);
        }
    }
    __syncthreads();
    const Divider by_half(half);
    for (int e = tid; e < rows * half; e += kAppendThreads) {
        const int j = by_half(e), p = e - j * half;
        const RowPlace& at = place[j];
        if (at.seq < 0) continue;
        double2 t = turn_of(a.turns[p], (a.positions ? a.positions[at.seq] : (int64_t)seqs.ctx[at.seq]) + at.index);
        t.x *= a.magnitude;
        t.y *= a.magnitude;
        const int to = j * 8 * n8 + turn_place(p, n8);
        const float2 high = make_float2((float)t.x, (float)t.y);
        tab[to] = high;
        low[to] = make_float2((float)(t.x - high.x), (float)(t.y - high.y));
    }
    __syncthreads();
    // a row has its own share of the threads, whole warps
    const int share = kAppendThreads / a.rows, j = tid / share, mine = tid - j * share;
    if (j >= rows) return;
    const RowPlace at = place[j];
    const float2* const row = tab + j * 8 * n8;
    if (kv) {
        if (at.page < 0) return;
        // blocks of 16 dims, of the row's keys, then of its values; a warp's lanes go through this together
        const int blocks = hd >> 4, all = (h1 - h0) * blocks;
        const Divider by_blocks(blocks);
        const float by_magnitude = fmaxf(1.0f, fabsf((float)a.magnitude));
        const T* const k_row = (const T*)a.k + (int64_t)(row0 + j) * a.k_stride;
        const T* const v_row = (const T*)a.v + (int64_t)(row0 + j) * a.v_stride;
        for (int e0 = mine & ~31; e0 < 2 * all; e0 += share) {
            const int e = min(e0 + lane, 2 * all - 1);
            const bool here = e0 + lane < 2 * all, is_k = e < all;
            const int f = is_k ? e : e - all, g = by_blocks(f), h = h0 + g, b = f - g * blocks;
            const float head = (is_k ? pool.k_scale : pool.v_scale)[h];
            const T* const x = (is_k ? k_row : v_row) + h * hd;
            Block4 out;
            float y[16], off = 0.0f;
            if (is_k && half > 0) off = turned16<T, VEC>(x, 16 * b, half, a.interleaved, row, n8, y) * by_magnitude;
            else load16f<T, VEC>(x + 16 * b, y);
            const bool sure = quantised32(y, off, head, out);
            for (uint32_t left = __ballot_sync(0xffffffffu, here && !sure); left; left &= left - 1)
                out = quantised64(x, 16 * b, is_k ? half : 0, row, low + j * 8 * n8, n8, a.interleaved, head, __ffs(left) - 1, out);
            if (here) {
                const size_t to = (((size_t)at.page * pool.n_kv + h) << pool.page_shift) + at.slot;
                *reinterpret_cast<uint2*>((is_k ? pool.k : pool.v) + to * (hd >> 1) + 8 * b) = out.words;
                (is_k ? pool.k_block : pool.v_block)[to * blocks + b] = (uint8_t)out.scale;
            }
        }
    } else if (at.slot >= 0) {
        const T* const q_in = (const T*)a.q + (int64_t)(row0 + j) * a.q_stride + (int64_t)h0 * hd;
        T* const q_out = (T*)a.q_out + (int64_t)(row0 + j) * a.qo_stride + (int64_t)h0 * hd;
        const TurnRow<T> turns{row, low + j * 8 * n8};
        const int heads = h1 - h0;
        if constexpr (VEC) {
            constexpr int B = kTurnHeads<T>;
            const int groups = (heads + B - 1) / B, pairs = half >> 3, copies = (hd - 2 * half) >> 3;
            const Divider by_pairs(pairs), by_copies(copies);
            for (int e = mine; e < groups * pairs; e += share) {
                const int gr = by_pairs(e), h = gr * B;
                turn_item(q_in + h * hd, q_out + h * hd, hd, min(B, heads - h), e - gr * pairs, half, a.interleaved, turns, n8);
            }
            for (int e = mine; e < heads * copies; e += share) {
                const int h = by_copies(e);
                if (q_in != q_out) copy_item(q_in + h * hd, q_out + h * hd, e - h * copies, half);
            }
        } else {
            const int items = hd - half;
            for (int e = mine; e < heads * items; e += share) {
                const int h = e / items;
                turn_item_plain(q_in + h * hd, q_out + h * hd, e - h * items, half, a.interleaved, turns, n8);
            }
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
__global__ void __launch_bounds__(kAppendThreads, 5) kv4_read_kernel(Kv4Pool pool, Kv8Seqs seqs, Read4Args a) {
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
    const int h0 = pool.n_kv * blockIdx.y / gridDim.y, h1 = pool.n_kv * (blockIdx.y + 1) / gridDim.y;
    // a row has its own share of the threads; four blocks of 16 dims a thread, whose loads go out together
    const int share = kAppendThreads / a.rows, j = tid / share, mine = tid - j * share;
    if (j >= rows) return;
    const RowPlace at = place[j];
    if (at.seq < 0) return;
    const int blocks = pool.hd >> 4, all = (h1 - h0) * blocks;
    const Divider by_blocks(blocks);
    constexpr int B = 4;
    for (int e0 = mine; e0 < 2 * all; e0 += B * share) {
        uint2 w[B];
        float scale[B], head[B];
#pragma unroll
        for (int x = 0; x < B; x++) {
            const int e = min(e0 + x * share, 2 * all - 1);
            const bool is_k = e < all;
            const int f = is_k ? e : e - all, g = by_blocks(f), h = h0 + g, b = f - g * blocks;
            w[x] = make_uint2(0, 0);
            scale[x] = __int_as_float(0x7fffffff);
            head[x] = (is_k ? pool.k_scale : pool.v_scale)[h];
            if (at.page >= 0) {
                const size_t row = (((size_t)at.page * pool.n_kv + h) << pool.page_shift) + at.slot;
                w[x] = *reinterpret_cast<const uint2*>((is_k ? pool.k : pool.v) + row * (pool.hd >> 1) + 8 * b);
                scale[x] = scale4_f((is_k ? pool.k_block : pool.v_block)[row * blocks + b]);
            }
        }
#pragma unroll
        for (int x = 0; x < B; x++) {
            const int e = e0 + x * share;
            const bool is_k = e < all;
            const int f = is_k ? e : e - all;
            T* out = (T*)(is_k ? a.k : a.v);
            if (e >= 2 * all || !out) continue;
            __align__(16) T t[16];
#pragma unroll
            for (int y = 0; y < 16; y++) t[y] = to_elem<T>((float)(int)(((y < 8 ? w[x].x : w[x].y) >> (4 * (y & 7)) & 15u) - 8u) * scale[x] * head[x]);
            out += (int64_t)(row0 + j) * (is_k ? a.k_stride : a.v_stride) + (int64_t)h0 * pool.hd + 16 * f;
            if (a.vec) {
#pragma unroll
                for (int y = 0; y < (int)sizeof(T); y++) reinterpret_cast<uint4*>(out)[y] = reinterpret_cast<const uint4*>(t)[y];
            } else {
#pragma unroll
                for (int y = 0; y < 16; y++) out[y] = t[y];
            }
        }
    }
}

// Rows of a block: as many as leave two blocks for each SM; few rows: their heads over several blocks, of at least `least` heads
struct RowGrid {
    int rows, groups;
};
RowGrid row_grid(int n_rows) {
    RowGrid g;
    g.rows = 1;
    while (2 * g.rows <= kAppendRows && 2 * g.rows <= n_rows / (2 * sm_count())) g.rows *= 2;
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
    const size_t smem = (size_t)a.rows * ((a.half + 7) / 8 * 8) * sizeof(float4);
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
