// Eviction from the 4-bit cache: of every sequence and kv head the first, the last and the heaviest rows stay and move to the front of its pages, in their order.
//
// First kernel, a block per sequence and kv head: the smallest sum that stays, by counting digits of the sums as whole numbers of the same order (11, 11 and 10 bits); then the slots that
// stay, in ascending order, and the sums, which move with them.  Second kernel: the rows' bytes, in their places.  The row that goes to slot j comes from kept[j] >= j, so chunks of rows are read as a whole before they
// are written, in ascending order, and what a chunk writes is behind no row that a later one still reads.
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"

namespace lc {

namespace {

struct EvictArgs {
    float* mass;
    int64_t mass_stride, mass_head_stride;
    int capacity, keep, limit, recent, first;
    int32_t* kept;
    int32_t* ctx_out;
};
constexpr int kSelectThreads = 1024, kMoveThreads = 512, kMovePieces = 4;

// whole numbers in the order of f32, NaN at the bottom
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    if (x != x) return 0;
    return x == 0.0f ? 0x80000000u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
// the sum over all threads in front of this one; `all`: of all of them
__device__ __forceinline__ int before_me(int v, int* sums, int& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int off = 0;
    all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        const int u = sums[w];
        if (w < warp) off += u;
        all += u;
    }
    return off + incl - v;
}
// What a sequence holds (-1: it raises the status and stays as it is); by one whole block.
__device__ __forceinline__ int evict_length(const Kv8Seqs& s, const Kv8Pool& p, int i, int capacity, int* flag) {
    const int ctx = s.ctx[i], n = s.row_start[i + 1] - s.row_start[i];
    bool ok = n >= 0 && ctx >= 0 && (long long)ctx + n <= ((long long)s.width << p.page_shift) && (long long)ctx + n <= capacity;
    const int pages = ok ? (ctx + n + (1 << p.page_shift) - 1) >> p.page_shift : 0;
    if (threadIdx.x == 0) *flag = 0;
    __syncthreads();
    bool bad = false;
    for (int x = threadIdx.x; x < pages; x += blockDim.x) {
        const int number = s.table[(size_t)i * s.width + x];
        bad = bad || number < 0 || number >= p.n_pages;
    }
    if (bad) *flag = 1;
    __syncthreads();
    return ok && !*flag ? ctx + n : -1;
}

// grid: (sequences, kv heads)
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a) {
    __shared__ int hist[2048];
    __shared__ int sums[32], flag, chosen[2];
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int length = evict_length(seqs, pool, i, a.capacity, &flag);
    int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    const bool cut = length > a.limit;
    if (tid == 0 && h == 0) {
        if (length < 0) kv8_raise(seqs, i);
        a.ctx_out[i] = cut ? a.keep : length < 0 ? seqs.ctx[i] + max(seqs.row_start[i + 1] - seqs.row_start[i], 0) : length;
    }
    if (!cut) {
        for (int j = tid; j < a.limit; j += kSelectThreads) kept[j] = j < length ? j : -1;
        return;
    }
    float* mass = a.mass + (int64_t)i * a.mass_stride + (int64_t)h * a.mass_head_stride;
    const int lo = a.first, hi = length - a.recent, most = a.keep - a.first - a.recent;
    // the most-th largest of [lo, hi): its digits one after the other; `left`: how many of those that share the digits so far stay
    uint32_t value = 0;
    int left = most;
    if (most > 0) {
        const int bits[3] = {11, 11, 10};
        int shift = 32;
        for (int d = 0; d < 3; d++) {
            shift -= bits[d];
            for (int x = tid; x < 2048; x += kSelectThreads) hist[x] = 0;
            __syncthreads();
            for (int x = lo + tid; x < hi; x += kSelectThreads) {
                const uint32_t v = ordered(mass[x]);
                if (d == 0 || v >> (shift + bits[d]) == value >> (shift + bits[d])) atomicAdd(&hist[v >> shift & ((1u << bits[d]) - 1)], 1);
            }
            __syncthreads();
            // counts from the top: a thread has two places
            const int p1 = 2047 - 2 * tid, c1 = hist[p1], c0 = hist[p1 - 1];
            int all;
            const int before = before_me(c1 + c0, sums, all);
            if (before < left && before + c1 >= left) { chosen[0] = p1; chosen[1] = left - before; }
            else if (before + c1 < left && before + c1 + c0 >= left) { chosen[0] = p1 - 1; chosen[1] = left - before - c1; }
            __syncthreads();
            value |= (uint32_t)chosen[0] << shift;
            left = chosen[1];
            __syncthreads();
        }
    }
    // slots in ascending order: all above the value, and the first `left` equal to it
    int out = 0, equals = 0;
    for (int x0 = 0; x0 < length; x0 += kSelectThreads) {
        const int x = x0 + tid;
        const float w = x < length ? mass[x] : 0.0f;
        const bool fixed = x < length && (x < lo || x >= hi), in = x >= lo && x < hi && most > 0;
        const uint32_t v = ordered(w);
        int n_equal, n_out;
        const bool equal = in && v == value;
        const int e = equals + before_me(equal, sums, n_equal);
        const bool stays = fixed || (in && v > value) || (equal && e < left);
        const int to = out + before_me(stays, sums, n_out);
        __syncthreads();  // every sum of the stretch is read
        if (stays) {
            kept[to] = x;
            mass[to] = w;
        }
        out += n_out;
        equals += n_equal;
    }
    __syncthreads();
    for (int x = a.keep + tid; x < length; x += kSelectThreads) mass[x] = 0.0f;
    for (int x = a.keep + tid; x < a.limit; x += kSelectThreads) kept[x] = -1;
}

// Rows of `unit`-byte pieces (T) by one block: slot j of the sequence from kept[j].
template <typename T>
__device__ __forceinline__ void move_rows(const Kv4Pool& pool, const int32_t* table, const int32_t* kept, int keep, int h, uint8_t* base, int row_bytes, int p0, int pieces) {
    const int per_chunk = kMoveThreads * kMovePieces / pieces;
    const int mask = (1 << pool.page_shift) - 1;
    auto at = [&](int slot) { return base + ((((size_t)table[slot >> pool.page_shift] * pool.n_kv + h) << pool.page_shift) + (slot & mask)) * row_bytes; };
    for (int j0 = 0; j0 < keep; j0 += per_chunk) {
        T v[kMovePieces];
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int e = u * kMoveThreads + threadIdx.x, j = j0 + e / pieces;
            if (e < per_chunk * pieces && j < keep) v[u] = reinterpret_cast<const T*>(at(kept[j]))[p0 + e % pieces];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int e = u * kMoveThreads + threadIdx.x, j = j0 + e / pieces;
            if (e < per_chunk * pieces && j < keep) reinterpret_cast<T*>(at(j))[p0 + e % pieces] = v[u];
        }
        __syncthreads();
    }
}
// grid: (sequences, kv heads, planes: keys, values, their scales)
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a) {
    __shared__ int flag;
    const int i = blockIdx.x, h = blockIdx.y, hd = pool.hd;
    if (evict_length(seqs, pool, i, a.capacity, &flag) <= a.limit) return;
    const int32_t* table = seqs.table + (size_t)i * seqs.width;
    const int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    if (blockIdx.z < 2) move_rows<uint2>(pool, table, kept, a.keep, h, (uint8_t*)(blockIdx.z ? pool.v : pool.k), hd >> 1, 0, hd >> 4);
    else move_rows<uint8_t>(pool, table, kept, a.keep, h, blockIdx.z == 3 ? pool.v_block : pool.k_block, hd >> 4, 0, hd >> 4);
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" int32_t lc_kv4_evict_dev(const lc_kv4_cache* cache, const lc_kv8_rows* rows, float* mass_dev, int64_t mass_stride, int64_t mass_head_stride, int32_t capacity, int32_t keep, int32_t limit,
                                    int32_t recent, int32_t first, int32_t* kept_dev, int32_t* ctx_out_dev, void* stream_) {
    const char* call = "lc_kv4_evict_dev";
    Kv4Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv4_check(call, cache, rows, LC_TYPE_F32, 0, &pool, &seqs));
    LC_CHECK(recent >= 0 && first >= 0 && keep > 0 && (int64_t)recent + first <= keep && keep <= limit && limit <= capacity, LC_ERR_INVALID,
             "%s: first=%d + recent=%d <= keep=%d (1 or more) <= limit=%d <= capacity=%d expected", call, first, recent, keep, limit, capacity);
    LC_CHECK(mass_head_stride >= capacity && mass_stride >= capacity, LC_ERR_INVALID, "%s: capacity=%d (the strides of the sums are %lld and %lld)", call, capacity, (long long)mass_stride,
             (long long)mass_head_stride);
    LC_CHECK(seqs.n_seqs <= 1 || pool.n_kv == 1 || mass_stride >= (int64_t)(pool.n_kv - 1) * mass_head_stride + capacity || mass_head_stride >= (int64_t)(seqs.n_seqs - 1) * mass_stride + capacity,
             LC_ERR_INVALID, "%s: the sums of sequences and heads overlap (strides %lld and %lld)", call, (long long)mass_stride, (long long)mass_head_stride);
    if (seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(seqs.table && seqs.ctx && seqs.row_start && mass_dev && kept_dev && ctx_out_dev, LC_ERR_INVALID, "%s: null pointer", call);
    LC_CHECK(ctx_out_dev != seqs.ctx, LC_ERR_INVALID, "%s: the new lengths need a place of their own", call);  // the old ones are read to the end
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    const EvictArgs a{mass_dev, mass_stride, mass_head_stride, capacity, keep, limit, recent, first, kept_dev, ctx_out_dev};
    cudaStream_t s = stream_or_own(stream_);
    kv4_select_kernel<<<dim3((unsigned)seqs.n_seqs, (unsigned)pool.n_kv), kSelectThreads, 0, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    kv4_move_kernel<<<dim3((unsigned)seqs.n_seqs, (unsigned)pool.n_kv, 4), kMoveThreads, 0, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
