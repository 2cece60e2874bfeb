// Eviction from the 4-bit cache: of every sequence and kv head the first, the last and the heaviest rows stay and move to the front of its pages, in their order.
//
// First kernel, a cluster of 1, 2, 4 or 8 blocks per sequence and kv head, which keep its sums in shared memory: the smallest sum that stays, by counting digits of the sums as whole numbers of the same
// order (11, 11 and 10 bits, the blocks' counts added over distributed shared memory); then the slots that stay, in ascending order, and the sums, which move with them.  Second kernel: the rows' bytes, in their
// places, a cluster per sequence, kv head and plane (keys, values, their scales).  The row that goes to slot j comes from kept[j] >= j, so a stretch of rows is read as a whole, by all threads of the
// cluster into registers, before it is written, in ascending order, and what a stretch writes is behind no row that a later one still reads.
#include <cooperative_groups.h>
#include <algorithm>
#include "lc_kernels.h"
#include "lc_kv4.cuh"

namespace cg = cooperative_groups;

namespace lc {

namespace {

struct EvictArgs {
    float* mass;
    int64_t mass_stride, mass_head_stride;
    int capacity, keep, limit, recent, first;
    int32_t* kept;
    int32_t* ctx_out;
};
constexpr int kSelectThreads = 512, kFarThreads = 1024, kMoveThreads = 512, kMovePieces = 8, kMostCluster = 8;
constexpr size_t kSelectSmem = 196 * 1024;  // of a block's sums, at most

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

// What both kernels that choose do first: the new length, and the slots of a sequence that is not cut; false for these.
__device__ __forceinline__ bool begins_cut(const Kv4Pool& pool, const Kv8Seqs& seqs, const EvictArgs& a, int i, int h, int length, int32_t* kept, bool lead, int at, int step) {
    const bool cut = length > a.limit;
    if (lead && h == 0) {
        if (length < 0) kv8_raise(seqs, i);
        a.ctx_out[i] = cut ? a.keep : length < 0 ? seqs.ctx[i] + max(seqs.row_start[i + 1] - seqs.row_start[i], 0) : length;
    }
    if (!cut)
        for (int j = at; j < a.limit; j += step) kept[j] = j < length ? j : -1;
    return cut;
}

// grid: (cluster, sequences * kv heads); `per`: slots of a block, a multiple of 32
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a, int per) {
    constexpr int W = kSelectThreads / 32;
    extern __shared__ float sum[];               // [per]
    __shared__ __align__(16) int hist[3][2048];
    __shared__ int sums[32], flag, chosen[2];
    __shared__ int2 warp_counts[W], block_counts;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = cluster.num_blocks(), rank = cluster.block_rank();
    const int i = blockIdx.y / pool.n_kv, h = blockIdx.y - i * pool.n_kv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    const int length = evict_length(seqs, pool, i, a.capacity, &flag);
    if (!begins_cut(pool, seqs, a, i, h, length, kept, rank == 0 && tid == 0, rank * kSelectThreads + tid, size * kSelectThreads)) return;  // the whole cluster
    float* mass = a.mass + (int64_t)i * a.mass_stride + (int64_t)h * a.mass_head_stride;
    const int lo = a.first, hi = length - a.recent, most = a.keep - a.first - a.recent;
    const int base = rank * per, mine = max(0, min(per, length - base));
    for (int x = tid; x < 3 * 2048; x += kSelectThreads) (&hist[0][0])[x] = 0;
    for (int x = tid; x < mine; x += kSelectThreads) sum[x] = mass[base + x];
    // the most-th largest of [lo, hi): its digits one after the other; `left`: how many of those that share the digits so far stay
    uint32_t value = 0;
    int left = most;
    const int in0 = max(lo - base, 0), in1 = min(hi - base, mine);  // the block's part of [lo, hi)
    if (most > 0) {
        const int bits[3] = {11, 11, 10};
        int shift = 32;
#pragma unroll
        for (int d = 0; d < 3; d++) {
            shift -= bits[d];
            __syncthreads();
            for (int x = in0 + tid; x < in1; x += kSelectThreads) {
                const uint32_t v = ordered(sum[x]);
                if (d == 0 || v >> (shift + bits[d]) == value >> (shift + bits[d])) atomicAdd(&hist[d][v >> shift & ((1u << bits[d]) - 1)], 1);
            }
            cluster.sync();
            // counts from the top: a thread has four places, of all blocks at once
            int4 part[kMostCluster];
#pragma unroll
            for (int r = 0; r < kMostCluster; r++)
                part[r] = r < size ? *cluster.map_shared_rank(reinterpret_cast<const int4*>(&hist[d][2044 - 4 * tid]), r) : make_int4(0, 0, 0, 0);
            int c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < kMostCluster; r++) { c[0] += part[r].w; c[1] += part[r].z; c[2] += part[r].y; c[3] += part[r].x; }
            const int mysum = (c[0] + c[1]) + (c[2] + c[3]);
            int all, before = before_me(mysum, sums, all);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (before < left && before + c[k] >= left) { chosen[0] = 2047 - 4 * tid - k; chosen[1] = left - before; }
                before += c[k];
            }
            __syncthreads();
            value |= (uint32_t)chosen[0] << shift;
            left = chosen[1];
        }
    }
    // Slots in ascending order: all above the value, and the first `left` equal to it.  A warp counts those of its stretch, then knows what is before it and goes over it again.
    __syncthreads();
    const int stretch = ((mine + W - 1) / W + 31) & ~31, x0 = min(warp * stretch, mine), x1 = min(x0 + stretch, mine);
    auto kind = [&](int x, bool& above, bool& equal) {
        const bool here = x < x1, in = x >= in0 && x < in1;
        const uint32_t v = here ? ordered(sum[x]) : 0;
        above = here && (!in || (most > 0 && v > value));
        equal = here && in && most > 0 && v == value;
    };
    int2 mc = make_int2(0, 0);
    for (int x = x0; x < x1; x += 32) {
        bool above, equal;
        kind(x + lane, above, equal);
        mc.x += __popc(__ballot_sync(0xffffffffu, above));
        mc.y += __popc(__ballot_sync(0xffffffffu, equal));
    }
    if (lane == 0) warp_counts[warp] = mc;
    __syncthreads();
    if (tid == 0) {
        int2 t = make_int2(0, 0);
        for (int w = 0; w < W; w++) { t.x += warp_counts[w].x; t.y += warp_counts[w].y; }
        block_counts = t;
    }
    cluster.sync();  // and every sum is in shared memory
    int equals = 0, out = 0;
    auto pass = [&](const int2& n) {
        out += n.x + min(max(left - equals, 0), n.y);
        equals += n.y;
    };
    for (int r = 0; r < rank; r++) pass(*cluster.map_shared_rank(&block_counts, r));
    for (int w = 0; w < warp; w++) pass(warp_counts[w]);
    for (int x = x0; x < x1; x += 32) {
        bool above, equal;
        kind(x + lane, above, equal);
        const uint32_t below = (1u << lane) - 1, eq = __ballot_sync(0xffffffffu, equal);
        const bool stays = above || (equal && equals + __popc(eq & below) < left);
        const uint32_t st = __ballot_sync(0xffffffffu, stays);
        if (stays) {
            const int to = out + __popc(st & below);
            kept[to] = base + x + lane;
            mass[to] = sum[x + lane];
        }
        equals += __popc(eq);
        out += __popc(st);
    }
    for (int x = a.keep + rank * kSelectThreads + tid; x < length; x += size * kSelectThreads) mass[x] = 0.0f;
    for (int x = a.keep + rank * kSelectThreads + tid; x < a.limit; x += size * kSelectThreads) kept[x] = -1;
    cluster.sync();  // no block leaves while another reads its counts
}

// The same for contexts that a cluster's shared memory does not hold: a block per sequence and kv head, over the sums in global memory.  grid: (sequences, kv heads)
__global__ void __launch_bounds__(kFarThreads) kv4_select_far_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a) {
    __shared__ int hist[2048];
    __shared__ int sums[32], flag, chosen[2];
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int length = evict_length(seqs, pool, i, a.capacity, &flag);
    int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    if (!begins_cut(pool, seqs, a, i, h, length, kept, tid == 0, tid, kFarThreads)) return;
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
            for (int x = tid; x < 2048; x += kFarThreads) hist[x] = 0;
            __syncthreads();
            for (int x = lo + tid; x < hi; x += kFarThreads) {
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
    for (int x0 = 0; x0 < length; x0 += kFarThreads) {
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
    for (int x = a.keep + tid; x < length; x += kFarThreads) mass[x] = 0.0f;
    for (int x = a.keep + tid; x < a.limit; x += kFarThreads) kept[x] = -1;
}

// Rows of pieces (T) by one cluster: slot j of the sequence from kept[j].
template <typename T>
__device__ __forceinline__ void move_rows(const Kv4Pool& pool, const int32_t* table, const int32_t* kept, int keep, int h, uint8_t* base, int row_bytes) {
    cg::cluster_group cluster = cg::this_cluster();
    const int threads = kMoveThreads * cluster.num_blocks(), me = cluster.block_rank() * kMoveThreads + threadIdx.x;
    const int pieces = row_bytes / (int)sizeof(T), mask = (1 << pool.page_shift) - 1;
    const int all = keep * pieces;               // in 31 bits: checked by the call
    auto at = [&](int slot, int piece) {
        return reinterpret_cast<T*>(base + ((((size_t)table[slot >> pool.page_shift] * pool.n_kv + h) << pool.page_shift) + (slot & mask)) * row_bytes) + piece;
    };
    for (int e0 = 0; e0 < all; e0 += threads * kMovePieces) {
        T v[kMovePieces];
        int from[kMovePieces];
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int e = e0 + u * threads + me;
            from[u] = e < all ? kept[e / pieces] : -1;
        }
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int e = e0 + u * threads + me;
            if (from[u] >= 0 && from[u] != e / pieces) v[u] = *at(from[u], e % pieces);
        }
        cluster.sync();
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int e = e0 + u * threads + me;
            if (from[u] >= 0 && from[u] != e / pieces) *at(e / pieces, e % pieces) = v[u];
        }
        if (e0 + threads * kMovePieces < all) cluster.sync();
    }
}
// grid: (cluster, sequences * kv heads, planes: keys, values, their scales)
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a) {
    const int i = blockIdx.y / pool.n_kv, h = blockIdx.y - i * pool.n_kv, hd = pool.hd;
    // sequences that are cut, and not left alone: only these have a new length
    if ((long long)seqs.ctx[i] + seqs.row_start[i + 1] - seqs.row_start[i] <= a.limit || a.ctx_out[i] != a.keep) return;
    const int32_t* table = seqs.table + (size_t)i * seqs.width;
    const int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    uint8_t* const base = blockIdx.z == 0 ? (uint8_t*)pool.k : blockIdx.z == 1 ? (uint8_t*)pool.v : blockIdx.z == 2 ? pool.k_block : pool.v_block;
    const int bytes = blockIdx.z < 2 ? hd >> 1 : hd >> 4;
    if (bytes % 16 == 0) move_rows<uint4>(pool, table, kept, a.keep, h, base, bytes);
    else if (bytes % 8 == 0) move_rows<uint2>(pool, table, kept, a.keep, h, base, bytes);
    else if (bytes % 4 == 0) move_rows<uint32_t>(pool, table, kept, a.keep, h, base, bytes);
    else move_rows<uint8_t>(pool, table, kept, a.keep, h, base, bytes);
}

cudaLaunchConfig_t clusters(dim3 grid, int threads, size_t smem, cudaStream_t s, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = grid.x;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
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
    LC_CHECK((int64_t)keep * (pool.hd / 16) < 0x70000000, LC_ERR_INVALID, "%s: keep=%d rows of %d dims are too many for one call", call, keep, pool.hd);
    LC_CHECK((int64_t)seqs.n_seqs * pool.n_kv <= 65535, LC_ERR_INVALID, "%s: %d sequences of %d kv heads are too many for one call", call, seqs.n_seqs, pool.n_kv);
    if (seqs.n_seqs == 0) return LC_OK;
    LC_CHECK(seqs.table && seqs.ctx && seqs.row_start && mass_dev && kept_dev && ctx_out_dev, LC_ERR_INVALID, "%s: null pointer", call);
    LC_CHECK(ctx_out_dev != seqs.ctx, LC_ERR_INVALID, "%s: the new lengths need a place of their own", call);  // the old ones are read to the end
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, call));
    const EvictArgs a{mass_dev, mass_stride, mass_head_stride, capacity, keep, limit, recent, first, kept_dev, ctx_out_dev};
    cudaStream_t s = stream_or_own(stream_);
    cudaLaunchAttribute attr[1];
    // blocks of a cluster: as many as leave all sequences and heads about two blocks for each SM, and at least what holds the longest context's sums
    const int64_t slots = std::min<int64_t>((int64_t)seqs.width << pool.page_shift, capacity), units = (int64_t)seqs.n_seqs * pool.n_kv;
    auto per_block = [&](int size) { return (slots + 32 * size - 1) / (32 * size) * 32; };
    int size = 1;
    while (size < kMostCluster && (2 * size * units <= 2 * sm_count() || per_block(size) * sizeof(float) > kSelectSmem)) size *= 2;
    if (per_block(size) * sizeof(float) <= kSelectSmem) {
        const size_t smem = per_block(size) * sizeof(float);
        LC_CUDA(ensure_smem_limit((const void*)kv4_select_kernel, smem));
        const cudaLaunchConfig_t cfg = clusters(dim3((unsigned)size, (unsigned)units), kSelectThreads, smem, s, attr);
        LC_CUDA(cudaLaunchKernelEx(&cfg, kv4_select_kernel, pool, seqs, a, (int)per_block(size)));
    } else {
        kv4_select_far_kernel<<<dim3((unsigned)seqs.n_seqs, (unsigned)pool.n_kv), kFarThreads, 0, s>>>(pool, seqs, a);
        LC_CUDA(cudaGetLastError());
    }
    // blocks of a cluster that moves rows: what has a plane's 16-byte pieces in two stretches
    size = 1;
    while (size < kMostCluster && (int64_t)keep * ((pool.hd + 31) / 32) > (int64_t)2 * size * kMoveThreads * kMovePieces) size *= 2;
    const cudaLaunchConfig_t cfg = clusters(dim3((unsigned)size, (unsigned)units, 4), kMoveThreads, 0, s, attr);
    LC_CUDA(cudaLaunchKernelEx(&cfg, kv4_move_kernel, pool, seqs, a));
    return LC_OK;
}
