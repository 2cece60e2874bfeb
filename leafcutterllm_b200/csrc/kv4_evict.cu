// Eviction from the 4-bit cache: of every sequence and kv head the first, the last and the heaviest rows stay and move to the front of its pages, in their order.
//
// First kernel, a cluster of 1, 2, 4 or 8 blocks per sequence and kv head, which keep its sums in shared memory: the smallest sum that stays, by counting digits of the sums as whole numbers of the same
// order (11, 11 and 10 bits, the blocks' counts added over distributed shared memory); then the slots that stay, in ascending order, and the sums, which move with them.  Second kernel: the rows' bytes, in their
// places, a cluster per sequence, kv head and plane (keys, values, their scales).  The row that goes to slot j comes from kept[j] >= j, so a stretch of rows is read as a whole, by all threads of the
// cluster into registers, before it is written, in ascending order, and what a stretch writes is behind no row that a later one still reads.
//
// 64 sequences and 8 kv heads of 128 cut to 1,024 slots where they have more than 1,280, a first eviction with L2 cold: 36 us, 56 MB (a floor of 8.5); two of them cut to 16,384: 70 us, 85 MB (12.9; an empty kernel reads
// 9 the same way).  What bounds it is a chain of waits: the sums, three rounds of digits in clusters of 8 (a count of 1,700 to 3,200 cycles, a barrier, other blocks' counts, a scan), the list, a launch, kept slot ->
// page -> row.  Cut again as they are, so that an eighth and a thirtieth of the rows move, replayed: 26 and 66 us; none above the limit: 9.  Of the second kernel's shapes four pieces a thread and three blocks on an SM
// are the best, 36 and 70 us (eight and two: 40 and 73; two and three: 40 and 73).  First kernels, a block for a sequence and head over sums in global memory: 80 and 612, replayed.
// Blocks are sized by what sequences may hold, the smaller of the tables' length and the sums' capacity, not by the contexts, which only the device knows: in tables of 131,072 slots the 64 sequences take 209 us (blocks of 16,384 sums, of which one in eight has any), in tables beyond
// clusters, of 524,288, 63.  One sequence of 500,000 slots cut to 65,536, a block for each head: 1,640.
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
constexpr int kFarThreads = 1024, kMoveThreads = 512, kMovePieces = 4, kMostCluster = 8;
constexpr size_t kSelectSmem = 190 * 1024;  // of a block's sums and slots, at most

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

// What a thread of the block's first eight warps has before it, of their v; `totals`: of these warps, for this call alone.
__device__ __forceinline__ int before_thread(int v, int* totals) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31 && warp < 8) totals[warp] = incl;
    __syncthreads();
    return incl - v + __reduce_add_sync(0xffffffffu, lane < min(warp, 8) ? totals[lane] : 0);
}
// grid: (cluster, sequences * kv heads); `per`: slots of a block, a multiple of 128
template <int T>
__global__ void __launch_bounds__(T, T == 512 ? 4 : 1) kv4_select_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a, int per) {
    constexpr int W = T / 32, AT_ONCE = T == 512 ? 2 : kMostCluster;   // AT_ONCE: blocks whose counts are read together; four blocks of 512 on an SM have 32 registers a thread
    extern __shared__ __align__(16) uint32_t key[];              // [per], sums as whole numbers of their order
    uint16_t* const list = reinterpret_cast<uint16_t*>(key + per);   // [per], the block's slots that stay
    __shared__ __align__(16) uint32_t hist[3][1024];             // counts of 16 bits, two in a word: a block has fewer sums than that
    __shared__ int totals[3][8];
    __shared__ int flag, chosen[3][2];
    __shared__ int2 warp_counts[W], block_counts;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = cluster.num_blocks(), rank = cluster.block_rank();
    const int i = blockIdx.y / pool.n_kv, h = blockIdx.y - i * pool.n_kv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t* kept = a.kept + ((int64_t)i * pool.n_kv + h) * a.limit;
    float* mass = a.mass + (int64_t)i * a.mass_stride + (int64_t)h * a.mass_head_stride;
    const int base = rank * per;
    {
        // the sums set out while the pages are looked at: of a length that may turn out to be none
        const int maybe = min(max(seqs.ctx[i] + seqs.row_start[i + 1] - seqs.row_start[i], 0), a.capacity), mine = max(0, min(per, maybe - base));
        if (maybe > a.limit) {
            const int quads = (uintptr_t)mass % 16 == 0 ? mine >> 2 : 0;
#pragma unroll 4
            for (int q = tid; q < quads; q += T) {
                const float4 v = reinterpret_cast<const float4*>(mass + base)[q];
                reinterpret_cast<uint4*>(key)[q] = make_uint4(ordered(v.x), ordered(v.y), ordered(v.z), ordered(v.w));
            }
#pragma unroll 4
            for (int x = 4 * quads + tid; x < ((mine + 3) & ~3); x += T) key[x] = x < mine ? ordered(mass[base + x]) : 0;
        }
    }
    for (int x = tid; x < 3 * 256; x += T) reinterpret_cast<int4*>(&hist[0][0])[x] = make_int4(0, 0, 0, 0);
    const int length = evict_length(seqs, pool, i, a.capacity, &flag);
    if (!begins_cut(pool, seqs, a, i, h, length, kept, rank == 0 && tid == 0, rank * T + tid, size * T)) return;  // the whole cluster
    const int lo = a.first, hi = length - a.recent, most = a.keep - a.first - a.recent;
    const int mine = max(0, min(per, length - base)), quads = (mine + 3) >> 2;
    // the most-th largest of [lo, hi): its digits one after the other; `left`: how many of those that share the digits so far stay
    uint32_t value = 0;
    int left = most;
    const int in0 = max(lo - base, 0), in1 = min(hi - base, mine);  // the block's part of [lo, hi)
    const uint4* const key4 = reinterpret_cast<const uint4*>(key);
    if (most > 0) {
        const int bits[3] = {11, 11, 10};
        int shift = 32;
#pragma unroll
        for (int d = 0; d < 3; d++) {
            shift -= bits[d];
            __syncthreads();
            auto count = [&](uint32_t v) {
                if (d == 0 || v >> (shift + bits[d]) == value >> (shift + bits[d])) {
                    const uint32_t digit = v >> shift & ((1u << bits[d]) - 1);
                    atomicAdd(&hist[d][digit >> 1], digit & 1 ? 0x10000u : 1u);
                }
            };
            const int f0 = (in0 + 3) >> 2, f1 = in1 >> 2;   // quads of nothing else
#pragma unroll 2
            for (int q = f0 + tid; q < f1; q += T) {
                const uint4 v = key4[q];
                count(v.x);
                count(v.y);
                count(v.z);
                count(v.w);
            }
            if (tid < 8) {
                const int x = tid < 4 ? 4 * f0 - 4 + tid : 4 * max(f1, f0) + tid - 4;   // around them
                if (x >= in0 && x < in1) count(key[x]);
            }
            cluster.sync();
            // counts from the top, of all blocks at once: a thread of the first eight warps has eight places in a row
            int c[8] = {}, all = 0;
            if (tid < 256) {
                for (int r0 = 0; r0 < size; r0 += AT_ONCE) {
                    uint4 part[AT_ONCE];
#pragma unroll
                    for (int r = 0; r < AT_ONCE; r++)
                        part[r] = r0 + r < size ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&hist[d][1020 - 4 * tid], r0 + r)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < AT_ONCE; r++) {
                        c[0] += part[r].w >> 16; c[1] += part[r].w & 0xffff; c[2] += part[r].z >> 16; c[3] += part[r].z & 0xffff;
                        c[4] += part[r].y >> 16; c[5] += part[r].y & 0xffff; c[6] += part[r].x >> 16; c[7] += part[r].x & 0xffff;
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++) all += c[k];
            }
            int before = before_thread(all, totals[d]);
            if (tid < 256 && before < left && before + all >= left)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (before < left && before + c[k] >= left) { chosen[d][0] = 2047 - 8 * tid - k; chosen[d][1] = left - before; }
                    before += c[k];
                }
            __syncthreads();
            value |= (uint32_t)chosen[d][0] << shift;
            left = chosen[d][1];
        }
    } else {
        __syncthreads();
    }
    // Slots in ascending order: all above the value, and the first `left` equal to it.  A warp counts those of its stretch, four in a row a lane, then knows what is before it.
    const int stretch = ((quads + W - 1) / W + 31) & ~31, q0 = min(warp * stretch, quads), q1 = min(q0 + stretch, quads);
    // bits 0-3: of a lane's four those above, 4-7: those equal
    auto kinds = [&](int q) {
        uint32_t bits = 0;
        if (q + lane >= q1) return bits;
        const uint4 k4 = key4[q + lane];
        const uint32_t v[4] = {k4.x, k4.y, k4.z, k4.w};
        if (most > 0)
#pragma unroll
            for (int e = 0; e < 4; e++) bits |= (v[e] > value ? 1u << e : 0u) | (v[e] == value ? 16u << e : 0u);
        const int x0 = 4 * (q + lane);
        if (x0 < in0 || x0 + 4 > in1) {  // some are not chosen by their sums
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int x = x0 + e;
                if (x < in0 || x >= in1) bits = (bits & ~(17u << e)) | (x < mine ? 1u << e : 0u);
            }
        }
        return bits;
    };
    int n_both = 0;                                              // above, and in the upper half equal: 16 bits are enough for a block's
    uint64_t kept_kinds = 0;                                     // a byte for each of the stretch's eight rounds at most (a block's slots are 32,384 at most)
    for (int q = q0, at = 0; q < q1; q += 32, at += 8) {
        const uint32_t b = kinds(q);
        kept_kinds |= (uint64_t)b << at;
        n_both += __popc(b & 15u) + (__popc(b & 240u) << 16);
    }
    const int2 mc = make_int2(__reduce_add_sync(0xffffffffu, n_both & 0xffff), __reduce_add_sync(0xffffffffu, n_both >> 16));
    if (lane == 0) warp_counts[warp] = mc;
    __syncthreads();
    if (warp == 0) {
        const int2 t = lane < W ? warp_counts[lane] : make_int2(0, 0);
        const int x = __reduce_add_sync(0xffffffffu, t.x), y = __reduce_add_sync(0xffffffffu, t.y);
        if (lane == 0) block_counts = make_int2(x, y);
    }
    cluster.sync();  // and every sum is in shared memory
    // what is in front: above and equal of the blocks before, of the warps before
    int2 mine_before = lane < rank ? *cluster.map_shared_rank(&block_counts, lane) : make_int2(0, 0);
    const int b_above = __reduce_add_sync(0xffffffffu, mine_before.x), b_equal = __reduce_add_sync(0xffffffffu, mine_before.y);
    mine_before = lane < warp ? warp_counts[lane] : make_int2(0, 0);
    int above = b_above + __reduce_add_sync(0xffffffffu, mine_before.x), equals = b_equal + __reduce_add_sync(0xffffffffu, mine_before.y);
    // of the equal ones the first `left` stay: out = above + min(equals, left)
    const int begin = b_above + min(b_equal, left);              // of the block
    auto put = [&](int q, uint32_t b, int to, int e_before) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool eq = b >> (4 + e) & 1, stays = (b >> e & 1) || (eq && e_before < left);
            if (stays) list[to++] = (uint16_t)(4 * (q + lane) + e);
            e_before += eq;
        }
    };
    for (int q = q0; q < q1; q += 64, kept_kinds >>= 16) {
        // two rounds at once: four counts of 128 at most in a word
        const uint32_t b0 = (uint32_t)kept_kinds & 255u, b1 = (uint32_t)kept_kinds >> 8 & 255u;
        const uint32_t n = __popc(b0 & 15u) | __popc(b0 >> 4) << 8 | __popc(b1 & 15u) << 16 | __popc(b1 >> 4) << 24;
        uint32_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        const uint32_t before = incl - n, total = __shfl_sync(0xffffffffu, incl, 31);
        int e_before = equals + (before >> 8 & 255u);
        put(q, b0, above + (before & 255u) + min(e_before, left) - begin, e_before);
        above += total & 255u;
        equals += total >> 8 & 255u;
        e_before = equals + (before >> 24);
        put(q + 32, b1, above + (before >> 16 & 255u) + min(e_before, left) - begin, e_before);
        above += total >> 16 & 255u;
        equals += total >> 24;
    }
    if (warp == W - 1 && lane == 0) chosen[0][0] = above + min(equals, left) - begin;   // the last warp knows how many there are
    __syncthreads();
    const int n_list = chosen[0][0];
#pragma unroll 4
    for (int o = tid; o < n_list; o += T) {
        const int x = list[o];
        const uint32_t v = key[x];
        kept[begin + o] = base + x;
        mass[begin + o] = v == 0 ? __int_as_float(0x7fffffff) : __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v);
    }
    for (int x = a.keep + rank * T + tid; x < length; x += size * T) mass[x] = 0.0f;
    for (int x = a.keep + rank * T + tid; x < a.limit; x += size * T) kept[x] = -1;
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

// Rows of pieces (T) by one cluster: slot j of the sequence from kept[j].  A thread has the same piece of some rows.
template <typename T>
__device__ __forceinline__ void move_rows(const Kv4Pool& pool, const int32_t* table, const int32_t* kept, int keep, int h, uint8_t* base, int row_bytes) {
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = cluster.num_blocks(), mask = (1 << pool.page_shift) - 1;
    const int pieces = row_bytes / (int)sizeof(T), rows = kMoveThreads / pieces;   // rows of a block at a time
    const int mine = threadIdx.x / pieces, piece = threadIdx.x - mine * pieces, step = blocks * rows;
    T* const from0 = reinterpret_cast<T*>(base) + piece;
    auto at = [&](int number, int slot) { return from0 + ((((size_t)(uint32_t)number * (uint32_t)pool.n_kv + h) << pool.page_shift) + (slot & mask)) * (uint32_t)pieces; };
    const int j_first = (int)cluster.block_rank() * rows + mine;
    // what is not there reads the first slot's row
    auto there = [&](int j) { return mine < rows && j < keep; };
    int from[kMovePieces];
#pragma unroll
    for (int u = 0; u < kMovePieces; u++) from[u] = kept[there(j_first + u * step) ? j_first + u * step : 0];
    for (int j0 = 0; j0 < keep; j0 += step * kMovePieces) {
        const int j = j0 + j_first, next = j + step * kMovePieces;
        // all loads of a kind go out together, the next stretch's first ones too
        T v[kMovePieces];
        int page[kMovePieces];
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) page[u] = table[from[u] >> pool.page_shift];
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) v[u] = *at(page[u], from[u]);
#pragma unroll
        for (int u = 0; u < kMovePieces; u++) {
            const int to = j + u * step;
            page[u] = there(to) && from[u] != to ? table[to >> pool.page_shift] : -1;
        }
        if (j0 + step * kMovePieces < keep)
#pragma unroll
            for (int u = 0; u < kMovePieces; u++) from[u] = kept[there(next + u * step) ? next + u * step : 0];
        if (blocks == 1) __syncthreads();
        else cluster.sync();
#pragma unroll
        for (int u = 0; u < kMovePieces; u++)
            if (page[u] >= 0) *at(page[u], j + u * step) = v[u];
        // nothing to wait for: the next stretch reads behind what this one writes, and writes when all have read it
    }
}
// grid: (cluster, sequences * kv heads, planes: keys, values, their scales)
__global__ void __launch_bounds__(kMoveThreads, 3) kv4_move_kernel(Kv4Pool pool, Kv8Seqs seqs, EvictArgs a) {
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
    LC_CHECK(limit <= 1 << 30, LC_ERR_INVALID, "%s: limit=%d (2^30 at most)", call, limit);
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
    auto per_block = [&](int size) { return (slots + 128 * size - 1) / (128 * size) * 128; };
    auto bytes = [&](int size) { return (size_t)per_block(size) * 6; };
    int size = 1;
    while (size < kMostCluster && (2 * size * units <= 2 * sm_count() || bytes(size) > kSelectSmem)) size *= 2;
    if (bytes(size) <= kSelectSmem) {
        const bool wide = per_block(size) > 8192;   // blocks of so many sums are one for an SM
        const auto kern = wide ? kv4_select_kernel<1024> : kv4_select_kernel<512>;
        LC_CUDA(ensure_smem_limit((const void*)kern, bytes(size)));
        const cudaLaunchConfig_t cfg = clusters(dim3((unsigned)size, (unsigned)units), wide ? 1024 : 512, bytes(size), s, attr);
        LC_CUDA(cudaLaunchKernelEx(&cfg, kern, pool, seqs, a, (int)per_block(size)));
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
