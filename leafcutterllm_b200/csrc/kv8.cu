// The key/value cache in 8 bits: appending rows (with the position rotation on the way), reading rows back.
//
// A page holds page_tokens rows of one sequence for every kv head, as integers q with one f32 scale S per page and head: x ~ q S.
// An append gives a page and head the scale S = max(S_before, f32(A / 127)), A the largest finite magnitude of its new rows, S_before that of
// the rows that the page already holds (none: 0).  Those are rounded again where S grew: q <- rint(q S_before / S); new rows: q = rint(x / S).
//
// The keys' rotation, the quotients and their rounding are defined in 64 bits: an integer then depends on the definition alone and not on how
// a kernel orders its arithmetic, so that every implementation holds the same cache.  (f32 stands in for them where its bounds decide an integer.)  The angle comes from a table of turns per
// position, as 64-bit fractions of a turn: position * entry wraps around by itself, and what is left is the angle's fraction of a turn
// to 2^-64 of one, however far the position is (cos and sin of an f32 angle lose 2^-24 of the ANGLE: 0.06 at 10^6).
//
// Both kernels move bytes: an append reads its rows once from HBM (a page's second pass over them finds them in L1/L2) and writes a quarter or half of that.  Prompts
// are bound by the passes' instructions (57 % of the issue slots; 61 MB read at 1.2 TB/s), single tokens by the launch and a chain of loads: row_start, context, table, scale, rows.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include "lc_rope.cuh"
#include "lc_tma.cuh"

namespace lc {

int32_t DeviceScope::enter(const void* dev_ptr, const char* what) {
    cudaPointerAttributes a;
    const cudaError_t e = cudaPointerGetAttributes(&a, dev_ptr);
    if (e != cudaSuccess && !have_device()) return LC_ERR_CUDA;
    if (e != cudaSuccess || (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)) {
        (void)cudaGetLastError();
        set_error("%s: not a device pointer", what);
        return LC_ERR_INVALID;
    }
    int cur = 0;
    LC_CUDA(cudaGetDevice(&cur));
    if (a.device != cur && a.type == cudaMemoryTypeDevice) {
        LC_CUDA(cudaSetDevice(a.device));
        before = cur;
    }
    return LC_OK;
}

int32_t kv8_check(const char* call, const lc_kv8_cache* c, const lc_kv8_rows* r, uint32_t typ, int32_t n_rows, Kv8Pool* view, Kv8Seqs* seqs) {
    LC_CHECK(c && r, LC_ERR_INVALID, "%s: null cache or rows", call);
    LC_CHECK(typ == LC_TYPE_F32 || typ == LC_TYPE_F16 || typ == LC_TYPE_BF16, LC_ERR_UNSUPPORTED, "%s: type %u (f32, f16 and bf16 are taken)", call, typ);
    LC_CHECK(c->k_dev && c->v_dev && c->k_scale_dev && c->v_scale_dev, LC_ERR_INVALID, "%s: null pointer in the cache", call);
    LC_CHECK(((uintptr_t)c->k_dev | (uintptr_t)c->v_dev) % 16 == 0, LC_ERR_INVALID, "%s: the pools must be 16-byte aligned", call);
    LC_CHECK(c->n_pages > 0, LC_ERR_INVALID, "%s: n_pages=%d", call, c->n_pages);
    LC_CHECK(c->n_kv_heads > 0 && c->n_kv_heads <= 1024, LC_ERR_INVALID, "%s: n_kv_heads=%d (1 .. 1024)", call, c->n_kv_heads);
    LC_CHECK(c->head_dim >= 16 && c->head_dim <= 256 && c->head_dim % 16 == 0, LC_ERR_INVALID, "%s: head_dim=%d (a multiple of 16, 256 at most)", call, c->head_dim);
    int shift = 4;
    while (shift < 8 && (1 << shift) != c->page_tokens) shift++;
    LC_CHECK((1 << shift) == c->page_tokens, LC_ERR_INVALID, "%s: page_tokens=%d (16, 32, 64, 128 or 256)", call, c->page_tokens);
    LC_CHECK(r->n_seqs >= 0 && r->n_seqs <= kKv8MaxSeqs, LC_ERR_INVALID, "%s: n_seqs=%d (0 .. %d)", call, r->n_seqs, kKv8MaxSeqs);
    LC_CHECK(r->table_width >= 0 && ((int64_t)r->table_width << shift) <= (int64_t)1 << 30, LC_ERR_INVALID, "%s: table_width=%d (2^30 positions at most)", call, r->table_width);
    LC_CHECK(r->max_rows >= 0, LC_ERR_INVALID, "%s: max_rows=%d", call, r->max_rows);
    LC_CHECK(n_rows >= 0 && n_rows <= 1 << 24, LC_ERR_INVALID, "%s: n_rows=%d (0 .. 2^24)", call, n_rows);
    if (n_rows > 0 && r->n_seqs > 0)
        LC_CHECK(r->page_table_dev && r->ctx_dev && r->row_start_dev, LC_ERR_INVALID, "%s: null pointer in the rows", call);
    *view = Kv8Pool{(int8_t*)c->k_dev, (int8_t*)c->v_dev, c->k_scale_dev, c->v_scale_dev, c->n_pages, c->n_kv_heads, shift, c->head_dim};
    *seqs = Kv8Seqs{r->page_table_dev, r->ctx_dev, r->row_start_dev, r->status_dev, r->n_seqs, r->table_width, n_rows};
    return LC_OK;
}

namespace {

struct AppendArgs {
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    int64_t k_stride, v_stride, q_stride, qo_stride;
    int n_heads, half;            // half = rot_dim / 2
    const uint64_t* turns;
    int window, table_rows;       // rows of a block's window; rows that its table of rotations has room for
    int kv_slices;                // blocks of a window for the keys and values; the others are the queries'
};

__device__ __forceinline__ double finite_abs(double x) { return isfinite(x) ? fabs(x) : 0.0; }
// x / S, correctly rounded: inv = 1 / S is, and the remainder of the first quotient brings it there (Markstein); ties of x / S are ties then
__device__ __forceinline__ double quotient(double x, double scale, double inv) {
    const double q = x * inv;
    return fma(fma(-q, scale, x), inv, q);
}
// Added to 1.5 2^52, a number below 2^51 is rounded to a whole one, to the nearest even, which is then the sum's lower word.
// For finite x no larger than 127.5 S: what is left after a page's largest magnitude has made its scale (S of 0: inv is 0 as well).
__device__ __forceinline__ int near_int8(double x, double scale, double inv) {
    return max(-127, min(127, __double2loint(quotient(x, scale, inv) + 0x1.8p52)));
}
__device__ __forceinline__ int to_int8(double x, double scale, double inv) {
    if (!(fabs(x) < INFINITY)) return isnan(x) || inv == 0.0 ? 0 : x > 0.0 ? 127 : -127;
    return near_int8(x, scale, inv);
}

// four elements in a row
template <typename T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* p, float (&v)[4]) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
template <> __device__ __forceinline__ void load4<__half>(const __half* p, float (&v)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
template <> __device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u); v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    __align__(16) T t[4];
#pragma unroll
    for (int e = 0; e < 4; e++) t[e] = to_elem<T>(v[e]);
    if (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
}
// The rotations of rows pos0 .. pos0 + n - 1: (cosine, sine) of every pair.  Sine and cosine themselves for every eighth row and for the first
// eight turns; the rest are products of the two, 2^-52 off.  SPREAD: pair d lies at place (d mod 4) half / 4 + d / 4, so that lanes with four pairs each read
// neighbouring places.  They are kept as two f32 each, 2^-48 of them off.
// a pair's rotation in 64 bits
__device__ __forceinline__ void turned64(float u, float w, const float4& t, double& y0, double& y1) {
    const double c = (double)t.x + (double)t.y, s = (double)t.z + (double)t.w;
    y0 = u * c - w * s;
    y1 = u * s + w * c;
}
template <bool SPREAD>
__device__ __forceinline__ void fill_table(float4* tab, double2* bases, const uint64_t* __restrict__ turns, int half, int pos0, int n) {
    auto pair_at = [&](int at) {  // the pair at a place
        if (!SPREAD) return at;
        const int quarter = half >> 2, c = at / quarter;
        return (at - c * quarter) * 4 + c;
    };
    if (n <= 8) {
        for (int e = threadIdx.x; e < n * half; e += blockDim.x) {
            const int j = e / half;
            set_turn(tab[e], turn_of(turns[pair_at(e - j * half)], pos0 + j));
        }
        return;
    }
    const int n8 = (n + 7) >> 3;     // [n8 bases, then 8 first turns][half]
    for (int e = threadIdx.x; e < (n8 + 8) * half; e += blockDim.x) {
        const int j = e / half, at = e - j * half;
        bases[e] = turn_of(turns[pair_at(at)], j < n8 ? pos0 + j * 8 : j - n8);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n * half; e += blockDim.x) {
        const int j = e / half, at = e - j * half;
        const double2 x = bases[(j >> 3) * half + at], y = bases[(n8 + (j & 7)) * half + at];
        set_turn(tab[e], make_double2(x.x * y.x - x.y * y.y, x.x * y.y + x.y * y.x));
    }
}

// What of a group - the rows of one sequence in one page - a block serves.
struct Group {
    int row, cnt, pos, slot;
    size_t page_head;             // page * kv heads
    bool held;
};

// Keys and values of a group: an item is (keys or values, head) and belongs to one warp, which passes over its rows up to three times:
//   kMost   the rows' largest magnitude, of keys after their rotation, in f32;
//   kFine   of the rotated keys that may be the largest (a rotation is off by 2^-22 of the pair's length, at most 1.42 of the largest magnitude: those within 2^-19 of it), the
//           largest in 64 bits;
//   kInts   integers: x / S in f32 is within 2e-4 of the quotient (rotation 2^-22 of at most 180 S, product and inverse 2^-22 of 127.5), so that it gives the integer of
//           the 64-bit quotient unless it lies so near a half; eight elements with such a one among them, one group in 300, are taken in 64 bits.
// Rows with infinities or NaN, which the first maximum shows, and maxima and scales below 1e-30 go the long way, all in 64 bits.  Five prompts of 300 - 2,100 tokens, 8 kv heads and 32 of queries
// of 128, bf16: 171 us with everything in 64 bits and an element per lane, 44 now (a table of rotations 2.3 of a block's 12, each pass 2 to 4: their instructions).
enum : int { kMost, kFine, kInts };
struct Item {
    double top, scale, inv;
    float most, least, inv32;  // the largest magnitude in f32, what may be the largest in 64 bits, 1 / scale
    bool slow;
};
// Rows row0 .. row0 + cn - 1 of an item by one warp: a lane has four pairs (d, d + hd / 2) of a row, a warp as many rows at a time as it has lanes for.
template <typename T, int PASS, bool TURN>
__device__ __forceinline__ void rows_pass(Item& it, const T* rows, int64_t stride, int cn, int8_t* dst, int hd, const float4* tab) {
    const int lane = threadIdx.x & 31, lanes = hd >> 3, at_once = 32 / lanes, jl = lane / lanes, d = (lane - jl * lanes) * 4, other = hd >> 1, half = hd >> 1, quarter = hd >> 3;
    if (jl >= at_once) return;
    rows += d;
    for (int j0 = jl; j0 < cn; j0 += 2 * at_once) {
        float u[2][4], w[2][4];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const T* row = rows + (int64_t)min(j0 + b * at_once, cn - 1) * stride;
            load4(row, u[b]);
            load4(row + other, w[b]);
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int j = j0 + b * at_once;
            if (j >= cn) break;
            const float4* t = tab + j * half + (d >> 2);
            float y0[4], y1[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                y0[e] = u[b][e];
                y1[e] = w[b][e];
                if (TURN) {
                    const float4 cs = t[e * quarter];
                    y0[e] = u[b][e] * cs.x - w[b][e] * cs.z;
                    y1[e] = u[b][e] * cs.z + w[b][e] * cs.x;
                }
            }
            if (PASS == kMost) {
#pragma unroll
                for (int e = 0; e < 4; e++) it.most = max_nan(max_nan(it.most, fabsf(y0[e])), fabsf(y1[e]));
            } else if (PASS == kFine) {
                float here = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) here = fmaxf(here, fmaxf(fabsf(y0[e]), fabsf(y1[e])));
                if (it.slow || here >= it.least) {
#pragma unroll 1
                    for (int e = 0; e < 4; e++) {
                        double z0 = u[b][0], z1 = w[b][0];
                        if (TURN) turned64(u[b][0], w[b][0], t[e * quarter], z0, z1);
                        it.top = fmax(it.top, fmax(finite_abs(z0), finite_abs(z1)));
#pragma unroll
                        for (int k = 0; k < 3; k++) { u[b][k] = u[b][k + 1]; w[b][k] = w[b][k + 1]; }
                    }
                }
            } else {
                float r0[4], r1[4], off = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float q0 = y0[e] * it.inv32, q1 = y1[e] * it.inv32;
                    r0[e] = q0 + 12582912.0f;  // 1.5 2^23: rounded to a whole number, in the low bits
                    r1[e] = q1 + 12582912.0f;
                    off = fmaxf(off, fmaxf(fabsf(q0 - (r0[e] - 12582912.0f)), fabsf(q1 - (r1[e] - 12582912.0f))));
                }
                uint32_t b0 = pack4(__float_as_int(r0[0]), __float_as_int(r0[1]), __float_as_int(r0[2]), __float_as_int(r0[3]));
                uint32_t b1 = pack4(__float_as_int(r1[0]), __float_as_int(r1[1]), __float_as_int(r1[2]), __float_as_int(r1[3]));
                if (it.slow || !(off < 0.4998f)) {
                    b0 = b1 = 0;
#pragma unroll 1
                    for (int e = 0; e < 4; e++) {
                        double z0 = u[b][0], z1 = w[b][0];
                        if (TURN) turned64(u[b][0], w[b][0], t[e * quarter], z0, z1);
                        b0 |= (uint32_t)(to_int8(z0, it.scale, it.inv) & 0xff) << (8 * e);
                        b1 |= (uint32_t)(to_int8(z1, it.scale, it.inv) & 0xff) << (8 * e);
#pragma unroll
                        for (int k = 0; k < 3; k++) { u[b][k] = u[b][k + 1]; w[b][k] = w[b][k + 1]; }
                    }
                }
                int8_t* o = dst + (size_t)j * hd + d;
                *reinterpret_cast<uint32_t*>(o) = b0;
                *reinterpret_cast<uint32_t*>(o + other) = b1;
            }
        }
    }
}
// The same for any strides, alignment and rotated part of the dims, all in 64 bits.
template <typename T, int PASS>
__device__ __forceinline__ void rows_pass_plain(Item& it, const T* rows, int64_t stride, int cn, int8_t* dst, int hd, const float4* tab, int half) {
    const int lane = threadIdx.x & 31;
    for (int j = 0; j < cn; j++) {
        const T* row = rows + (int64_t)j * stride;
        int8_t* o = dst + (size_t)j * hd;
        for (int d = lane; d < half; d += 32) {
            double y0, y1;
            turned64(elem_f(row[d]), elem_f(row[d + half]), tab[j * half + d], y0, y1);
            if (PASS == kFine) {
                it.top = fmax(it.top, fmax(finite_abs(y0), finite_abs(y1)));
            } else {
                o[d] = (int8_t)to_int8(y0, it.scale, it.inv);
                o[d + half] = (int8_t)to_int8(y1, it.scale, it.inv);
            }
        }
        for (int d = 2 * half + lane; d < hd; d += 32) {
            const double y = elem_f(row[d]);
            if (PASS == kFine) it.top = fmax(it.top, finite_abs(y));
            else o[d] = (int8_t)to_int8(y, it.scale, it.inv);
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void append_kv(const Kv8Pool& pool, const AppendArgs& a, const Group& gr, float4* tab, double2* bases, int kv0, int kv1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int page = 1 << pool.page_shift, hd = pool.hd, half = a.half;
    const bool one_table = gr.cnt <= a.table_rows;
    const int items = gr.held ? 2 * (kv1 - kv0) : 0;
    if (one_table) {
        __syncthreads();  // the group before has done with the table
        fill_table<VEC>(tab, bases, a.turns, half, gr.pos, gr.cnt);
        __syncthreads();
    }
    // every warp takes as many turns as the one with most items: the table's refills are the block's
    const int rounds = (items + nw - 1) / nw;
    for (int round = 0; round < rounds; round++) {
        const int n = round * nw + warp;
        const bool mine = n < items;
        const bool is_k = n < (kv1 - kv0), turn = is_k && half > 0;
        const int h = kv0 + (is_k ? n : n - (kv1 - kv0));
        const int64_t stride = is_k ? a.k_stride : a.v_stride;
        const T* x = (const T*)(is_k ? a.k : a.v) + (int64_t)h * hd + (int64_t)gr.row * stride;
        const size_t ph = gr.page_head + h;
        int8_t* dst = (is_k ? pool.k : pool.v) + ph * page * hd;
        Item it;
        it.top = it.scale = it.inv = 0.0;
        it.most = it.least = it.inv32 = 0.0f;
        it.slow = !VEC;               // infinities or NaN among the rows, or a scale too small for f32
        auto pass = [&](auto which) {
            constexpr int PASS = decltype(which)::value;
            for (int c0 = 0; c0 < gr.cnt; c0 += a.table_rows) {
                const int cn = min(a.table_rows, gr.cnt - c0);
                if (!one_table) {
                    __syncthreads();
                    fill_table<VEC>(tab, bases, a.turns, half, gr.pos + c0, cn);
                    __syncthreads();
                }
                if (!mine || (PASS == kFine && !it.slow && !turn)) continue;
                const T* rows = x + (int64_t)c0 * stride;
                int8_t* to = dst + (size_t)(gr.slot + c0) * hd;
                if constexpr (!VEC) {
                    if (PASS != kMost) rows_pass_plain<T, PASS>(it, rows, stride, cn, to, hd, tab, turn ? half : 0);
                } else if (turn) {
                    rows_pass<T, PASS, true>(it, rows, stride, cn, to, hd, tab);
                } else {
                    rows_pass<T, PASS, false>(it, rows, stride, cn, to, hd, tab);
                }
            }
        };
        pass(std::integral_constant<int, kMost>());
        if (VEC) {
            it.slow = __any_sync(0xffffffffu, !(it.most < INFINITY));
            it.most = warp_max(it.most);
            it.slow = it.slow || it.most < 1e-30f;  // what follows of f32's relative errors does not hold next to its smallest numbers
            it.least = it.most * (1.0f - 0x1p-19f);
            it.top = it.slow || turn ? 0.0 : (double)it.most;
        }
        pass(std::integral_constant<int, kFine>());
        if (mine) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) it.top = fmax(it.top, __shfl_xor_sync(0xffffffffu, it.top, o));
            float* sp = (is_k ? pool.k_scale : pool.v_scale) + ph;
            const float before = gr.slot > 0 ? *sp : 0.0f;
            const float now = fmaxf(before, (float)(it.top / 127.0));
            it.scale = (double)now;
            it.inv = now > 0.0f ? 1.0 / it.scale : 0.0;
            it.slow = it.slow || !(now > 1e-30f);
            it.inv32 = (float)it.inv;
            if (gr.slot > 0 && now != before) {
                for (int e = lane * 4; e < gr.slot * hd; e += 128) {
                    char4 b = *reinterpret_cast<char4*>(dst + e);
                    b.x = (signed char)(int)rint((double)b.x * (double)before / (double)now);
                    b.y = (signed char)(int)rint((double)b.y * (double)before / (double)now);
                    b.z = (signed char)(int)rint((double)b.z * (double)before / (double)now);
                    b.w = (signed char)(int)rint((double)b.w * (double)before / (double)now);
                    *reinterpret_cast<char4*>(dst + e) = b;
                }
            }
            __syncwarp();
            if (lane == 0) *sp = now;
        }
        pass(std::integral_constant<int, kInts>());
    }
}

// The queries of a group, heads q0 .. q1 - 1.
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_q(const Kv8Pool& pool, const AppendArgs& a, const Group& gr, float4* tab, double2* bases, int q0, int q1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5, hd = pool.hd, half = a.half;
    for (int c0 = 0; c0 < gr.cnt; c0 += a.table_rows) {
        const int cn = min(a.table_rows, gr.cnt - c0);
        __syncthreads();
        fill_table<VEC>(tab, bases, a.turns, half, gr.pos + c0, cn);
        __syncthreads();
        if constexpr (VEC) {
            // the lanes and pairs as above; a lane keeps its rotations for four heads, whose loads go out together
            constexpr int B = 4;
            const int lanes = hd >> 3, at_once = 32 / lanes, jl = lane / lanes, d = (lane - jl * lanes) * 4, other = hd >> 1;
            const int quads = (q1 - q0 + B - 1) / B, rows = (cn + at_once - 1) / at_once;
            for (int e = warp; e < rows * quads; e += nw) {
                const int rj = e / quads, j = rj * at_once + jl, h = q0 + B * (e - rj * quads);
                if (jl >= at_once || j >= cn) continue;
                const int64_t row = gr.row + c0 + j;
                const T* src = (const T*)a.q + row * a.q_stride + (int64_t)h * hd + d;
                T* o = (T*)a.q_out + row * a.qo_stride + (int64_t)h * hd + d;
                float u[B][4], w[B][4];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const int64_t at = (int64_t)min(b, q1 - 1 - h) * hd;
                    load4(src + at, u[b]);
                    load4(src + at + other, w[b]);
                }
                float4 t[4];
#pragma unroll
                for (int k = 0; k < 4; k++) t[k] = half ? tab[j * half + k * (half >> 2) + (d >> 2)] : make_float4(1.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int b = 0; b < B; b++) {
                    if (h + b >= q1) break;
                    float y0[4], y1[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        y0[k] = turned(u[b][k], w[b][k], t[k].x, t[k].y, t[k].z, t[k].w);
                        y1[k] = turned(u[b][k], -w[b][k], t[k].z, t[k].w, t[k].x, t[k].y);
                    }
                    store4(o + (int64_t)b * hd, y0);
                    store4(o + (int64_t)b * hd + other, y1);
                }
            }
        } else {
            for (int e = warp; e < cn * (q1 - q0); e += nw) {
                const int j = e / (q1 - q0), h = q0 + e - j * (q1 - q0);
                const T* src = (const T*)a.q + (int64_t)(gr.row + c0 + j) * a.q_stride + (int64_t)h * hd;
                T* o = (T*)a.q_out + (int64_t)(gr.row + c0 + j) * a.qo_stride + (int64_t)h * hd;
                for (int d = lane; d < half; d += 32) {
                    const float u = elem_f(src[d]), w = elem_f(src[d + half]);
                    const float4 t = tab[j * half + d];
                    o[d] = to_elem<T>(turned(u, w, t.x, t.y, t.z, t.w));
                    o[d + half] = to_elem<T>(turned(u, -w, t.z, t.w, t.x, t.y));
                }
                for (int d = 2 * half + lane; d < hd; d += 32) o[d] = src[d];
            }
        }
    }
}

// grid: (windows of rows, slices of kv heads and then of query heads).  A block serves the groups that begin in its window.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 3) kv8_append_kernel(Kv8Pool pool, Kv8Seqs seqs, AppendArgs a) {
    extern __shared__ float4 tab[];
    double2* const bases = reinterpret_cast<double2*>(tab + a.table_rows * a.half);
    if (blockIdx.x == 0 && blockIdx.y == 0) kv8_check_seqs(seqs, pool);
    const int page = 1 << pool.page_shift;
    const bool kv = (int)blockIdx.y < a.kv_slices;
    const int slices = kv ? a.kv_slices : gridDim.y - a.kv_slices, sl = kv ? blockIdx.y : blockIdx.y - a.kv_slices, heads = kv ? pool.n_kv : a.n_heads;
    const int h0 = heads * sl / slices, h1 = heads * (sl + 1) / slices;
    int r = blockIdx.x * a.window;
    const int r_end = min(r + a.window, seqs.n_rows);
    while (r < r_end) {
        int next;
        const int i = kv8_seq_of_row(seqs, r, next);
        if (i < 0) { r = next; continue; }
        int first, n;
        kv8_span(seqs, i, first, n);
        const int ctx = seqs.ctx[i], end = first + n;
        if (!kv8_in_table(seqs, pool, ctx, n)) { r = end; continue; }
        const int32_t* table = seqs.table + (size_t)i * seqs.width;
        if (r != first) r = min(end, r + ((-(ctx + r - first)) & (page - 1)));  // inside a group that another window has: to the next page or sequence
        while (r < min(r_end, end)) {
            const int pos = ctx + (r - first), slot = pos & (page - 1);
            const int number = table[pos >> pool.page_shift];
            Group gr;
            gr.row = r;
            gr.cnt = min(page - slot, end - r);
            gr.pos = pos;
            gr.slot = slot;
            gr.held = number >= 0 && number < pool.n_pages;
            gr.page_head = (size_t)(gr.held ? number : 0) * pool.n_kv;
            if (kv) {
                if (!gr.held && threadIdx.x == 0) kv8_raise(seqs, i);
                append_kv<T, VEC>(pool, a, gr, tab, bases, h0, h1);
            } else {
                rotate_q<T, VEC>(pool, a, gr, tab, bases, h0, h1);
            }
            r += gr.cnt;
        }
    }
}

struct ReadArgs {
    void* k;
    void* v;
    int64_t k_stride, v_stride;
    int vec;  // whether 16 elements are stored in 16-byte pieces
};

// A warp takes 32 pieces of 16 integers (of the keys', then the values' heads) of a row.
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8Pool pool, Kv8Seqs seqs, ReadArgs a) {
    if (blockIdx.x == 0) kv8_check_seqs(seqs, pool);
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    const int pieces = pool.hd >> 4, all = pool.n_kv * pieces, parts = (2 * all + 31) >> 5;
    const int64_t units = (int64_t)seqs.n_rows * parts;
    for (int64_t unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); unit < units; unit += warps) {
        const int r = (int)(unit / parts), e = (int)(unit - (int64_t)r * parts) * 32 + lane;
        int next;
        const int i = kv8_seq_of_row(seqs, r, next);
        if (i < 0) continue;
        int first, n;
        kv8_span(seqs, i, first, n);
        const int ctx = seqs.ctx[i];
        const bool inside = kv8_in_table(seqs, pool, ctx, n);
        const int pos = inside ? ctx + (r - first) : 0;
        const int number = inside ? seqs.table[(size_t)i * seqs.width + (pos >> pool.page_shift)] : -1;
        const bool held = number >= 0 && number < pool.n_pages;
        if (!held && lane == 0) kv8_raise(seqs, i);
        const int slot = pos & ((1 << pool.page_shift) - 1);
        const bool is_k = e < all;
        T* out = (T*)(is_k ? a.k : a.v);
        if (e >= 2 * all || !out) continue;
        const int f = is_k ? e : e - all, h = f / pieces, c = f - h * pieces;
        float scale = __int_as_float(0x7fffffff);
        uint4 w = make_uint4(0, 0, 0, 0);
        if (held) {
            const size_t ph = (size_t)number * pool.n_kv + h;
            w = *reinterpret_cast<const uint4*>((is_k ? pool.k : pool.v) + ((ph << pool.page_shift) + slot) * pool.hd + c * 16);
            scale = (is_k ? pool.k_scale : pool.v_scale)[ph];
        }
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        __align__(16) T t[16];
#pragma unroll
        for (int b = 0; b < 16; b++) t[b] = to_elem<T>((float)(int8_t)(words[b >> 2] >> (8 * (b & 3))) * scale);
        out += (int64_t)r * (is_k ? a.k_stride : a.v_stride) + (int64_t)h * pool.hd + c * 16;
        if (a.vec) {
#pragma unroll
            for (int b = 0; b < (int)sizeof(T); b++) reinterpret_cast<uint4*>(out)[b] = reinterpret_cast<const uint4*>(t)[b];
        } else {
#pragma unroll
            for (int b = 0; b < 16; b++) out[b] = t[b];
        }
    }
}

template <typename T>
int32_t append_as(const Kv8Pool& pool, const Kv8Seqs& seqs, AppendArgs a, int max_rows, cudaStream_t s) {
    const int page = 1 << pool.page_shift;
    // a window about as long as a sequence's rows, a page at most: single tokens have a block each, prompts one for each page
    int win = 1;
    while (win * 2 <= page && win * 2 <= seqs.n_rows / seqs.n_seqs) win *= 2;
    a.window = win;
    a.table_rows = 1;
    while (a.table_rows < 32 && a.table_rows < page && a.table_rows < max_rows) a.table_rows *= 2;
    const int windows = (seqs.n_rows + win - 1) / win;
    auto slices_of = [&](int heads, int least) {
        int n = (2 * sm_count() + windows - 1) / windows;
        n = std::min(n, (heads + least - 1) / least);
        return std::max(n, 1);
    };
    const bool vec = pool.hd % 8 == 0 && pool.hd <= 256 && (a.half == 0 || 2 * a.half == pool.hd) && rows_aligned(a.k, a.k_stride, sizeof(T), 4 * sizeof(T)) &&
                     rows_aligned(a.v, a.v_stride, sizeof(T), 4 * sizeof(T)) &&
                     (!a.q || (rows_aligned(a.q, a.q_stride, sizeof(T), 4 * sizeof(T)) && rows_aligned(a.q_out, a.qo_stride, sizeof(T), 4 * sizeof(T))));
    // rows of the table, and behind it every eighth and the eight first turns of more than eight rows
    const size_t smem = (size_t)(a.table_rows + (a.table_rows > 8 ? a.table_rows / 8 + 8 : 0)) * a.half * sizeof(float4);
    a.kv_slices = slices_of(pool.n_kv, 4);  // a block's eight warps have an item each
    const int slices = a.kv_slices + (a.q ? slices_of(a.n_heads, 4) : 0);
    const auto kern = vec ? kv8_append_kernel<T, true> : kv8_append_kernel<T, false>;
    LC_CUDA(ensure_smem_limit((const void*)kern, smem));
    kern<<<dim3((unsigned)windows, (unsigned)slices), 256, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
template <typename T>
int32_t read_as(const Kv8Pool& pool, const Kv8Seqs& seqs, ReadArgs a, cudaStream_t s) {
    a.vec = (!a.k || rows_aligned(a.k, a.k_stride, sizeof(T), 16)) && (!a.v || rows_aligned(a.v, a.v_stride, sizeof(T), 16));
    const int64_t units = (int64_t)seqs.n_rows * ((2 * pool.n_kv * (pool.hd >> 4) + 31) >> 5);
    const int blocks = (int)std::min<int64_t>((units + 7) / 8, (int64_t)8 * sm_count());
    kv8_read_kernel<T><<<blocks, 256, 0, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_rope_turns(double theta, int32_t rot_dim, uint64_t* out) {
    LC_CHECK(out, LC_ERR_INVALID, "lc_rope_turns: null pointer");
    LC_CHECK(rot_dim >= 0 && rot_dim % 2 == 0, LC_ERR_INVALID, "lc_rope_turns: rot_dim=%d must be even", rot_dim);
    LC_CHECK(theta >= 1.0 && std::isfinite(theta), LC_ERR_INVALID, "lc_rope_turns: theta=%g (1 or more)", theta);
    const long double turn = 6.283185307179586476925286766559L;
    for (int32_t d = 0; d < rot_dim / 2; d++) {
        const long double f = powl((long double)theta, -2.0L * d / rot_dim) / turn;  // below 1 / (2 pi)
        const long double whole = f * 0x1p64L;
        out[d] = (uint64_t)whole + (whole - (long double)(uint64_t)whole >= 0.5L ? 1u : 0u);
    }
    return LC_OK;
}

int32_t lc_kv8_append_dev(const lc_kv8_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, const void* k_dev,
                          int64_t k_stride, const void* v_dev, int64_t v_stride, const void* q_dev, int64_t q_stride, void* q_out_dev,
                          int64_t q_out_stride, int32_t n_heads, const uint64_t* turns_dev, int32_t rot_dim, void* stream_) {
    Kv8Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv8_check("lc_kv8_append_dev", cache, rows, typ, n_rows, &pool, &seqs));
    LC_CHECK(rot_dim >= 0 && rot_dim <= pool.hd && rot_dim % 2 == 0, LC_ERR_INVALID, "lc_kv8_append_dev: rot_dim=%d (even, head_dim %d at most)", rot_dim, pool.hd);
    LC_CHECK(rot_dim == 0 || turns_dev, LC_ERR_INVALID, "lc_kv8_append_dev: a rotation needs its table");
    if (n_rows == 0 || seqs.n_seqs == 0) return LC_OK;
    const int64_t row = (int64_t)pool.n_kv * pool.hd;
    LC_CHECK(k_dev && v_dev, LC_ERR_INVALID, "lc_kv8_append_dev: null keys or values");
    LC_CHECK(k_stride >= row && v_stride >= row, LC_ERR_INVALID, "lc_kv8_append_dev: rows of keys or values overlap (strides %lld, %lld below %lld)", (long long)k_stride, (long long)v_stride, (long long)row);
    if (q_dev) {
        LC_CHECK(q_out_dev, LC_ERR_INVALID, "lc_kv8_append_dev: queries without a place for them");
        LC_CHECK(n_heads > 0 && n_heads <= 65536, LC_ERR_INVALID, "lc_kv8_append_dev: n_heads=%d", n_heads);
        LC_CHECK(q_stride >= (int64_t)n_heads * pool.hd && q_out_stride >= (int64_t)n_heads * pool.hd, LC_ERR_INVALID, "lc_kv8_append_dev: rows of queries overlap");
    }
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_kv8_append_dev: cache"));
    AppendArgs a{k_dev, v_dev, q_dev, q_out_dev, k_stride, v_stride, q_stride, q_out_stride, q_dev ? n_heads : 0, rot_dim / 2, turns_dev, 0, 0, 0};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return append_as<float>(pool, seqs, a, rows->max_rows, s);
    if (typ == LC_TYPE_F16) return append_as<__half>(pool, seqs, a, rows->max_rows, s);
    return append_as<__nv_bfloat16>(pool, seqs, a, rows->max_rows, s);
}

int32_t lc_kv8_read_dev(const lc_kv8_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, void* k_out_dev,
                        int64_t k_stride, void* v_out_dev, int64_t v_stride, void* stream_) {
    Kv8Pool pool;
    Kv8Seqs seqs;
    LC_TRY(kv8_check("lc_kv8_read_dev", cache, rows, typ, n_rows, &pool, &seqs));
    const int64_t row = (int64_t)pool.n_kv * pool.hd;
    LC_CHECK((!k_out_dev || k_stride >= row) && (!v_out_dev || v_stride >= row), LC_ERR_INVALID, "lc_kv8_read_dev: rows overlap");
    if (n_rows == 0 || seqs.n_seqs == 0 || (!k_out_dev && !v_out_dev)) return LC_OK;
    DeviceScope dev;
    LC_TRY(dev.enter(cache->k_dev, "lc_kv8_read_dev: cache"));
    ReadArgs a{k_out_dev, v_out_dev, k_stride, v_stride, 0};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return read_as<float>(pool, seqs, a, s);
    if (typ == LC_TYPE_F16) return read_as<__half>(pool, seqs, a, s);
    return read_as<__nv_bfloat16>(pool, seqs, a, s);
}

}  // extern "C"
