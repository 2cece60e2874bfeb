// The key/value cache in 8 bits: appending rows (with the position rotation on the way), reading rows back.
//
// A page holds page_tokens rows of one sequence for every kv head, as integers q with one f32 scale S per page and head: x ~ q S.
// An append gives a page and head the scale S = max(S_before, f32(A / 127)), A the largest finite magnitude of its new rows, S_before that of
// the rows that the page already holds (none: 0).  Those are rounded again where S grew: q <- rint(q S_before / S); new rows: q = rint(x / S).
//
// The keys' rotation, the quotients and their rounding are done in 64 bits: an integer then depends on the definition alone and not on how
// a kernel orders its arithmetic, so that every implementation holds the same cache.  The angle comes from a table of turns per
// position, as 64-bit fractions of a turn: position * entry wraps around by itself, and what is left is the angle's fraction of a turn
// to 2^-64 of one, however far the position is (cos and sin of an f32 angle lose 2^-24 of the ANGLE: 0.06 at 10^6).
//
// Both kernels move bytes: an append reads its rows once from HBM (a page's second pass over them finds them in L1/L2) and writes a quarter or half of that.
#include <cmath>
#include <cstring>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
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
};

__device__ __forceinline__ double finite_abs(double x) { return isfinite(x) ? fabs(x) : 0.0; }
// x / S as an integer of 8 bits; inv = 1 / S in 64 bits (0 where S is 0): one rounding more than the quotient, 2^-53 of it
__device__ __forceinline__ int to_int8(double x, double inv) {
    if (isnan(x) || inv == 0.0) return 0;
    return (int)rint(fmin(fmax(x * inv, -127.0), 127.0));
}

// The rotations of rows pos0 .. pos0 + n - 1: (cosine, sine) of every pair.
__device__ __forceinline__ void fill_table(double2* tab, const uint64_t* __restrict__ turns, int half, int pos0, int n) {
    for (int e = threadIdx.x; e < n * half; e += blockDim.x) {
        const int j = e / half, d = e - j * half;
        const int64_t frac = (int64_t)((uint64_t)(pos0 + j) * turns[d]);
        double s, c;
        sincospi((double)frac * 0x1p-63, &s, &c);  // frac 2^-64 turns = frac 2^-63 pi
        tab[e] = make_double2(c, s);
    }
}

// grid: (windows of rows, slices of heads).  A block serves the groups that begin in its window; a group is the rows of one sequence
// in one page.  An item is a (keys or values, head) of the group and belongs to one warp, which passes over its rows twice: largest
// magnitude, then integers.  The rotations are taken once for all heads of the slice.
template <typename T>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8Pool pool, Kv8Seqs seqs, AppendArgs a) {
    extern __shared__ double2 tab[];
    if (blockIdx.x == 0 && blockIdx.y == 0) kv8_check_seqs(seqs, pool);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int page = 1 << pool.page_shift, hd = pool.hd, half = a.half, rot = 2 * half;
    const int slices = gridDim.y, sl = blockIdx.y;
    const int kv0 = (int)((long long)pool.n_kv * sl / slices), kv1 = (int)((long long)pool.n_kv * (sl + 1) / slices);
    const int q0 = (int)((long long)a.n_heads * sl / slices), q1 = (int)((long long)a.n_heads * (sl + 1) / slices);
    int r = blockIdx.x * a.window;
    const int r_end = min(r + a.window, seqs.n_rows);
    while (r < r_end) {
        const int i = kv8_seq_of_row(seqs, r);
        if (i < 0) { r++; continue; }
        int first, n;
        kv8_span(seqs, i, first, n);
        const int ctx = seqs.ctx[i];
        if (!kv8_in_table(seqs, pool, ctx, n)) { r = first + n; continue; }
        const int pos = ctx + (r - first), slot = pos & (page - 1);
        if (slot != 0 && r != first) { r += min(page - slot, first + n - r); continue; }  // inside a group that another window has
        const int cnt = min(page - slot, first + n - r);
        const int number = seqs.table[(size_t)i * seqs.width + (pos >> pool.page_shift)];
        const bool held = number >= 0 && number < pool.n_pages;
        if (!held && threadIdx.x == 0) kv8_raise(seqs, i);
        const bool one_table = cnt <= a.table_rows;
        const int items = held ? 2 * (kv1 - kv0) : 0;
        if (one_table) {
            __syncthreads();  // the group before has done with the table
            fill_table(tab, a.turns, half, pos, cnt);
            __syncthreads();
        }
        // every warp takes as many turns as the one with most items: the table's refills are the block's
        const int rounds = (items + nw - 1) / nw;
        for (int round = 0; round < rounds; round++) {
            const int it = round * nw + warp;
            const bool mine = it < items;
            const bool is_k = it < (kv1 - kv0);
            const int h = kv0 + (is_k ? it : it - (kv1 - kv0));
            const T* x = (const T*)(is_k ? a.k : a.v) + (int64_t)h * hd;
            const int64_t stride = is_k ? a.k_stride : a.v_stride;
            const int hf = is_k ? half : 0, rt = is_k ? rot : 0;
            const size_t ph = (size_t)number * pool.n_kv + h;
            int8_t* dst = (is_k ? pool.k : pool.v) + ph * page * hd;
            double top = 0.0, inv = 0.0;
            for (int pass = 0; pass < 2; pass++) {
                for (int c0 = 0; c0 < cnt; c0 += a.table_rows) {
                    const int cn = min(a.table_rows, cnt - c0);
                    if (!one_table) {
                        __syncthreads();
                        fill_table(tab, a.turns, half, pos + c0, cn);
                        __syncthreads();
                    }
                    if (!mine) continue;
                    for (int j = 0; j < cn; j++) {
                        const T* row = x + (int64_t)(r + c0 + j) * stride;
                        int8_t* o = dst + (size_t)(slot + c0 + j) * hd;
                        for (int d = lane; d < hf; d += 32) {
                            const double u = elem_f(row[d]), w = elem_f(row[d + hf]);
                            const double2 cs = tab[j * hf + d];
                            const double y0 = u * cs.x - w * cs.y, y1 = u * cs.y + w * cs.x;
                            if (pass == 0) {
                                top = fmax(top, fmax(finite_abs(y0), finite_abs(y1)));
                            } else {
                                o[d] = (int8_t)to_int8(y0, inv);
                                o[d + hf] = (int8_t)to_int8(y1, inv);
                            }
                        }
                        for (int d = rt + lane; d < hd; d += 32) {
                            const double y = elem_f(row[d]);
                            if (pass == 0) top = fmax(top, finite_abs(y));
                            else o[d] = (int8_t)to_int8(y, inv);
                        }
                    }
                }
                if (pass == 0 && mine) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
                    float* sp = (is_k ? pool.k_scale : pool.v_scale) + ph;
                    const float before = slot > 0 ? *sp : 0.0f;
                    const float now = fmaxf(before, (float)(top / 127.0));
                    inv = now > 0.0f ? 1.0 / (double)now : 0.0;
                    if (slot > 0 && now != before) {
                        for (int e = lane * 4; e < slot * hd; e += 128) {
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
            }
        }
        if (a.q) {
            for (int c0 = 0; c0 < cnt; c0 += a.table_rows) {
                const int cn = min(a.table_rows, cnt - c0);
                if (!one_table) {
                    __syncthreads();
                    fill_table(tab, a.turns, half, pos + c0, cn);
                    __syncthreads();
                }
                for (int e = warp; e < cn * (q1 - q0); e += nw) {
                    const int j = e / (q1 - q0), h = q0 + e - j * (q1 - q0);
                    const T* src = (const T*)a.q + (int64_t)(r + c0 + j) * a.q_stride + (int64_t)h * hd;
                    T* o = (T*)a.q_out + (int64_t)(r + c0 + j) * a.qo_stride + (int64_t)h * hd;
                    for (int d = lane; d < half; d += 32) {
                        const float u = elem_f(src[d]), w = elem_f(src[d + half]);
                        const double2 cs = tab[j * half + d];
                        o[d] = to_elem<T>((float)(u * cs.x - w * cs.y));
                        o[d + half] = to_elem<T>((float)(u * cs.y + w * cs.x));
                    }
                    for (int d = rot + lane; d < hd; d += 32) o[d] = src[d];
                }
            }
        }
        r += cnt;
    }
}

struct ReadArgs {
    void* k;
    void* v;
    int64_t k_stride, v_stride;
    int vec;  // whether 16 elements are stored in 16-byte pieces
};

// A warp per row: 16 integers of a head per lane.
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8Pool pool, Kv8Seqs seqs, ReadArgs a) {
    if (blockIdx.x == 0) kv8_check_seqs(seqs, pool);
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    const int pieces = pool.hd >> 4, all = pool.n_kv * pieces;
    for (int r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < seqs.n_rows; r += warps) {
        const int i = kv8_seq_of_row(seqs, r);
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
        for (int e = lane; e < 2 * all; e += 32) {
            const bool is_k = e < all;
            T* out = (T*)(is_k ? a.k : a.v);
            if (!out) continue;
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
    int slices = (2 * sm_count() + windows - 1) / windows;
    if (slices > pool.n_kv) slices = pool.n_kv;
    if (slices < 1) slices = 1;
    const size_t smem = (size_t)a.table_rows * a.half * sizeof(double2);
    LC_CUDA(ensure_smem_limit((const void*)kv8_append_kernel<T>, smem));
    kv8_append_kernel<T><<<dim3((unsigned)windows, (unsigned)slices), 256, smem, s>>>(pool, seqs, a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}
template <typename T>
int32_t read_as(const Kv8Pool& pool, const Kv8Seqs& seqs, ReadArgs a, cudaStream_t s) {
    a.vec = (!a.k || rows_aligned(a.k, a.k_stride, sizeof(T), 16)) && (!a.v || rows_aligned(a.v, a.v_stride, sizeof(T), 16));
    int blocks = (seqs.n_rows + 7) / 8;
    if (blocks > 8 * sm_count()) blocks = 8 * sm_count();
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
    AppendArgs a{k_dev, v_dev, q_dev, q_out_dev, k_stride, v_stride, q_stride, q_out_stride, q_dev ? n_heads : 0, rot_dim / 2, turns_dev, 0, 0};
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
