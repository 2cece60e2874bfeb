// Rotary positions as an operator of their own: rows of heads turned by their positions, in either layout of the pairs, over a part of the head, with frequencies
// scaled for long contexts; and the tables of turns.
//
//   y_a = m (a cos t - b sin t), y_b = m (a sin t + b cos t), t = 2 pi frac(position * turns[p])
//
// A block takes a few rows and a share of their heads: first the rows' sines and cosines, once for all heads and of both tensors (64 bits, kept as two f32 each
// for f32 outputs and as one for 16-bit ones), then eight pairs of four heads a thread (two in f32),
// which share what the table says.  It moves bytes: each element is read and written once.  8,192 rows of 32 and 8 heads of 128 in bf16, 96 dims turned as neighbours: 35.4 us, 168 MB at 4.7 TB/s (a first, simple
// kernel: 53).  What bounds it is the loads' latency at three blocks on an SM, a third of its warps (80 registers); the instructions take a third of the issue slots.  Two heads a thread, 37 to 47 us; four blocks, 42, for
// their registers spill.  One row of 36 heads in f32: 4.2 us, a launch and sine and cosine in 64 bits.
#include <algorithm>
#include <cmath>
#include "lc_kv8.cuh"
#include "lc_kernels.h"
#include "lc_rope.cuh"

namespace lc {

namespace {

struct RopeTensor {
    const void* in;
    void* out;
    int64_t in_stride, out_stride;
    int heads;
};
struct RopeArgs {
    RopeTensor x, y;
    const int64_t* positions;
    const uint64_t* turns;
    int n_rows, rows;             // of the call, of a block
    int half, hd;                 // half = rot_dim / 2
    bool interleaved, inverse;
    double magnitude;
};

constexpr int kRopeThreads = 256;

// grid: (groups of rows, shares of the heads of x and y)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeArgs a) {
    using Entry = typename TurnEntry<T>::type;
    extern __shared__ __align__(16) unsigned char smem[];
    Entry* const tab = reinterpret_cast<Entry*>(smem);
    const int row0 = blockIdx.x * a.rows, rows = min(a.rows, a.n_rows - row0);
    const int heads = a.x.heads + a.y.heads, h0 = heads * blockIdx.y / gridDim.y, h1 = heads * (blockIdx.y + 1) / gridDim.y, mine = h1 - h0;
    const int n8 = (a.half + 7) >> 3;
    if (VEC && (int)threadIdx.x < rows) {
        const int x1 = min(h1, a.x.heads), y0 = max(h0, a.x.heads);
        if (h0 < x1) prefetch_l2((const T*)a.x.in + (row0 + threadIdx.x) * a.x.in_stride + (int64_t)h0 * a.hd, (uint32_t)((x1 - h0) * a.hd * sizeof(T)));
        if (y0 < h1) prefetch_l2((const T*)a.y.in + (row0 + threadIdx.x) * a.y.in_stride + (int64_t)(y0 - a.x.heads) * a.hd, (uint32_t)((h1 - y0) * a.hd * sizeof(T)));
    }
    const Divider by_half(a.half);
    for (int e = threadIdx.x; e < rows * a.half; e += kRopeThreads) {
        const int j = by_half(e), p = e - j * a.half;
        double2 t = turn_of(a.turns[p], a.positions[row0 + j]);
        t.x *= a.magnitude;
        t.y *= a.inverse ? -a.magnitude : a.magnitude;
        put_turn(tab[j * 8 * n8 + turn_place(p, n8)], t);
    }
    __syncthreads();
    // a row has its own share of the threads, whole warps
    const int share = kRopeThreads / a.rows, j = threadIdx.x / share, at = threadIdx.x - j * share;
    if (j >= rows) return;
    const Entry* const row = tab + j * 8 * n8;
    const T* const x_in = (const T*)a.x.in + (int64_t)(row0 + j) * a.x.in_stride;
    const T* const y_in = (const T*)a.y.in + (int64_t)(row0 + j) * a.y.in_stride;
    T* const x_out = (T*)a.x.out + (int64_t)(row0 + j) * a.x.out_stride;
    T* const y_out = (T*)a.y.out + (int64_t)(row0 + j) * a.y.out_stride;
    auto head_at = [&](int h, const T*& in, T*& out) {
        const bool x = h < a.x.heads;
        const int64_t off = (int64_t)(x ? h : h - a.x.heads) * a.hd;
        in = (x ? x_in : y_in) + off;
        out = (x ? x_out : y_out) + off;
    };
    const T* in;
    T* out;
    if constexpr (VEC) {
        // groups of heads of one tensor: x's that are in [h0, h1), then y's
        constexpr int B = kTurnHeads<T>;
        const int x0 = min(h0, a.x.heads), x1 = min(h1, a.x.heads), groups_x = (x1 - x0 + B - 1) / B;
        const int y0 = max(h0, a.x.heads), y1 = max(h1, a.x.heads), groups = groups_x + (y1 - y0 + B - 1) / B;
        const int pairs = a.half >> 3, copies = (a.hd - 2 * a.half) >> 3;
        const Divider by_pairs(pairs), by_copies(copies);
        for (int e = at; e < groups * pairs; e += share) {
            const int gr = by_pairs(e), h = gr < groups_x ? x0 + gr * B : y0 + (gr - groups_x) * B, n = min(B, (gr < groups_x ? x1 : y1) - h);
            head_at(h, in, out);
            turn_item(in, out, a.hd, n, e - gr * pairs, a.half, a.interleaved, row, n8);
        }
        // what is not turned
        for (int e = at; e < mine * copies; e += share) {
            const int h = by_copies(e);
            head_at(h0 + h, in, out);
            if (in != out) copy_item(in, out, e - h * copies, a.half);
        }
    } else {
        const int items = a.hd - a.half;
        for (int e = at; e < mine * items; e += share) {
            const int h = e / items;
            head_at(h0 + h, in, out);
            turn_item_plain(in, out, e - h * items, a.half, a.interleaved, row, n8);
        }
    }
}

template <typename T> int32_t rope_as(RopeArgs a, cudaStream_t s) {
    const int heads = a.x.heads + a.y.heads;
    // a block's table is made once for all of its heads, so it has all heads of its rows, and as many rows (8 at most) as leave four blocks for each SM; few rows: heads apart
    a.rows = 1;
    while (a.rows < 8 && 2 * a.rows <= a.n_rows / (4 * sm_count())) a.rows *= 2;
    while (a.rows > 1 && (size_t)a.rows * (a.half + 7) * sizeof(typename TurnEntry<T>::type) > 24 * 1024) a.rows /= 2;
    const int groups = (a.n_rows + a.rows - 1) / a.rows;
    const int slices = std::max(1, std::min({(2 * sm_count() + groups - 1) / groups, (heads + 7) / 8, 64}));
    auto fits = [&](const RopeTensor& t) { return t.heads == 0 || (rows_aligned(t.in, t.in_stride, sizeof(T), 16) && rows_aligned(t.out, t.out_stride, sizeof(T), 16)); };
    const bool vec = a.hd % 8 == 0 && a.half % 8 == 0 && fits(a.x) && fits(a.y);
    const size_t smem = (size_t)a.rows * ((a.half + 7) / 8 * 8) * sizeof(typename TurnEntry<T>::type);
    const auto kern = vec ? rope_kernel<T, true> : rope_kernel<T, false>;
    kern<<<dim3((unsigned)groups, (unsigned)slices), kRopeThreads, smem, s>>>(a);
    LC_CUDA(cudaGetLastError());
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" {

int32_t lc_rope_turns_scaled(double theta, int32_t rot_dim, int32_t kind, double factor, int32_t original, double fast, double slow, uint64_t* out, double* magnitude) {
    const char* call = "lc_rope_turns_scaled";
    LC_CHECK(out && magnitude, LC_ERR_INVALID, "%s: null pointer", call);
    LC_CHECK(kind >= LC_ROPE_PLAIN && kind <= LC_ROPE_LLAMA3, LC_ERR_INVALID, "%s: kind=%d", call, kind);
    LC_CHECK(rot_dim >= 0 && rot_dim % 2 == 0, LC_ERR_INVALID, "%s: rot_dim=%d must be even", call, rot_dim);
    LC_CHECK(theta >= 1.0 && std::isfinite(theta), LC_ERR_INVALID, "%s: theta=%g (1 or more)", call, theta);
    LC_CHECK(kind == LC_ROPE_PLAIN || (factor >= 1.0 && std::isfinite(factor)), LC_ERR_INVALID, "%s: factor=%g (1 or more)", call, factor);
    const bool mixed = kind == LC_ROPE_YARN || kind == LC_ROPE_LLAMA3;
    if (mixed) {
        if (fast == 0.0) fast = kind == LC_ROPE_YARN ? 32.0 : 4.0;
        if (slow == 0.0) slow = 1.0;
        LC_CHECK(original > 0, LC_ERR_INVALID, "%s: original=%d", call, original);
        LC_CHECK(std::isfinite(fast) && slow > 0.0 && fast > slow, LC_ERR_INVALID, "%s: fast=%g, slow=%g (fast above slow, both positive)", call, fast, slow);
        LC_CHECK(kind != LC_ROPE_YARN || theta > 1.0, LC_ERR_INVALID, "%s: theta=%g (above 1)", call, theta);
    }
    LC_CHECK(kind != LC_ROPE_NTK || rot_dim != 2, LC_ERR_INVALID, "%s: rot_dim=2 has one frequency, which a raised base leaves as it is", call);
    *magnitude = kind == LC_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    const long double turn = 6.283185307179586476925286766559L;
    const long double base = kind == LC_ROPE_NTK && rot_dim > 0 ? (long double)theta * powl((long double)factor, (long double)rot_dim / (rot_dim - 2)) : (long double)theta;
    // the pair that turns so often within the original length
    auto pair_of = [&](double turns) { return rot_dim * std::log(original / (turns * (double)turn)) / (2.0 * std::log(theta)); };
    const double low = kind == LC_ROPE_YARN ? std::max(std::floor(pair_of(fast)), 0.0) : 0.0, high = kind == LC_ROPE_YARN ? std::min(std::ceil(pair_of(slow)), rot_dim - 1.0) : 0.0;
    for (int32_t d = 0; d < rot_dim / 2; d++) {
        long double f = powl(base, -2.0L * d / rot_dim) / turn;  // of a turn
        if (kind == LC_ROPE_LINEAR) f /= factor;
        if (mixed) {
            long double keep = kind == LC_ROPE_YARN ? 1.0L - (d - (long double)low) / std::max(high - low, 0.001) : ((long double)original * f - slow) / ((long double)fast - slow);
            keep = std::min(1.0L, std::max(0.0L, keep));
            f = f * keep + f / factor * (1.0L - keep);
        }
        const long double whole = f * 0x1p64L;
        out[d] = (uint64_t)whole + (whole - (long double)(uint64_t)whole >= 0.5L ? 1u : 0u);
    }
    return LC_OK;
}

int32_t lc_rope_dev(uint32_t typ, int32_t n_rows, const int64_t* positions_dev, const uint64_t* turns_dev, int32_t rot_dim, int32_t head_dim, int32_t layout, int32_t inverse, double magnitude,
                    const void* x_dev, int64_t x_stride, void* x_out_dev, int64_t x_out_stride, int32_t x_heads, const void* y_dev, int64_t y_stride, void* y_out_dev, int64_t y_out_stride,
                    int32_t y_heads, void* stream_) {
    const char* call = "lc_rope_dev";
    LC_CHECK(typ == LC_TYPE_F32 || typ == LC_TYPE_F16 || typ == LC_TYPE_BF16, LC_ERR_UNSUPPORTED, "%s: type %u (f32, f16 and bf16 are taken)", call, typ);
    LC_CHECK(n_rows >= 0 && n_rows <= 1 << 24, LC_ERR_INVALID, "%s: n_rows=%d (0 .. 2^24)", call, n_rows);
    LC_CHECK(head_dim >= 1 && head_dim <= 1024, LC_ERR_INVALID, "%s: head_dim=%d (1 .. 1024)", call, head_dim);
    LC_CHECK(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, LC_ERR_INVALID, "%s: rot_dim=%d (even, head_dim %d at most)", call, rot_dim, head_dim);
    LC_CHECK(layout == LC_ROPE_HALF || layout == LC_ROPE_INTERLEAVED, LC_ERR_INVALID, "%s: layout=%d", call, layout);
    LC_CHECK(std::isfinite(magnitude) && std::fabs(magnitude) <= 1e30, LC_ERR_INVALID, "%s: magnitude=%g", call, magnitude);
    LC_CHECK(x_heads >= 1 && x_heads <= 65536 && (!y_dev || (y_heads >= 1 && y_heads <= 65536)), LC_ERR_INVALID, "%s: %d and %d heads (1 .. 65536)", call, x_heads, y_heads);
    if (n_rows == 0) return LC_OK;
    LC_CHECK(positions_dev && x_dev && x_out_dev && (!y_dev || y_out_dev) && (rot_dim == 0 || turns_dev), LC_ERR_INVALID, "%s: null pointer", call);
    const int64_t xr = (int64_t)x_heads * head_dim, yr = (int64_t)y_heads * head_dim;
    LC_CHECK(x_stride >= xr && x_out_stride >= xr && (!y_dev || (y_stride >= yr && y_out_stride >= yr)), LC_ERR_INVALID, "%s: rows overlap", call);
    LC_CHECK((x_dev != x_out_dev || x_stride == x_out_stride || n_rows == 1) && (!y_dev || y_dev != y_out_dev || y_stride == y_out_stride || n_rows == 1), LC_ERR_INVALID,
             "%s: in place with another stride", call);
    DeviceScope dev;
    LC_TRY(dev.enter(x_dev, call));
    RopeArgs a{{x_dev, x_out_dev, x_stride, x_out_stride, x_heads}, {y_dev, y_out_dev, y_stride, y_out_stride, y_dev ? y_heads : 0}, positions_dev, turns_dev, n_rows, 1, rot_dim / 2, head_dim,
               layout == LC_ROPE_INTERLEAVED, inverse != 0, magnitude};
    cudaStream_t s = stream_or_own(stream_);
    if (typ == LC_TYPE_F32) return rope_as<float>(a, s);
    if (typ == LC_TYPE_F16) return rope_as<__half>(a, s);
    return rope_as<__nv_bfloat16>(a, s);
}

}  // extern "C"
