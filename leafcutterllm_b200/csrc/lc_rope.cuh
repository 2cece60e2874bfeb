// Rotations by position: angles from tables of turns, tables of sines and cosines in shared memory, pairs turned in f32 and 64 bits.
#pragma once
#include "lc_kv8.cuh"

namespace lc {

#ifdef __CUDACC__
// Quotients by a number d that a kernel learns when it runs, for dividends below 2^32 / d (heads times pieces of 8 or 16 dims of a head: below 2^30).
struct Divider {
    uint32_t d, m;
    __device__ __forceinline__ explicit Divider(int by) : d((uint32_t)max(by, 1)), m(0xffffffffu / d + 1) {}
    __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, m); }
};
// Brings bytes that will be read soon into L2: a multiple of 16, 16-byte aligned.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
    if (bytes) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes));
}
// (cosine, sine) of `positions` times an entry of turns: the product wraps around by itself, and what is left is the angle's fraction of a turn to 2^-64 of one,
// however far the position is (cos and sin of an f32 angle lose 2^-24 of the ANGLE: 0.06 at 10^6).
__device__ __forceinline__ double2 turn_of(uint64_t per_position, int64_t positions) {
    const int64_t frac = (int64_t)((uint64_t)positions * per_position);
    double2 r;
    sincospi((double)frac * 0x1p-63, &r.y, &r.x);  // frac 2^-64 turns = frac 2^-63 pi
    return r;
}
// u c - w s in f32 with the cosine and sine as two f32 each: the difference of the products with what the second lost (Kahan), 1.5 2^-24 of the result off,
// and what the high parts leave out
__device__ __forceinline__ float turned(float u, float w, float ch, float cl, float sh, float sl) {
    const float p = w * sh, lost = fmaf(-w, sh, p), d = fmaf(u, ch, -p);
    const float y = d + (lost + fmaf(u, cl, -w * sl));
    return fabsf(d) < INFINITY ? y : d;
}
__device__ __forceinline__ void set_turn(float4& at, double2 t) {
    at.x = (float)t.x; at.y = (float)(t.x - at.x);
    at.z = (float)t.y; at.w = (float)(t.y - at.z);
}
// Where pair p of a row of a table lies: lanes that have eight pairs in a row each then read neighbouring places.  A row has 8 * n8 places, n8 = ceil(pairs / 8).
__device__ __forceinline__ int turn_place(int p, int n8) { return (p & 7) * n8 + (p >> 3); }
// What a table holds for a pair: for f32 outputs sine and cosine as two f32 each, for 16-bit ones as one.
template <typename T> struct TurnEntry { using type = float2; };
template <> struct TurnEntry<float> { using type = float4; };
__device__ __forceinline__ void put_turn(float2& at, double2 t) { at = make_float2((float)t.x, (float)t.y); }
__device__ __forceinline__ void put_turn(float4& at, double2 t) { set_turn(at, t); }
// f32: 1.5 2^-24 of the result; 16-bit types: 2^-23 of the pair's length, far below their rounding
__device__ __forceinline__ void turn_pair(float u, float w, const float4& t, float& a, float& b) {
    a = turned(u, w, t.x, t.y, t.z, t.w);
    b = turned(u, -w, t.z, t.w, t.x, t.y);
}
__device__ __forceinline__ void turn_pair(float u, float w, const float2& t, float& a, float& b) {
    a = u * t.x - w * t.y;
    b = u * t.y + w * t.x;
}
// A row of a table that is kept as cosines and sines in f32 and, apart, what f32 lost of them.
template <typename T> struct TurnRow {
    const float2* high;
    const float2* low;
    __device__ __forceinline__ typename TurnEntry<T>::type operator[](int at) const {
        if constexpr (sizeof(T) == 2) return high[at];
        else return make_float4(high[at].x, low[at].x, high[at].y, low[at].y);
    }
};
template <typename T> __device__ __forceinline__ void load8(const T* p, T (&v)[8]) {
#pragma unroll
    for (int u = 0; u < (int)sizeof(T) / 2; u++) reinterpret_cast<uint4*>(v)[u] = reinterpret_cast<const uint4*>(p)[u];
}
template <typename T> __device__ __forceinline__ void store8(T* p, const T (&v)[8]) {
#pragma unroll
    for (int u = 0; u < (int)sizeof(T) / 2; u++) reinterpret_cast<uint4*>(p)[u] = reinterpret_cast<const uint4*>(v)[u];
}

// What a thread turns at a time: eight pairs (8 i ..) of kTurnHeads neighbouring heads, of which n are there; their loads go out together and share what the table says.  half and the heads' dims multiples
// of 8, 16-byte accesses.
template <typename T> constexpr int kTurnHeads = sizeof(T) == 2 ? 4 : 2;
template <typename T, typename Row>
__device__ __forceinline__ void turn_item(const T* in, T* out, int hd, int n, int i, int half, bool interleaved, const Row& row, int n8) {
    constexpr int B = kTurnHeads<T>;
    const int d0 = interleaved ? 16 * i : 8 * i, d1 = interleaved ? d0 + 8 : half + d0;
    __align__(16) T u[B][8], w[B][8];
#pragma unroll
    for (int b = 0; b < B; b++) {
        const T* from = in + min(b, n - 1) * hd;
        load8(from + d0, u[b]);
        load8(from + d1, w[b]);
    }
    typename TurnEntry<T>::type t[8];
#pragma unroll
    for (int k = 0; k < 8; k++) t[k] = row[k * n8 + i];
#pragma unroll
    for (int b = 0; b < B; b++) {
        if (b >= n) break;
        if (interleaved) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                T(&v)[8] = k < 4 ? u[b] : w[b];
                const int k2 = 2 * (k & 3);
                float y0, y1;
                turn_pair(elem_f(v[k2]), elem_f(v[k2 + 1]), t[k], y0, y1);
                v[k2] = to_elem<T>(y0);
                v[k2 + 1] = to_elem<T>(y1);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                float y0, y1;
                turn_pair(elem_f(u[b][k]), elem_f(w[b][k]), t[k], y0, y1);
                u[b][k] = to_elem<T>(y0);
                w[b][k] = to_elem<T>(y1);
            }
        }
        store8(out + b * hd + d0, u[b]);
        store8(out + b * hd + d1, w[b]);
    }
}
// Eight dims behind the turned ones (8 i ..), copied.
template <typename T> __device__ __forceinline__ void copy_item(const T* in, T* out, int i, int half) {
    __align__(16) T u[8];
    load8(in + 2 * half + 8 * i, u);
    store8(out + 2 * half + 8 * i, u);
}
// The same for any sizes and alignment: a pair, or one dim behind them (hd - half items).
template <typename T, typename Row>
__device__ __forceinline__ void turn_item_plain(const T* in, T* out, int p, int half, bool interleaved, const Row& row, int n8) {
    if (p >= half) {
        out[half + p] = in[half + p];
        return;
    }
    const int d0 = interleaved ? 2 * p : p, d1 = interleaved ? d0 + 1 : p + half;
    float y0, y1;
    turn_pair(elem_f(in[d0]), elem_f(in[d1]), row[turn_place(p, n8)], y0, y1);
    out[d0] = to_elem<T>(y0);
    out[d1] = to_elem<T>(y1);
}
#endif

}  // namespace lc
