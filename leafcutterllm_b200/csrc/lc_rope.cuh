// Rotations by position: angles from tables of turns, tables of sines and cosines in shared memory, pairs turned in f32 and 64 bits.
#pragma once
#include "lc_kv8.cuh"

namespace lc {

#ifdef __CUDACC__
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
template <typename T> __device__ __forceinline__ void load8(const T* p, T (&v)[8]) {
#pragma unroll
    for (int u = 0; u < (int)sizeof(T) / 2; u++) reinterpret_cast<uint4*>(v)[u] = reinterpret_cast<const uint4*>(p)[u];
}
template <typename T> __device__ __forceinline__ void store8(T* p, const T (&v)[8]) {
#pragma unroll
    for (int u = 0; u < (int)sizeof(T) / 2; u++) reinterpret_cast<uint4*>(p)[u] = reinterpret_cast<const uint4*>(v)[u];
}

// What a thread turns at a time: eight pairs, or copies: eight dims behind them.  hd and half multiples of 8, 16-byte accesses.  A head has turn_items of them, the copies last.
__device__ __forceinline__ int turn_items(int hd, int half) { return (half >> 3) + ((hd - 2 * half) >> 3); }
template <typename T, typename Entry>
__device__ __forceinline__ void turn_item(const T* in, T* out, int i, int half, bool interleaved, const Entry* row, int n8) {
    const int pairs = half >> 3;
    __align__(16) T u[8], w[8];
    if (i >= pairs) {
        const int d = 2 * half + 8 * (i - pairs);
        load8(in + d, u);
        store8(out + d, u);
        return;
    }
    const int d0 = interleaved ? 16 * i : 8 * i, d1 = interleaved ? d0 + 8 : half + d0;
    load8(in + d0, u);
    load8(in + d1, w);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const Entry at = row[k * n8 + i];
        const int k2 = 2 * (k & 3);
        const T p = interleaved ? (k < 4 ? u[k2] : w[k2]) : u[k], q = interleaved ? (k < 4 ? u[k2 + 1] : w[k2 + 1]) : w[k];
        float y0, y1;
        turn_pair(elem_f(p), elem_f(q), at, y0, y1);
        if (interleaved) {
            (k < 4 ? u : w)[k2] = to_elem<T>(y0);
            (k < 4 ? u : w)[k2 + 1] = to_elem<T>(y1);
        } else {
            u[k] = to_elem<T>(y0);
            w[k] = to_elem<T>(y1);
        }
    }
    store8(out + d0, u);
    store8(out + d1, w);
}
// The same for any sizes and alignment: a pair, or one dim behind them (hd - half items).
template <typename T, typename Entry>
__device__ __forceinline__ void turn_item_plain(const T* in, T* out, int p, int half, bool interleaved, const Entry* row, int n8) {
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
