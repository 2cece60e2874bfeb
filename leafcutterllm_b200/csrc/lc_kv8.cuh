// What the kernels over the 8-bit key/value cache share: views of the cache and of a call's rows, the sequence of a row, activations of
// three types, and on the host the checks of arguments and the device that a call runs on.
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include "lc_common.cuh"

namespace lc {

constexpr int kKv8MaxSeqs = 4096;

struct Kv8Pool {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int n_pages, n_kv, page_shift, hd;  // page_tokens = 1 << page_shift
};
struct Kv8Seqs {
    const int32_t* table;
    const int32_t* ctx;
    const int32_t* row_start;
    int32_t* status;
    int n_seqs, width, n_rows;
};

// Device of the call's pointers, current while this lives.
struct DeviceScope {
    int before = -1;
    int32_t enter(const void* dev_ptr, const char* what);
    ~DeviceScope() {
        if (before >= 0) (void)cudaSetDevice(before);
    }
};
inline cudaStream_t stream_or_own(void* s) { return s ? (cudaStream_t)s : stream(); }
// kv8.cu: the arguments that all calls over the cache have; `view` and `seqs` are filled
int32_t kv8_check(const char* call, const lc_kv8_cache* cache, const lc_kv8_rows* rows, uint32_t typ, int32_t n_rows, Kv8Pool* view, Kv8Seqs* seqs);
// nothing but a cache line's worth of alignment is asked of activations: 16-byte accesses where pointer and stride (in bytes) allow them
inline bool rows_aligned(const void* p, int64_t stride_elems, size_t elem, size_t to) {
    return ((uintptr_t)p % to) == 0 && ((size_t)stride_elems * elem) % to == 0;
}

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float elem_f(T v);
template <> __device__ __forceinline__ float elem_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float elem_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float elem_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T to_elem(float v);
template <> __device__ __forceinline__ float to_elem<float>(float v) { return v; }
template <> __device__ __forceinline__ __half to_elem<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 to_elem<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// the larger one, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// two f32 at a time
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// four numbers' low bytes
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); }

// Rows [first, first + n) of sequence i; false where row_start is not ascending within the call's rows.
__device__ __forceinline__ bool kv8_span(const Kv8Seqs& s, int i, int& first, int& n) {
    const int a = s.row_start[i], b = s.row_start[i + 1];
    first = a;
    n = b - a;
    return a >= 0 && b >= a && b <= s.n_rows;
}
// Whether positions ctx .. ctx + n - 1 lie in the table.
__device__ __forceinline__ bool kv8_in_table(const Kv8Seqs& s, const Kv8Pool& p, int ctx, int n) {
    return ctx >= 0 && (long long)ctx + n <= ((long long)s.width << p.page_shift);
}
__device__ __forceinline__ void kv8_raise(const Kv8Seqs& s, int i) {
    if (s.status) atomicMax(s.status, i + 1);
}
// By one whole block: raises the status for sequences that the arrays themselves rule out.
__device__ __forceinline__ void kv8_check_seqs(const Kv8Seqs& s, const Kv8Pool& p) {
    if (!s.status) return;
    for (int i = threadIdx.x; i < s.n_seqs; i += blockDim.x) {
        int first, n;
        if (!kv8_span(s, i, first, n) || (n > 0 && !kv8_in_table(s, p, s.ctx[i], n))) kv8_raise(s, i);
    }
}
// By one whole warp: the first of all sequences that has row `r` (-1: none), and where there is none the next row that one of them begins with.  For rows that the
// search below does not find: in front of, between and behind the sequences, or where row_start goes back and forth.
[[maybe_unused]] static __device__ __noinline__ int2 kv8_seq_among(const int32_t* row_start, int n_seqs, int n_rows, int r) {
    const int lane = threadIdx.x & 31;
    int next = 0x7fffffff;
    for (int i0 = 0; i0 < n_seqs; i0 += 32) {
        const int i = i0 + lane, a = i < n_seqs ? row_start[i] : 0, b = i < n_seqs ? row_start[i + 1] : 0;
        const bool rows = a >= 0 && b > a && b <= n_rows;
        const unsigned has = __ballot_sync(0xffffffffu, rows && r >= a && r < b);
        if (has) return make_int2(i0 + __ffs(has) - 1, r);
        if (rows && a > r) next = min(next, a);
    }
    return make_int2(-1, __reduce_min_sync(0xffffffffu, next));
}
// By one whole warp: the sequence whose rows row `r` is one of (-1: none; `next` is then the next row that has one), 32 probes a step.
__device__ __forceinline__ int kv8_seq_of_row(const Kv8Seqs& s, int r, int& next) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = s.n_seqs + 1;
    for (;;) {
        const int step = (len + 31) >> 5, at = lane * step;
        const bool le = at < len && s.row_start[lo + at] <= r;
        const int cnt = __popc(__ballot_sync(0xffffffffu, le));
        if (cnt == 0) { lo = s.n_seqs; break; }
        lo += (cnt - 1) * step;
        len = min(step, len - (cnt - 1) * step);
        if (step == 1) break;
    }
    int first, n;
    if (lo < s.n_seqs && kv8_span(s, lo, first, n) && r - first < n && r >= first) return lo;
    const int2 found = kv8_seq_among(s.row_start, s.n_seqs, s.n_rows, r);
    next = found.y;
    return found.x;
}
#endif

}  // namespace lc
