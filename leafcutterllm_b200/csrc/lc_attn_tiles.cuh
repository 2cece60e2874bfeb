// What attention in tiles on tcgen05 shares between the 8-bit and the 4-bit cache: tensor-memory accesses, products that one lane of a warp issues, the swizzled
// places of an operand, and the kernel that joins units whose keys are cut.
#pragma once
#include "lc_kv8_attn.cuh"
#include "lc_umma.cuh"

namespace lc {

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    tmem_ld16(taddr, r);
    tmem_ld16(taddr + 16, r + 16);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// products issued by the lane whose `by` is set, in a warp that goes through this together
__device__ __forceinline__ void mma_ss_by(uint32_t by, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(da), "l"(db),
                 "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
__device__ __forceinline__ void mma_ts_by(uint32_t by, uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(db),
                 "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
// The same with descriptors as their lower words, for an issuing lane that elect_lane has chosen.  Both let the compiler keep the operands in the warp's registers: a product then takes 50 cycles
// to issue, less than it runs, instead of 105 to 155 (64-bit descriptors, lane 0 by its number), which made the issue the bottleneck of attention in tiles.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(r));
    return r;
}
// of umma_desc_sw128, whose upper word is 0x40004040
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr) { return ((saddr >> 4) & 0x3fffu) | 0x10000u; }
__device__ __forceinline__ void mma_ss_low(uint32_t by, uint32_t d, uint32_t da, uint32_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 x, y;\n mov.b64 x, {%1, 0x40004040};\n mov.b64 y, {%2, 0x40004040};\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d), "r"(da), "r"(db), "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
__device__ __forceinline__ void mma_ts_low(uint32_t by, uint32_t d, uint32_t a, uint32_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 y;\n mov.b64 y, {%2, 0x40004040};\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(db), "r"(idesc), "r"(accumulate), "r"(by)
                 : "memory");
}
// 16-byte chunk `ch` (of 8) of a row of 128 bytes
__device__ __forceinline__ int sw128(int row, int ch) { return row * 128 + ((ch ^ (row & 7)) << 4); }

// Joins the parts of units whose keys are cut: a warp per row.
template <int HD>
__global__ void __launch_bounds__(256) kv_tiles_join_kernel(Kv8Pool pool, Kv8Seqs seqs, AttnArgs a, int splits) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint2 sums[8];
    uint32_t* units = reinterpret_cast<uint32_t*>(smem);
    uint32_t* cum = units + seqs.n_seqs + 1;
    line_up<kTileRows2>(seqs, pool, a, cum, units, sums);
    pdl_wait();
    if (blockIdx.x >= units[seqs.n_seqs]) return;
    const int seq = seq_at(units, seqs.n_seqs, blockIdx.x), in = blockIdx.x - units[seq];
    const SeqWork w = seq_work<kTileRows2>(seqs, pool, a, seq);
    const int kvh = in % pool.n_kv, row_lo = (w.blocks - 1 - in / pool.n_kv) * kTileRows2, row_n = min(kTileRows2, w.n * a.group - row_lo);
    const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= row_n) return;
    constexpr int PER = HD / 32;
    float mx = kNegInf, sum = 0.0f, v[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) v[e] = 0.0f;
    for (int s = 0; s < splits; s++) {
        const float* p = a.part + (size_t)(blockIdx.x * splits + s) * (kTileRows2 * (HD + 2));
        const float pm = p[r], ps = p[kTileRows2 + r];
        if (pm == kNegInf && ps == 0.0f) continue;      // no keys: its sums are not there
        const float m2 = fmaxf(mx, pm), ref = m2 == kNegInf ? 0.0f : m2;
        const float f0 = exp2_fast(mx - ref), f1 = exp2_fast(pm - ref);
        sum = f0 * sum + (isnan(ps) ? ps : f1 * ps);
#pragma unroll
        for (int e = 0; e < PER; e++) v[e] = fmaf(f0, v[e], f1 * p[2 * kTileRows2 + (size_t)r * HD + lane * PER + e]);
        mx = m2;
    }
    const int tok = (row_lo + r) / a.group;
    const int64_t dst = (int64_t)(w.first + tok) * a.out_stride + ((int64_t)kvh * a.group + (row_lo + r - tok * a.group)) * pool.hd;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (a.lse && lane == 0) a.lse[(int64_t)(w.first + tok) * a.lse_stride + kvh * a.group + row_lo + r - tok * a.group] = (mx + (log2f(sum) - a.lse_less)) * 0.693147180559945f;
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (lane * PER + e < pool.hd) store1(a.out, dst + lane * PER + e, a.typ, v[e] * inv);
}

}  // namespace lc
