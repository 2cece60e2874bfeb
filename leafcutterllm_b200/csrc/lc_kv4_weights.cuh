// Arguments of the kernels that add up the weights of the 4-bit cache's keys.
#pragma once
#include "lc_kv4.cuh"

namespace lc {

struct WeightArgs {
    const void* q;
    const float* lse;
    float* mass;
    int64_t q_stride, lse_stride, mass_stride, mass_head_stride;
    int typ, group, window, capacity;
    bool q_vec;
    float scale_log2;
};
// kv4_weights_tiles.cu: many rows per sequence, heads of up to 128
int32_t launch_kv4_weights_tiles(const Kv4Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a, cudaStream_t s);

#ifdef __CUDACC__
// By one whole block: raises the status for sequences that the arrays themselves rule out, or whose sums have no room.
__device__ __forceinline__ void weights_check_seqs(const Kv8Pool& pool, const Kv8Seqs& seqs, const WeightArgs& a) {
    kv8_check_seqs(seqs, pool);
    for (int i = threadIdx.x; i < seqs.n_seqs; i += blockDim.x) {
        int first, n;
        if (kv8_span(seqs, i, first, n) && n > 0 && (long long)seqs.ctx[i] + n > a.capacity) kv8_raise(seqs, i);
    }
}
#endif

}  // namespace lc
