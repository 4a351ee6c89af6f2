// paged_attn_bf16.cu - gcuda_op_paged_attn's kernels over a bf16 cache.
#include "paged_attn_launch.cuh"

int gcu::launch_paged_attn_bf16(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    return launch_paged_cache<GCUDA_BF16>(a, p, st);
}
