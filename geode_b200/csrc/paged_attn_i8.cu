// paged_attn_i8.cu - gcuda_op_paged_attn's kernels over a int8 cache.
#include "paged_attn_launch.cuh"

int gcu::launch_paged_attn_i8(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    return launch_paged_cache<GCUDA_I8>(a, p, st);
}
