// paged_attn_launch.cuh - the attention kernels' instantiations and launches for one cache type (included by the
// paged_attn_*.cu files, one per type, which compile side by side).
#pragma once

#include "device.hpp"
#include "paged_attn.cuh"
#include "paged_attn_plan.hpp"

namespace gcu {

template <typename S>
int launch_paged_shape(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    const int grid = p.grid;
    if (!shared_opt_in<k_paged_attn<S>>(S::kSmem)) return GCUDA_E_CUDA;
    if (launch_ex(k_paged_attn<S>, dim3(grid), dim3(kPagedAttnThreads), S::kSmem, st, true, a) != cudaSuccess) return GCUDA_E_CUDA;
    if (grid == 1) return GCUDA_OK;   // (nothing is cut)
    const int units = S::NTT * S::OM / 2, per = kJoinThreads / 32 / p.split;
    return launch_ex(k_paged_attn_join<S>, dim3(p.cuts, (units + per - 1) / per), dim3(kJoinThreads), 0, st, true, a, p.split, grid) ==
                   cudaSuccess
               ? GCUDA_OK
               : GCUDA_E_CUDA;
}

template <int CACHE, int HD, bool SPLIT>
int launch_paged_rows(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    if (p.rows == 8) return launch_paged_shape<PagedShape<HD, CACHE, SPLIT, 1, 1>>(a, p, st);
    if (p.rows == 16) return launch_paged_shape<PagedShape<HD, CACHE, SPLIT, 2, 1>>(a, p, st);
    return launch_paged_shape<PagedShape<HD, CACHE, SPLIT, 2, 4>>(a, p, st);
}
template <int CACHE, int HD>
int launch_paged_split(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    const bool split = a.x.type == GCUDA_F32 || (a.x.type == GCUDA_F16 && CACHE == GCUDA_BF16);
    return split ? launch_paged_rows<CACHE, HD, true>(a, p, st) : launch_paged_rows<CACHE, HD, false>(a, p, st);
}
template <int CACHE>
int launch_paged_cache(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    if (a.kv.head_dim == 64) return launch_paged_split<CACHE, 64>(a, p, st);
    if (a.kv.head_dim == 128) return launch_paged_split<CACHE, 128>(a, p, st);
    return launch_paged_split<CACHE, 256>(a, p, st);
}

}  // namespace gcu
