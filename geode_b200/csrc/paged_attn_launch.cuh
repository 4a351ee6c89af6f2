// paged_attn_launch.cuh - the attention kernels' instantiations and launches for one cache type (included by the
// paged_attn_*.cu files, one per type, which compile side by side).
#pragma once

#include "device.hpp"
#include "paged_attn.cuh"
#include "paged_attn_plan.hpp"
#include "paged_attn_rows.cuh"

namespace gcu {

template <typename S, auto kern>
int launch_paged_shape(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    if (!shared_opt_in<kern>(S::kSmem)) return GCUDA_E_CUDA;
    if (launch_ex(kern, dim3(p.grid), dim3(kPagedAttnThreads), S::kSmem, st, true, a) != cudaSuccess) return GCUDA_E_CUDA;
    if (p.grid == 1) return GCUDA_OK;   // (nothing is cut)
    const int units = S::NT * S::OM / 2, threads = p.split == 1 ? kJoinThreads / 2 : kJoinThreads, per = threads / 32 / p.split;
    return launch_ex(k_paged_attn_join<S>, dim3(p.cuts, (units + per - 1) / per), dim3(threads), 0, st, true, a, p.split, p.grid) ==
                   cudaSuccess
               ? GCUDA_OK
               : GCUDA_E_CUDA;
}

template <int CACHE, int HD, bool SPLIT>
int launch_paged_rows(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    using S8 = PagedShape<HD, CACHE, SPLIT>;
    using S16 = PagedRowsShape<HD, CACHE, SPLIT, 2>;
    using S40 = PagedRowsShape<HD, CACHE, SPLIT, 5>;
    if (p.rows == S8::kRows) return launch_paged_shape<S8, k_paged_attn<S8>>(a, p, st);
    if (p.rows == S16::kRows) return launch_paged_shape<S16, k_paged_attn_rows<S16>>(a, p, st);
    return launch_paged_shape<S40, k_paged_attn_rows<S40>>(a, p, st);
}
template <int CACHE, int HD>
int launch_paged_split(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    if constexpr (CACHE == GCUDA_I8) {
        return launch_paged_rows<CACHE, HD, false>(a, p, st);   // (the queries' digits are the same for all activations)
    } else {
        const bool split = a.x.type == GCUDA_F32 || (a.x.type == GCUDA_F16 && CACHE == GCUDA_BF16);
        return split ? launch_paged_rows<CACHE, HD, true>(a, p, st) : launch_paged_rows<CACHE, HD, false>(a, p, st);
    }
}
template <int CACHE>
int launch_paged_cache(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st) {
    if (a.kv.head_dim == 64) return launch_paged_split<CACHE, 64>(a, p, st);
    if (a.kv.head_dim == 128) return launch_paged_split<CACHE, 128>(a, p, st);
    return launch_paged_split<CACHE, 256>(a, p, st);
}

}  // namespace gcu
