// paged_attn_plan.hpp - the host's side of gcuda_op_paged_attn: which kernel shape takes the call, its grid and scratch.
#pragma once

#include <algorithm>

#include "device.hpp"

namespace gcu {

struct PagedAttnArgs;
struct PagedAttnPlan {
    int rows;      // query rows of a block: 8 (k_paged_attn), 16 or 40 (k_paged_attn_rows)
    int grid;      // main CTAs
    int split;     // warps that share an item's parts in the join
    int cuts;      // the join's CTAs: one for each item that may be cut, or (many items, split 1) for each main CTA
    size_t cut, stats, part, total;   // scratch offsets
};

// Query rows sharing a key head, R = max_rows * n_heads / n_kv_heads, choose the shape: up to 8 leave each warp alone with
// its positions; more are worked on by all four warps together, in blocks of 16 or 40.
inline PagedAttnPlan plan_paged_attn(const gcuda_paged_kv &kv, const gcuda_paged_batch &b, int n_heads) {
    PagedAttnPlan p{};
    const int64_t R = static_cast<int64_t>(b.max_rows) * (n_heads / kv.n_kv_heads);
    p.rows = R <= 8 ? 8 : R <= 16 ? 16 : 40;
    // two resident CTAs an SM; no more than there can be work: a tile of 16 positions and an item's cost of up to 32 each
    const int64_t per_seq = std::max<int64_t>(1, (static_cast<int64_t>(b.max_pages) * kv.page_size + 15) / 16);
    const int64_t blocks = (R + p.rows - 1) / p.rows;
    const int64_t most = 2 * static_cast<int64_t>(sm_count());
    int64_t items = 1;
    for (const int64_t f : {static_cast<int64_t>(b.n_seq), static_cast<int64_t>(kv.n_kv_heads), blocks})
        items = std::min(most, items * std::min(most, f));   // (capped at each step: no overflow)
    p.grid = static_cast<int>(std::min(most, items * std::min(most, per_seq + 32)));
    // (few items: many parts each)
    p.split = items >= 64 ? 1 : items >= 16 ? 4 : 16;
    p.cuts = std::max(1, static_cast<int>(p.split == 1 ? p.grid - 1 : std::min<int64_t>(items, p.grid - 1)));
    auto take = [&](size_t bytes) {
        const size_t at = p.total;
        p.total += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t slots = 2 * static_cast<size_t>(p.grid);
    p.cut = take(static_cast<size_t>(p.grid) * 16);
    p.stats = take(slots * p.rows * 16);
    p.part = take(slots * p.rows * kv.head_dim * 4);
    return p;
}

// one per cache type, each in a translation unit of its own
int launch_paged_attn_i8(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st);
int launch_paged_attn_bf16(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st);
int launch_paged_attn_f16(const PagedAttnArgs &a, const PagedAttnPlan &p, cudaStream_t st);

}  // namespace gcu
