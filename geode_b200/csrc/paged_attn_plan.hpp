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
// its positions; more are worked on by all four warps together, in blocks of 16, or above 16 rows of 40: a block reads the cache
// and widens it once for all its rows. Measured: 64 conversations of one row and 8 query heads over int8 62 us in blocks of 8, 100
// in blocks of 16; 32 of 2 such rows 60 us in blocks of 16, 102 in one of 40; batches of alike sequences (32 x 6000 positions, 2
// key heads over int8, dims 64 / 128 / 256) of 24 rows 82 / 106 / 135 us in one block of 40 and 107 / 109 / 131 in two of 16, of 40
// rows 84 / 107 / 139 and 153 / 152 / 190; bf16 rows of 128 77 and 119. Blocks of 16 are the faster ones where sequences bring
// fewer rows than max_rows (1 to 5 of 8 heads: 84 us against 106), which the host does not know, and for 17 to 32 rows where two
// CTAs of 40 do not fit an SM (24 rows over bf16 rows of 256: 132 us against 153; 40 rows: 169 and 169).
inline PagedAttnPlan plan_paged_attn(const gcuda_paged_kv &kv, const gcuda_paged_batch &b, int n_heads) {
    PagedAttnPlan p{};
    const int64_t R = static_cast<int64_t>(b.max_rows) * (n_heads / kv.n_kv_heads);
    p.rows = R <= 8 ? 8 : R <= 16 ? 16 : 40;
    // two CTAs an SM, which are resident together but for 16-bit rows of 256 with more than 16 query rows or with 9 to 16 and
    // float queries (f16 ones over bf16), and float over bf16 rows of 128 with more than 16: their shared memory leaves room for one,
    // and the grid runs in two turns. No more than there can be work: a tile of 16 positions and an item's cost of up to 32 each
    const int64_t per_seq = std::max<int64_t>(1, (static_cast<int64_t>(b.max_pages) * kv.page_size + 15) / 16);
    const int64_t blocks = (R + p.rows - 1) / p.rows;
    const int64_t most = 2 * static_cast<int64_t>(sm_count());
    int64_t items = 1;
    for (const int64_t f : {static_cast<int64_t>(b.n_seq), static_cast<int64_t>(kv.n_kv_heads), blocks})
        items = std::min(most, items * std::min(most, f));   // (capped at each step: no overflow)
    p.grid = static_cast<int>(std::min(most, items * std::min(most, per_seq + 32)));
    // Few items have many parts each: measured with 1, 4 and 16 warps to an item's parts, 2 items 24, 18.5 and 15.7 us (1 x 8192
    // positions), 4 items 86, 77 and 73 (2 x 131072), 20 items 53.5, 52 and 63, 128 items 62, 68 and 83
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
