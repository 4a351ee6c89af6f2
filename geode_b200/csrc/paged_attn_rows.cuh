// paged_attn_rows.cuh - attention over a paged cache for more than 8 query rows an item (verify batches: T tokens times the
// G query heads of a key head): k_paged_attn_rows.
//
// Here the products weigh as much as the copies, so no cache row is widened twice: of a tile's 64 positions each of the
// four warps multiplies its 16 with all rows' queries (S^T = K Q^T), the weights go through shared memory as ready
// fragments, and in the second product each warp has a quarter of the dims for all rows and all 64 positions. The running
// maxima are the CTA's: a tile on which none grows far (nearly all but the first) costs one vote, folded into the barrier.
//
// Measured: 32 ragged verify batches of 5 rows (40 rows an item), up to 8192 positions of int8, 2 heads of 256, float
// activations: 106 us (142 MB; 68 us for each further 142 MB). The tensor pipe is busy 36% of the time: a warp and tile has 280
// products (at the 8.2 cycles of mma.sync the pipe's floor is 35 us) among 1900 instructions in dependent phases, two warps a
// scheduler, which wait for fixed latencies (2 warps an issue) and instruction fetches (1).
#pragma once

#include "paged_attn.cuh"

namespace gcu {

template <int HD_, int CACHE_, bool SPLIT_, int NT_>
struct PagedRowsShape : PagedBase<HD_, CACHE_, SPLIT_, NT_> {
    using B = PagedBase<HD_, CACHE_, SPLIT_, NT_>;
    using B::HD, B::RB, B::I8, B::OM, B::ES, B::NT, B::SPLIT, B::kRows;
    static constexpr int TP = 16, CT = 4 * TP;                    // positions of a warp, of a CTA's tile
    static constexpr int kItemCost = 131072 / (2 * CT * RB) > 0 ? 131072 / (2 * CT * RB) : 1;
    static constexpr int kEntry = CT * RB;                        // a tile's K or V rows
    static constexpr int E = 65536 / kEntry < 3 ? 3 : 65536 / kEntry > 8 ? 8 : 65536 / kEntry;
    static constexpr int TS = E / 2 + 2, kSegs = E / 2 + 5;
    static constexpr int kScale = (I8 ? 2 * TP * 4 : 0) + 16;
    static constexpr int DL = HD / 32, MW = HD / 64;              // dims of a lane, m tiles of a warp in the second product
    static constexpr int kP = 4 * NT * 32 * 8 * B::PN;              // the weights [16 positions][n tile][lane]
    static constexpr int kPTwo = B::THREE ? 4 * NT * 32 * 16 : 0;                // (where their third numbers start)
    static constexpr int o_ring = 0, o_q = o_ring + E * kEntry, o_p = o_q + B::kQ, o_scale = o_p + kP;
    static constexpr int o_col = o_scale + 4 * TS * kScale;       // [kRows] column factor, then the last position seen
    static constexpr int o_seg = o_col + kRows * 8;
    static constexpr int o_max = o_seg + 4 * kSegs * 48;          // [warp][kRows] a tile's maxima; at the end the sums
    static constexpr int kSmem = o_max + 4 * kRows * 8;
    static __device__ __forceinline__ int dim(int m, int gid) { return m / MW * (HD / 4) + gid * DL + 2 * (m % MW); }
};

template <typename S>
__global__ void __launch_bounds__(kPagedAttnThreads, 2) k_paged_attn_rows(PagedAttnArgs a) {
    constexpr int NT = S::NT, RB = S::RB, E = S::E, OM = S::OM, MW = S::MW, TP = S::TP;
    constexpr bool I8 = S::I8, BF16 = S::BF16, SPLIT = S::SPLIT;
    constexpr int PN = S::PN;
    extern __shared__ __align__(1024) uint8_t sm[];   // (a row of the ring starts on a multiple of its size)
    __shared__ PagedWalkShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.x.n_heads / a.kv.n_kv_heads, cta = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) a.cut[cta] = make_int4(0, 0, 0, 0);
    PagedWalk<S> walk{a, sh, reinterpret_cast<PagedSegment *>(sm + S::o_seg) + warp * S::kSegs};
    if (!walk.start()) return;

    const uint2 *q_one = reinterpret_cast<const uint2 *>(sm + S::o_q + S::kQTwo);
    const uint4 *q_two = reinterpret_cast<const uint4 *>(sm + S::o_q);
    float *col_s = reinterpret_cast<float *>(sm + S::o_col);
    int *lim_s = reinterpret_cast<int *>(sm + S::o_col) + S::kRows;
    float2 *max_s = reinterpret_cast<float2 *>(sm + S::o_max);
    uint8_t *scales = sm + S::o_scale + warp * S::TS * S::kScale;
    const uint32_t ring_a = smem_addr(sm + S::o_ring), scales_a = smem_addr(scales);

    // ---- the copies: a warp's 16 rows of K, then of V
    PagedTile ahead0 = walk.look(), ahead1 = walk.look();
    int in_slot = 0, in_tile = S::TS - 1;
    bool in_any = true, one_page = false;
    int64_t place = 0;
    uint32_t ok = 0;
    auto issue = [&](auto kind_) {
        constexpr bool is_v = decltype(kind_)::value % 2;
        if (!is_v && in_any) {
            const PagedTile t = ahead0;
            ahead0 = ahead1;
            ahead1 = walk.look();
            in_any = t.p0 >= 0;
            if (in_any) {
                in_tile = in_tile + 1 == S::TS ? 0 : in_tile + 1;
                const bool there = t.page >= 0 && t.page < a.kv.n_pages;
                if (t.page != -2 && !there) atomicOr(a.status, kErrBadShape);
                place = there ? t.page * a.kv.page_stride + t.in_page * a.kv.pos_stride + t.kh * a.kv.head_stride : 0;
                ok = __ballot_sync(0xffffffffu, there);
                one_page = ok == 0xffffu && __shfl_sync(0xffffffffu, t.in_page, 0) + TP <= a.kv.page_size;
                if (lane == 0) *reinterpret_cast<uint32_t *>(scales + in_tile * S::kScale) = ok;
                if constexpr (I8) {
                    if (lane < TP) {
                        const uint32_t d = scales_a + in_tile * S::kScale + 16 + lane * 4;
                        const int64_t sp = there ? t.page * a.kv.scale_page_stride + t.in_page * a.kv.scale_pos_stride + t.kh * a.kv.scale_head_stride : 0;
                        copy4(d, a.kv.k_scale + sp, there ? 4 : 0);
                        copy4(d + TP * 4, a.kv.v_scale + sp, there ? 4 : 0);
                    }
                }
            }
        }
        if (in_any) {
            const uint8_t *src = static_cast<const uint8_t *>(is_v ? a.kv.v : a.kv.k);
            copy_rows<RB, is_v, TP * (RB / 16) / 32, S::ES>(ring_a + in_slot * S::kEntry + warp * TP * RB, src, a.kv.pos_stride, place, ok, one_page, 0);
        }
        in_slot = in_slot + 1 == E ? 0 : in_slot + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for_kinds(issue, std::make_integer_sequence<int, E - 1>{});
    __syncwarp();

    int slot = 0, tile_at = 0;
    auto next_entry = [&](auto kind_) {   // all warps' rows of the entry have landed; all are through with the one before it
        asm volatile("cp.async.wait_group %0;" ::"n"(E - 2) : "memory");
        __syncthreads();
        issue(std::integral_constant<int, decltype(kind_)::value + E - 1>{});
        const uint8_t *ent = sm + S::o_ring + slot * S::kEntry;
        slot = slot + 1 == E ? 0 : slot + 1;
        return ent;
    };

    for (int done = 0; done < walk.opened; ++done) {
        const PagedSegment g = walk.segs[done % S::kSegs];
        const int R = g.rows * G;
        build_queries<S>(a, g, sm + S::o_q, col_s);
        if (tid < S::kRows) {   // the last position that a row sees (-1: none, or no such row)
            const int r = g.rb * S::kRows + tid;
            lim_s[tid] = r < R ? g.length - g.rows + r / G : -1;
        }
        __syncthreads();
        // rows of this block: all see [all_lo, all_hi]
        const int t_first = g.rb * S::kRows / G, t_last = (min(R, (g.rb + 1) * S::kRows) - 1) / G;
        const int all_hi = g.length - g.rows + t_first;
        const int all_lo = a.x.window > 0 ? g.length - g.rows + t_last + 1 - a.x.window : 0;
        float o[MW][NT][4], m[NT][2], mo[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) m[nt][c] = mo[nt][c] = -INFINITY, l[nt][c] = 0.0f;
#pragma unroll
            for (int k = 0; k < MW; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[k][nt][c] = 0.0f;
        }
        for (int i = 0; i < g.n; ++i) {
            const int tile0 = g.lo + (g.t0 + i) * S::CT, p0 = tile0 + warp * TP;
            const bool edge = tile0 < all_lo || tile0 + S::CT - 1 > all_hi;
            // ---- S^T = K Q^T of this warp's 16 positions
            const uint8_t *ent = next_entry(std::integral_constant<int, 0>{}) + warp * TP * RB;
            const KeyFragments<RB> keys(ent);
            float s[NT][4];
            if constexpr (I8) {
                // (sums on top of 1.5 * 2^23, whose float neighbours are the integers)
                int32_t acc[NT][3][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int y = 0; y < 3; ++y)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[nt][y][c] = static_cast<int32_t>(kBiasBits);
#pragma unroll 2   // (unrolled whole, the kernel outgrows the instruction cache)
                for (int ks = 0; ks < RB / 32; ++ks) {
                    const uint4 k = keys(ks);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 ab = q_two[(ks * NT + nt) * 32 + lane];
                        const uint2 cc = q_one[(ks * NT + nt) * 32 + lane];
                        mma_s8_16832(acc[nt][0], k.x, k.y, k.z, k.w, ab.x, ab.y);
                        mma_s8_16832(acc[nt][1], k.x, k.y, k.z, k.w, ab.z, ab.w);
                        mma_s8_16832(acc[nt][2], k.x, k.y, k.z, k.w, cc.x, cc.y);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[nt][c] = digits_sum(acc[nt][0][c], acc[nt][1][c], acc[nt][2][c]);
            } else {
                float lo[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[nt][c] = lo[nt][c] = 0.0f;
#pragma unroll 4
                for (int ks = 0; ks < RB / 32; ++ks) {
                    const uint4 k = keys(ks);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 b2 = SPLIT ? q_two[(ks * NT + nt) * 32 + lane] : make_uint4(0, 0, 0, 0);
                        const uint2 b = SPLIT ? make_uint2(b2.x, b2.y) : q_one[(ks * NT + nt) * 32 + lane];
                        mma_16816<BF16>(s[nt], k.x, k.y, k.z, k.w, b.x, b.y);
                        if constexpr (SPLIT) mma_16816<BF16>(lo[nt], k.x, k.y, k.z, k.w, b2.z, b2.w);
                        if constexpr (S::THREE) {
                            const uint2 b3 = q_one[(ks * NT + nt) * 32 + lane];
                            mma_16816<BF16>(lo[nt], k.x, k.y, k.z, k.w, b3.x, b3.y);
                        }
                    }
                }
                if constexpr (SPLIT)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[nt][c] += lo[nt][c];
            }
            // ---- scores in bits, masks, does a maximum grow far
            const uint8_t *sc = scales + tile_at * S::kScale;
            tile_at = tile_at + 1 == S::TS ? 0 : tile_at + 1;
            const uint32_t bits = *reinterpret_cast<const uint32_t *>(sc);
            const float *sv = reinterpret_cast<const float *>(sc + 16);
            const bool masked = edge || bits != 0xffffu;
            float ks[2] = {1.0f, 1.0f}, lv[2] = {0.0f, 0.0f};
            if constexpr (I8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) ks[h] = sv[8 * h + gid], lv[h] = lg2(sv[TP + 8 * h + gid]);
            }
            // an unseen scale may be anything: -inf + log2 vs is then no number, which the maxima pass over; the weight of
            // such a score (a bit of hidden) is set to 0
            uint32_t hidden = 0;
            const bool strange = I8 && masked && __any_sync(0xffffffffu, !(lv[0] < INFINITY) || !(lv[1] < INFINITY));
            bool grows = false;
            auto value = [&](int nt, int x) { return s[nt][x] + lv[x >> 1]; };
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 col = *reinterpret_cast<const float2 *>(col_s + 8 * nt + 2 * tig);
#pragma unroll
                for (int x = 0; x < 4; ++x) s[nt][x] *= (x & 1 ? col.y : col.x) * ks[x >> 1];
                if (masked) {
                    const int2 lim = *reinterpret_cast<const int2 *>(lim_s + 8 * nt + 2 * tig);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int p = 8 * (x >> 1) + gid, gp = p0 + p, last = x & 1 ? lim.y : lim.x;
                        if (gp > last || !(bits >> p & 1) || (a.x.window > 0 && gp <= last - a.x.window)) {
                            s[nt][x] = -INFINITY;
                            hidden |= 1u << (4 * nt + x);
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    grows = grows || fmaxf(s[nt][c], s[nt][2 + c]) > m[nt][c] + kSlack;
                    if constexpr (I8) grows = grows || fmaxf(value(nt, c), value(nt, 2 + c)) > mo[nt][c] + (kWeightBias + kSlack);
                }
            }
            if (__syncthreads_or(grows)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = fmaxf(s[nt][c], s[nt][2 + c]), topo = I8 ? fmaxf(value(nt, c), value(nt, 2 + c)) : 0.0f;
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            if constexpr (I8) topo = fmaxf(topo, __shfl_xor_sync(0xffffffffu, topo, x));
                        }
                        if (gid == 0) max_s[warp * S::kRows + 8 * nt + 2 * tig + c] = make_float2(top, topo);
                    }
                __syncthreads();
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mn = m[nt][c], on = mo[nt][c];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 x = max_s[w * S::kRows + 8 * nt + 2 * tig + c];
                            mn = fmaxf(mn, x.x);
                            if constexpr (I8) on = fmaxf(on, x.y - kWeightBias);
                        }
                        if constexpr (!I8) on = BF16 ? mn : mn - kWeightBias;
                        l[nt][c] *= m[nt][c] == -INFINITY ? 0.0f : ex2(m[nt][c] - mn);
                        const float f = mo[nt][c] == -INFINITY ? 0.0f : ex2(mo[nt][c] - on);
                        m[nt][c] = mn;
                        mo[nt][c] = on;
#pragma unroll
                        for (int k = 0; k < MW; ++k) o[k][nt][c] *= f, o[k][nt][2 + c] *= f;
                    }
            }
            // ---- weights, as the second product's fragments
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int c = x & 1;
                    const float oz = mo[nt][c] == -INFINITY ? 0.0f : mo[nt][c];
                    if constexpr (I8) {
                        const float mz = m[nt][c] == -INFINITY ? 0.0f : m[nt][c];
                        l[nt][c] += ex2(s[nt][x] - mz);
                        w[x] = ex2(value(nt, x) - oz);
                    } else {
                        w[x] = ex2(s[nt][x] - oz);
                        l[nt][c] += BF16 ? w[x] : w[x] * 0.015625f;   // 2^-kWeightBias
                    }
                }
                if (strange)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (hidden >> (4 * nt + x) & 1) w[x] = 0.0f;
                uint32_t part[PN][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = w[2 * h], y = w[2 * h + 1];
#pragma unroll
                    for (int n = 0; n < PN; ++n) {
                        const uint32_t b = pack2<BF16>(x, y);
                        part[n][h] = move_trans(b);
                        const float2 held = unpack2<BF16>(b);
                        x -= held.x, y -= held.y;
                    }
                }
                const int f = (warp * NT + nt) * 32 + lane;
                reinterpret_cast<uint4 *>(sm + S::o_p)[f] = make_uint4(part[0][0], part[0][1], part[1][0], part[1][1]);
                if constexpr (S::THREE) reinterpret_cast<uint2 *>(sm + S::o_p + S::kPTwo)[f] = make_uint2(part[2][0], part[2][1]);
            }
            // ---- O^T += V^T P^T of this warp's dims
            const uint8_t *ev = next_entry(std::integral_constant<int, 1>{});   // (its barrier: the weights are there too)
            constexpr int NB = S::DL * S::ES, NW = NB < 4 ? 1 : NB / 4;   // bytes, words of a lane's dims
            auto v_words = [&](int kt, uint32_t (&x)[4][NW]) {   // positions 2 tig, + 1, + 8, + 9 of 16
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int p = 16 * kt + 2 * tig + (k & 1) + 8 * (k >> 1), at = warp * (RB / 4) + gid * NB;
                    const int sw = RB == 64 ? (at >> 4) ^ ((p >> 1 & 1) << 1) : (at >> 4) ^ ((p >> 1 & 3) << 1);
                    const uint8_t *from = ev + p * RB + sw * 16 + (at & 15);
                    if constexpr (NB == 16) {
                        const uint4 t = *reinterpret_cast<const uint4 *>(from);
                        x[k][0] = t.x, x[k][1] = t.y, x[k][2] = t.z, x[k][3] = t.w;
                    } else if constexpr (NB == 8) {
                        const uint2 t = *reinterpret_cast<const uint2 *>(from);
                        x[k][0] = t.x, x[k][1] = t.y;
                    } else if constexpr (NB == 4) {
                        x[k][0] = *reinterpret_cast<const uint32_t *>(from);
                    } else {
                        x[k][0] = *reinterpret_cast<const uint16_t *>(from);
                    }
                }
            };
            auto v_frags = [&](const uint32_t (&x)[4][NW], uint32_t (&va)[MW][4]) {
#pragma unroll
                for (int w = 0; w < NW; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t xa = x[2 * h][w], xb = x[2 * h + 1][w];
                        if constexpr (I8) {
                            widen4(__byte_perm(xa, xb, 0x5140), va[2 * w < MW ? 2 * w : 0][2 * h], va[2 * w < MW ? 2 * w : 0][2 * h + 1]);
                            if constexpr (MW > 1) widen4(__byte_perm(xa, xb, 0x7362), va[2 * w + 1][2 * h], va[2 * w + 1][2 * h + 1]);
                        } else {
                            va[w][2 * h] = __byte_perm(xa, xb, 0x5410);
                            va[w][2 * h + 1] = __byte_perm(xa, xb, 0x7632);
                        }
                    }
            };
            auto weights = [&](int kt, int nt) { return reinterpret_cast<const uint4 *>(sm + S::o_p)[(kt * NT + nt) * 32 + lane]; };
            auto third = [&](int kt, int nt) { return reinterpret_cast<const uint2 *>(sm + S::o_p + S::kPTwo)[(kt * NT + nt) * 32 + lane]; };
            // (values that a row does not see: as in k_paged_attn)
            bool apart = false;
            if constexpr (!I8) {
                if (edge && g.rows > 1) {
                    bool odd = false;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) {
                        uint32_t x[4][NW];
                        v_words(kt, x);
                        constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int w = 0; w < NW; ++w)
                                odd = odd || (x[k][w] & kExp) == kExp || (x[k][w] & (kExp << 16)) == (kExp << 16);
                    }
                    apart = __any_sync(0xffffffffu, odd);
                }
            }
            if (!apart) {
#pragma unroll 1
                for (int kt = 0; kt < 4; ++kt) {
                    uint32_t x[4][NW], va[MW][4];
                    v_words(kt, x);
                    v_frags(x, va);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 b = weights(kt, nt);
#pragma unroll
                        for (int k = 0; k < MW; ++k) mma_16816<BF16>(o[k][nt], va[k][0], va[k][1], va[k][2], va[k][3], b.x, b.y);
#pragma unroll
                        for (int k = 0; k < MW; ++k) mma_16816<BF16>(o[k][nt], va[k][0], va[k][1], va[k][2], va[k][3], b.z, b.w);
                        if constexpr (S::THREE) {
                            const uint2 c = third(kt, nt);
#pragma unroll
                            for (int k = 0; k < MW; ++k) mma_16816<BF16>(o[k][nt], va[k][0], va[k][1], va[k][2], va[k][3], c.x, c.y);
                        }
                    }
                }
            } else if constexpr (!I8) {
                for (int t = 0; t < g.rows; ++t) {
                    const int last = g.length - g.rows + t, hi_p = last - tile0, lo_p = a.x.window > 0 ? hi_p - a.x.window + 1 : -(1 << 30);
#pragma unroll 1
                    for (int kt = 0; kt < 4; ++kt) {
                        uint32_t x[4][NW], va[MW][4];
                        v_words(kt, x);
                        v_frags(x, va);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int p = 16 * kt + 2 * tig + 8 * h;
                            const uint32_t keep = (p >= lo_p && p <= hi_p ? 0xffffu : 0u) | (p + 1 >= lo_p && p + 1 <= hi_p ? 0xffff0000u : 0u);
#pragma unroll
                            for (int k = 0; k < MW; ++k) va[k][2 * h] &= keep, va[k][2 * h + 1] &= keep;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint4 b = weights(kt, nt);
                            const int2 lim = *reinterpret_cast<const int2 *>(lim_s + 8 * nt + 2 * tig);
#pragma unroll
                            for (int k = 0; k < MW; ++k) {
                                float d[4] = {o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]};
                                mma_16816<BF16>(d, va[k][0], va[k][1], va[k][2], va[k][3], b.x, b.y);
                                mma_16816<BF16>(d, va[k][0], va[k][1], va[k][2], va[k][3], b.z, b.w);
                                if constexpr (S::THREE) {
                                    const uint2 c = third(kt, nt);
                                    mma_16816<BF16>(d, va[k][0], va[k][1], va[k][2], va[k][3], c.x, c.y);
                                }
#pragma unroll
                                for (int y = 0; y < 4; ++y)
                                    if ((y & 1 ? lim.y : lim.x) == last && last >= 0) o[k][nt][y] = d[y];
                            }
                        }
                    }
                }
            }
        }
        // ---- the segment's end: the positions' sums of weights over lanes and warps, then out or to the scratch
        float *sum_s = reinterpret_cast<float *>(max_s);
        __syncthreads();   // (the maxima's last readers are through)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
                if (gid == 0) sum_s[warp * S::kRows + 8 * nt + 2 * tig + c] = l[nt][c];
            }
        __syncthreads();
        const bool whole = g.t0 == 0 && g.n == g.tps;
        const int keep_slot = 2 * cta + (g.no == 0 ? 0 : 1);
        if (g.parts > 0 && tid == 0) a.cut[cta] = make_int4(2 * g.parts + (keep_slot & 1), g.item, g.r0, g.rows);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (g.rb * S::kRows + 8 * nt >= R) break;
            float Ls[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Ls[c] = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) Ls[c] += sum_s[w * S::kRows + 8 * nt + 2 * tig + c];
            }
            const float inv0 = row_factor(m[nt][0], Ls[0], mo[nt][0]), inv1 = row_factor(m[nt][1], Ls[1], mo[nt][1]);
            float4 v[MW];
#pragma unroll
            for (int k = 0; k < MW; ++k) v[k] = make_float4(o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]);
            if (whole) {
                if constexpr (MW == 1) {
                    write_one<S>(a, g.r0, g.rows, g.item, nt, warp, v[0], inv0, inv1);
                } else {
#pragma unroll
                    for (int k = 0; k < MW; k += 2) write_out<S>(a, g.r0, g.rows, g.item, nt, warp * MW + k, v[k], v[k + 1], inv0, inv1);
                }
            } else {
                float4 *d = a.part + ((static_cast<int64_t>(keep_slot) * NT + nt) * OM + warp * MW) * 32 + lane;
#pragma unroll
                for (int k = 0; k < MW; ++k) d[32 * k] = v[k];
            }
            if (warp == 0 && gid == 0)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int i = 8 * nt + 2 * tig + c;
                    if (whole) write_lse<S>(a, g.r0, g.rows, g.item, i, m[nt][c], Ls[c]);
                    else a.stats[static_cast<int64_t>(keep_slot) * S::kRows + i] = make_float4(m[nt][c], Ls[c], mo[nt][c], 0.0f);
                }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace gcu
