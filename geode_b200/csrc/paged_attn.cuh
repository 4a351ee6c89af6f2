// paged_attn.cuh - attention of each sequence's newest rows over its pages (flash decoding over a paged cache).
//
// An item is one (sequence, key head, block of query rows): the sequence's T rows times the G query heads that share the
// key head, R = T * G rows in blocks of kRows. Items are cut into tiles of positions and the tiles of all items, laid end
// to end, are dealt out evenly to the resident CTAs (each CTA finds its share by a scan over the lengths on the device:
// whatever the lengths, every CTA reads the same number of tiles). What a CTA holds of an item that it does not finish
// goes to the scratch and k_paged_attn_join adds the parts up.
//
// Both products run on the tensor cores (mma.sync m16n8k16, float sums) with the cache as the 16-row operand and the
// query rows as the 8-column one, so that one token's few rows fill the instruction: S^T = K Q^T, then O^T = V^T P^T.
// The order of dims inside a product is free as long as both operands agree, so a lane takes 16 consecutive bytes of a
// cache row as its fragments of several products: no transposition, no staging of widened rows. int8 codes are widened
// to f16 in registers (exact).
//
// Arithmetic: queries are f16 scaled by a power of two per row (bf16 for a bf16 cache). Float activations, and f16 ones
// over a bf16 cache, are held as a sum of two such numbers, the weights too: 22 bits (16 for bf16). Otherwise a weight
// is rounded once to 16 bits, an error of at most half a step relative to each weight, below the output's own rounding.
// int8 rows' value scales go into the weight's exponent: w = 2^(s + log2 vs - m'), with a maximum m' of its own, so that
// rows of any scale keep their bits. Scores, sums, maxima and outputs are float.
#pragma once

#include "paged.cuh"
#include "paged_attn_plan.hpp"

namespace gcu {

struct PagedAttnArgs {
    gcuda_paged_kv kv;
    gcuda_paged_batch b;
    gcuda_attn_rows x;
    uint32_t *status;
    int4 *desc;      // [grid][2] the parts that CTAs left: {flags, item, first row, rows}
    float4 *stats;   // [grid][2][kRows] {m, l, m', -} of each row
    float4 *part;    // [grid][2][n tile][m tile][lane]
};

constexpr int kPagedAttnThreads = 128;
constexpr int kPartHeld = 1, kPartStarts = 2, kPartEnds = 4;   // desc flags
constexpr float kWeightBias = 14.0f;   // f16 weights reach up to 2^14: the smallest kept is 2^-39 of the largest

// Shapes of one instantiation. NT: n tiles (8 query rows) a warp; WR: warps that share the positions (each with its own
// rows; the CTA's other factor, 4 / WR, takes positions).
template <int HD_, int CACHE_, bool SPLIT_, int NT_, int WR_>
struct PagedShape {
    static constexpr int HD = HD_, CACHE = CACHE_, NT = NT_, WR = WR_;
    static constexpr bool SPLIT = SPLIT_, I8 = CACHE == GCUDA_I8, BF16 = CACHE == GCUDA_BF16;
    static constexpr int WP = 4 / WR;
    static constexpr int ES = I8 ? 1 : 2, RB = HD * ES;          // bytes of a value, of a row
    static constexpr int MT = RB <= 128 || (RB == 256 && NT == 1) ? 2 : 1, TP = 16 * MT;   // positions of a warp's tile
    static constexpr int CT = TP * WP;                            // of a CTA's
    static constexpr int NTT = NT * WR, kRows = 8 * NTT;
    static constexpr int KS = HD / 16, OM = HD / 16;
    static constexpr int kEntry = TP * RB;                        // a tile's K or V rows in shared memory
    static constexpr int kRing = (WR > 1 ? 40 : NT == 1 || RB == 512 ? 24 : 20) * 1024;   // bytes of a position group's ring
    static constexpr int E = kRing / kEntry < 12 ? kRing / kEntry : 12;
    static constexpr int kScale = 2 * TP * 4 + 16;                // a slot's scales and valid bits
    static constexpr int kQ = KS * NTT * 32 * 8 * (SPLIT ? 2 : 1);
    static constexpr int kJoin = WR == 1 ? 4 * NT * OM * 32 * 16 : 0;   // (over the ring, drained)
    static constexpr int kRings = WP * E * kEntry > kJoin ? WP * E * kEntry : kJoin;
    static constexpr int o_q = 0, o_ring = o_q + kQ, o_scale = o_ring + kRings;
    static constexpr int o_col = o_scale + WP * E * kScale;       // [kRows] column factor
    static constexpr int o_join = o_col + kRows * 4;              // [4][kRows] m, l, m' of each position group
    static constexpr int kSmem = o_join + (WR == 1 ? 4 * kRows * 16 : 0);
    static_assert(E >= 3, "two entries in flight");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t move_trans(uint32_t x) {   // an 8x8 matrix of 16-bit values, transposed
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// two floats in the product's 16-bit type (lo the lower half); and what is left of each
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t r) {
    if constexpr (BF16) return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<__half2 *>(&r));
}
// four int8 (a word) -> two f16 pairs, exactly: the byte with its sign flipped under the f16 exponent of 1024 is
// 1024 + b + 128
__device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t x = w ^ 0x80808080u;
    lo = __byte_perm(x, 0x64646464u, 0x5140);
    hi = __byte_perm(x, 0x64646464u, 0x7362);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
    const __half2 l = __hsub2(*reinterpret_cast<__half2 *>(&lo), off), h = __hsub2(*reinterpret_cast<__half2 *>(&hi), off);
    lo = *reinterpret_cast<const uint32_t *>(&l);
    hi = *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {   // (bytes 0: zeros)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float load_act(const void *p, int type, int64_t i) {
    if (type == GCUDA_F32) return static_cast<const float *>(p)[i];
    if (type == GCUDA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_act4(void *p, int type, int64_t i, float4 v) {   // (rows of out are packed heads: aligned by 4 or by 1)
    const float f[4] = {v.x, v.y, v.z, v.w};
    if (type == GCUDA_F32) {
        float *d = static_cast<float *>(p) + i;
        if ((reinterpret_cast<uintptr_t>(d) & 15) == 0) *reinterpret_cast<float4 *>(d) = v;
        else
            for (int k = 0; k < 4; ++k) d[k] = f[k];
        return;
    }
    const uint32_t lo = type == GCUDA_BF16 ? pack2<true>(v.x, v.y) : pack2<false>(v.x, v.y);
    const uint32_t hi = type == GCUDA_BF16 ? pack2<true>(v.z, v.w) : pack2<false>(v.z, v.w);
    uint16_t *d = static_cast<uint16_t *>(p) + i;
    if ((reinterpret_cast<uintptr_t>(d) & 7) == 0) *reinterpret_cast<uint2 *>(d) = make_uint2(lo, hi);
    else {
        d[0] = static_cast<uint16_t>(lo), d[1] = static_cast<uint16_t>(lo >> 16);
        d[2] = static_cast<uint16_t>(hi), d[3] = static_cast<uint16_t>(hi >> 16);
    }
}

// The dims of m tile m's rows gid and gid + 8: the first of the two neighbours (a lane's 8th of a row is taken in pieces
// of at most 16 bytes, 8 pieces side by side)
template <int HD, int ES>
__device__ __forceinline__ int dim_of(int m, int gid) {
    constexpr int PB = HD * ES / 8 < 16 ? HD * ES / 8 : 16, DPP = PB / ES;
    return 2 * m / DPP * 8 * DPP + gid * DPP + 2 * m % DPP;
}

// One row block's finished values of m tiles m, m + 1 (four neighbouring dims) of the rows 2 tig, 2 tig + 1 of an n tile
template <typename S>
__device__ __forceinline__ void write_out(const PagedAttnArgs &a, int r0, int rows, int item, int nt, int m, const float4 &x,
                                          const float4 &y, float inv0, float inv1) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = rows * G, nrb = (R + S::kRows - 1) / S::kRows;
    const int kh = item / nrb, rb = item % nrb, d = dim_of<S::HD, S::ES>(m, gid);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int r = rb * S::kRows + 8 * nt + 2 * tig + c;
        if (r >= R) continue;
        const float inv = c ? inv1 : inv0;
        const int64_t at = static_cast<int64_t>(r0 + r / G) * a.x.out_stride + static_cast<int64_t>(kh * G + r % G) * S::HD + d;
        store_act4(a.x.out, a.x.type, at,
                   c ? make_float4(x.y * inv, x.w * inv, y.y * inv, y.w * inv) : make_float4(x.x * inv, x.z * inv, y.x * inv, y.z * inv));
    }
}
// a row's factor 1 / l (with O's own exponent) from its joined (m, l, m'): zeros where it saw nothing
__device__ __forceinline__ float row_factor(float m, float l, float mo) { return l == 0.0f ? 0.0f : ex2(mo - m) / l; }
template <typename S>
__device__ __forceinline__ void write_lse(const PagedAttnArgs &a, int r0, int rows, int item, int i, float m, float l) {
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = rows * G, nrb = (R + S::kRows - 1) / S::kRows;
    const int kh = item / nrb, r = item % nrb * S::kRows + i;
    if (!a.x.lse || r >= R) return;
    // log of the sum: in bits, then times ln 2
    a.x.lse[static_cast<int64_t>(r0 + r / G) * a.x.n_heads + kh * G + r % G] =
        l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

// The positions [lo, hi) that a sequence's rows see between them, and its tiles a (key head, row block)
template <typename S>
__device__ __forceinline__ int seq_tiles(const PagedAttnArgs &a, const SeqRows &q, int &lo) {
    lo = a.x.window > 0 ? max(0, q.length - q.rows + 1 - a.x.window) : 0;
    return max(1, (q.length - lo + S::CT - 1) / S::CT);
}
template <typename S>
__device__ __forceinline__ int64_t all_tiles(const PagedAttnArgs &a, const SeqRows &q) {
    if (q.rows == 0) return 0;
    int lo;
    const int64_t t = seq_tiles<S>(a, q, lo);
    return t * a.kv.n_kv_heads * ((q.rows * (a.x.n_heads / a.kv.n_kv_heads) + S::kRows - 1) / S::kRows);
}

template <typename S>
__global__ void __launch_bounds__(kPagedAttnThreads, 2) k_paged_attn(PagedAttnArgs a) {
    constexpr int HD = S::HD, NT = S::NT, WR = S::WR, TP = S::TP, MT = S::MT, RB = S::RB, E = S::E, OM = S::OM;
    constexpr int A = E / 2 + 1;   // tiles whose pages are looked up ahead
    constexpr bool I8 = S::I8, BF16 = S::BF16, SPLIT = S::SPLIT;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ int64_t s_sum[4], s_base;
    __shared__ int s_seq;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int wp = warp / WR, wr = warp % WR;
    const int G = a.x.n_heads / a.kv.n_kv_heads, cta = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    // this CTA's share [u, end) of all tiles: each thread sums a run of sequences, then a scan over the threads
    if (tid < 2) a.desc[2 * cta + tid] = make_int4(0, 0, 0, 0);
    const int run = (a.b.n_seq + kPagedAttnThreads - 1) / kPagedAttnThreads;
    const int s_lo = min(tid * run, a.b.n_seq), s_hi = min(s_lo + run, a.b.n_seq);
    int64_t mine = 0;
    for (int s = s_lo; s < s_hi; ++s) mine += all_tiles<S>(a, seq_rows(a.b, a.kv.page_size, s, a.status));
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    before -= mine;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
    if (cta >= ctas) return;
    const int64_t begin = total * cta / ctas, end = total * (cta + 1) / ctas;
    if (before <= begin && begin < before + mine) {
        int64_t base = before;
        int s = s_lo;
        for (; s < s_hi; ++s) {
            const int64_t n = all_tiles<S>(a, seq_rows(a.b, a.kv.page_size, s, a.status));
            if (begin < base + n) break;
            base += n;
        }
        s_seq = s;
        s_base = base;
    }
    __syncthreads();
    int seq = s_seq;
    int64_t base = s_base, u = begin;

    uint2 *q_hi = reinterpret_cast<uint2 *>(sm + S::o_q);       // fragments (b0, b1) [k step][n tile][lane]; SPLIT: uint4
    uint4 *q_both = reinterpret_cast<uint4 *>(sm + S::o_q);
    float *col_s = reinterpret_cast<float *>(sm + S::o_col);
    float4 *join_s = reinterpret_cast<float4 *>(sm + S::o_join);
    uint8_t *ring = sm + S::o_ring + wp * E * S::kEntry;
    uint8_t *scales = sm + S::o_scale + wp * E * S::kScale;
    const uint32_t ring_a = smem_addr(ring), scales_a = smem_addr(scales);
    const uint8_t *kb = static_cast<const uint8_t *>(a.kv.k), *vb = static_cast<const uint8_t *>(a.kv.v);

    while (u < end) {
        const SeqRows q = seq_rows(a.b, a.kv.page_size, seq, a.status);
        if (q.rows == 0) {
            ++seq;
            continue;
        }
        int lo;
        const int tps = seq_tiles<S>(a, q, lo), R = q.rows * G, nrb = (R + S::kRows - 1) / S::kRows;
        const int item = static_cast<int>((u - base) / tps), t0 = static_cast<int>((u - base) % tps);
        const int t1 = static_cast<int>(min(static_cast<int64_t>(tps), t0 + (end - u)));
        const int kh = item / nrb, rb = item % nrb;
        const int *pages = a.b.pages + seq * a.b.pages_stride;

        // ---- the copies: entry 2 i is tile i's K rows, entry 2 i + 1 its V rows; a lane knows one position's place
        const int n_tiles = t1 - t0, first = lo + t0 * S::CT + wp * TP;   // this group's first position
        int64_t place = 0;    // value offset of this lane's position (of the tile whose K was last issued)
        bool there = false;
        int page[A] = {};     // the pages of this lane's positions in the tiles whose K is issued next
        auto load_page = [&](int i) {
            const int p = first + i * S::CT + lane;
            return (i < n_tiles && lane < TP && p < q.length) ? pages[p / a.kv.page_size] : -1;
        };
        auto issue = [&](int e) {
            if (e < 2 * n_tiles) {
                const int slot = e % E, i = e >> 1;
                if (!(e & 1)) {
                    const int p = first + i * S::CT + lane;
                    const int pg = page[0];
#pragma unroll
                    for (int k = 0; k + 1 < A; ++k) page[k] = page[k + 1];
                    page[A - 1] = load_page(i + A);
                    there = pg >= 0 && pg < a.kv.n_pages;
                    if (lane < TP && p < q.length && !there) atomicOr(a.status, kErrBadShape);
                    const int ip = p % a.kv.page_size;
                    place = there ? pg * a.kv.page_stride + ip * a.kv.pos_stride + kh * a.kv.head_stride : 0;
                    const uint32_t bits = __ballot_sync(0xffffffffu, there);
                    if (wr == 0) {
                        uint8_t *sc = scales + slot * S::kScale;
                        if (lane == 0) *reinterpret_cast<uint32_t *>(sc + 2 * TP * 4) = bits;
                        if constexpr (I8) {
                            if (lane < TP) {
                                const int64_t sp = there ? pg * a.kv.scale_page_stride + ip * a.kv.scale_pos_stride + kh * a.kv.scale_head_stride : 0;
                                const uint32_t d = scales_a + slot * S::kScale + lane * 4;
                                copy4(d, a.kv.k_scale + sp, there ? 4 : 0);
                                copy4(d + TP * 4, a.kv.v_scale + sp, there ? 4 : 0);
                            }
                        }
                    }
                }
                const uint8_t *src = (e & 1) ? vb : kb;
                constexpr int CH = RB / 16;   // 16-byte pieces of a row
                const uint32_t ok = __ballot_sync(0xffffffffu, there);
#pragma unroll
                for (int k = 0; k < TP * CH / (32 * WR); ++k) {
                    const int idx = (k * WR + wr) * 32 + lane, p = idx / CH, c = idx % CH;
                    const int64_t at = __shfl_sync(0xffffffffu, place, p);
                    // pieces swapped within a row so that the fragment loads of K (8 rows x 4 pieces of 4 neighbouring
                    // lanes) and of V (every second row x 2 pieces) meet no bank twice
                    int sw;
                    if (e & 1) sw = RB == 64 ? c ^ ((p >> 1 & 1) << 1) : c ^ ((p >> 1 & 3) << 1);
                    else sw = RB == 64 ? c : c ^ ((p & 1) << 2);
                    copy16(ring_a + slot * S::kEntry + p * RB + sw * 16, src + at * S::ES + c * 16, (ok >> p & 1) ? 16 : 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < A; ++k) page[k] = load_page(k);
        __syncthreads();   // the last segment's shared memory is free
#pragma unroll
        for (int e = 0; e < E - 1; ++e) issue(e);

        // ---- the queries as fragments: warp w takes rows w, w + 4, ..; lane HD / 32 neighbouring dims
        for (int i = warp; i < S::kRows; i += 4) {
            constexpr int N = HD / 32;
            const int r = rb * S::kRows + i;
            float v[N], top = 0.0f;
            const int64_t at = r < R ? static_cast<int64_t>(q.r0 + r / G) * a.x.q_stride + static_cast<int64_t>(kh * G + r % G) * a.x.q_head_stride + lane * N : 0;
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = r < R ? load_act(a.x.q, a.x.type, at + k) : 0.0f;
            int ex = 0;
            if constexpr (!BF16) {
#pragma unroll
                for (int k = 0; k < N; ++k) top = fmaxf(top, fabsf(v[k]));
                top = warp_max(top);
                // 2^-ex brings the largest to [1, 2); zeros, infinities: as they are
                ex = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
#pragma unroll
                for (int k = 0; k < N; ++k) v[k] = scalbnf(v[k], -ex);
            }
            if (lane == 0) col_s[i] = scalbnf(a.x.scale * 1.44269504088896341f, ex);
            const int nt = i >> 3, n = i & 7;
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const int d = lane * N + k;
                constexpr int W = 16 / S::ES;   // dims of a 16-byte piece; 4 lanes' pieces side by side
                const int ks = d / (4 * W) * (W / 4) + d % W / 4, t = d % (4 * W) / W, b = d % 4 / 2;
                const int f = (ks * S::NTT + nt) * 32 + n * 4 + t;
                const uint32_t hi = pack2<BF16>(v[k], v[k + 1]);
                if constexpr (SPLIT) {
                    const float2 h = unpack2<BF16>(hi);
                    reinterpret_cast<uint32_t *>(q_both + f)[b] = hi;
                    reinterpret_cast<uint32_t *>(q_both + f)[2 + b] = pack2<BF16>(v[k] - h.x, v[k + 1] - h.y);
                } else {
                    reinterpret_cast<uint32_t *>(q_hi + f)[b] = hi;
                }
            }
        }
        __syncthreads();

        // ---- this lane's columns: rows 2 tig, 2 tig + 1 of each of the warp's n tiles
        float col[NT][2], m[NT][2], mo[NT][2], l[NT][2];
        int lim[NT][2];   // the last position that the row sees (-1: none, or no such row)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int i = 8 * (wr * NT + nt) + 2 * tig + c, r = rb * S::kRows + i;
                col[nt][c] = col_s[i];
                lim[nt][c] = r < R ? q.length - q.rows + r / G : -1;
                m[nt][c] = mo[nt][c] = -INFINITY;
                l[nt][c] = 0.0f;
            }
        // rows of this block: all see [all_lo, all_hi]
        const int t_first = rb * S::kRows / G, t_last = (min(R, (rb + 1) * S::kRows) - 1) / G;
        const int all_hi = q.length - q.rows + t_first;
        const int all_lo = a.x.window > 0 ? q.length - q.rows + t_last + 1 - a.x.window : 0;
        float o[OM][NT][4];
#pragma unroll
        for (int k = 0; k < OM; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[k][nt][c] = 0.0f;
        const bool busy = rb * S::kRows + 8 * wr * NT < R;   // this warp has rows

        uint32_t ph[MT][NT][2], pl[MT][NT][2];   // the weights as fragments: (b0, b1), and what is left of them
        bool edge = false;
        for (int e = 0; e < 2 * n_tiles; ++e) {
            asm volatile("cp.async.wait_group %0;" ::"n"(E - 2) : "memory");
            if constexpr (WR == 1) __syncwarp();
            else __syncthreads();
            issue(e + E - 1);
            if (!busy) continue;
            const int slot = e % E, p0 = first + (e >> 1) * S::CT;
            const uint8_t *ent = ring + slot * S::kEntry;
            if (!(e & 1)) {
                // ---- S^T = K Q^T
                float s[MT][NT][4], s2[MT][NT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[mt][nt][c] = s2[mt][nt][c] = 0.0f;
#pragma unroll
                for (int j = 0; j < RB / 64; ++j) {
                    uint4 kg[MT][2];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int p = 16 * mt + 8 * h + gid, c = 4 * j + tig, sw = RB == 64 ? c : c ^ ((p & 1) << 2);
                            kg[mt][h] = *reinterpret_cast<const uint4 *>(ent + p * RB + sw * 16);
                        }
#pragma unroll
                    for (int w = 0; w < (I8 ? 4 : 2); ++w) {
                        const int ks = j * (I8 ? 4 : 2) + w;
                        uint32_t ka[MT][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t *x = reinterpret_cast<const uint32_t *>(&kg[mt][h]);
                                if constexpr (I8) widen4(x[w], ka[mt][h], ka[mt][2 + h]);
                                else ka[mt][h] = x[2 * w], ka[mt][2 + h] = x[2 * w + 1];
                            }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const int f = (ks * S::NTT + wr * NT + nt) * 32 + lane;
                            if constexpr (SPLIT) {
                                const uint4 b = q_both[f];
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    mma_16816<BF16>(s[mt][nt], ka[mt][0], ka[mt][1], ka[mt][2], ka[mt][3], b.x, b.y);
                                    mma_16816<BF16>(s2[mt][nt], ka[mt][0], ka[mt][1], ka[mt][2], ka[mt][3], b.z, b.w);
                                }
                            } else {
                                const uint2 b = q_hi[f];
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt)
                                    mma_16816<BF16>(s[mt][nt], ka[mt][0], ka[mt][1], ka[mt][2], ka[mt][3], b.x, b.y);
                            }
                        }
                    }
                }
                // ---- scores in bits, masks, running maxima
                const uint8_t *sc = scales + slot * S::kScale;
                const uint32_t bits = *reinterpret_cast<const uint32_t *>(sc + 2 * TP * 4);
                edge = p0 < all_lo || p0 + TP - 1 > all_hi;
                const bool masked = edge || bits != (TP == 32 ? 0xffffffffu : (1u << (TP & 31)) - 1u);
                float y[MT][NT][4];   // int8: s + log2 vs (masked on its own: an unseen scale may be anything)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int p = 16 * mt + 8 * h + gid;
                        float ks = 1.0f, lv = 0.0f;
                        if constexpr (I8) {
                            ks = reinterpret_cast<const float *>(sc)[p];
                            lv = lg2(reinterpret_cast<const float *>(sc)[TP + p]);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float &v = s[mt][nt][2 * h + c];
                                if constexpr (SPLIT) v += s2[mt][nt][2 * h + c];
                                v *= col[nt][c] * ks;
                                if constexpr (I8) y[mt][nt][2 * h + c] = v + lv;
                                if (masked) {
                                    const int gp = p0 + p;
                                    if (gp > lim[nt][c] || !(bits >> p & 1) || (a.x.window > 0 && gp <= lim[nt][c] - a.x.window)) {
                                        v = -INFINITY;
                                        if constexpr (I8) y[mt][nt][2 * h + c] = -INFINITY;
                                    }
                                }
                            }
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float top[2] = {-INFINITY, -INFINITY}, topo[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                top[c] = fmaxf(top[c], s[mt][nt][2 * h + c]);
                                if constexpr (I8) topo[c] = fmaxf(topo[c], y[mt][nt][2 * h + c]);
                            }
                    // (the maxima grow seldom: the reduction over the positions' lanes and the rescaling only then)
                    const bool grows = top[0] > m[nt][0] || top[1] > m[nt][1] ||
                                       (I8 && (topo[0] - kWeightBias > mo[nt][0] || topo[1] - kWeightBias > mo[nt][1]));
                    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) {
                                top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], x));
                                if constexpr (I8) topo[c] = fmaxf(topo[c], __shfl_xor_sync(0xffffffffu, topo[c], x));
                            }
                            const float mn = fmaxf(m[nt][c], top[c]);
                            l[nt][c] *= m[nt][c] == -INFINITY ? 0.0f : ex2(m[nt][c] - mn);
                            const float on = I8 ? fmaxf(mo[nt][c], topo[c] - kWeightBias) : BF16 ? mn : mn - kWeightBias;
                            const float f = mo[nt][c] == -INFINITY ? 0.0f : ex2(mo[nt][c] - on);
                            m[nt][c] = mn;
                            mo[nt][c] = on;
#pragma unroll
                            for (int k = 0; k < OM; ++k) {
                                o[k][nt][c] *= f;
                                o[k][nt][2 + c] *= f;
                            }
                        }
                    }
                    // weights: l sums them at float; the products take them in the 16-bit type
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int c = x & 1;
                            const float mz = m[nt][c] == -INFINITY ? 0.0f : m[nt][c];
                            const float oz = mo[nt][c] == -INFINITY ? 0.0f : mo[nt][c];
                            if constexpr (I8) {
                                l[nt][c] += ex2(s[mt][nt][x] - mz);
                                w[x] = ex2(y[mt][nt][x] - oz);
                            } else {
                                w[x] = ex2(s[mt][nt][x] - oz);
                                l[nt][c] += BF16 ? w[x] : w[x] * 6.103515625e-5f;   // 2^-14
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t hi = pack2<BF16>(w[2 * h], w[2 * h + 1]);
                            ph[mt][nt][h] = move_trans(hi);
                            if constexpr (SPLIT) {
                                const float2 b = unpack2<BF16>(hi);
                                pl[mt][nt][h] = move_trans(pack2<BF16>(w[2 * h] - b.x, w[2 * h + 1] - b.y));
                            }
                        }
                    }
                }
                continue;
            }
            // ---- O^T += V^T P^T
            constexpr int PB = RB / 8 < 16 ? RB / 8 : 16, NP = RB / 8 / PB, NW = PB / 4;
            auto v_words = [&](int mt, int np, uint32_t (&x)[4][NW]) {   // positions 2 tig, + 1, + 8, + 9
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int p = 16 * mt + 2 * tig + (k & 1) + 8 * (k >> 1);
                    const uint8_t *row = ent + p * RB;
                    if constexpr (PB == 16) {
                        const int c = np * 8 + gid, sw = c ^ ((p >> 1 & 3) << 1);
                        const uint4 t = *reinterpret_cast<const uint4 *>(row + sw * 16);
                        x[k][0] = t.x, x[k][1] = t.y, x[k][2] = t.z, x[k][3] = t.w;
                    } else {
                        const int c = gid >> 1, sw = c ^ ((p >> 1 & 1) << 1);
                        const uint2 t = *reinterpret_cast<const uint2 *>(row + sw * 16 + (gid & 1) * 8);
                        x[k][0] = t.x, x[k][1] = t.y;
                    }
                }
            };
            // a row must not be touched by values that it does not see, and zero times an infinity is not zero: at the
            // edges of what the rows see a 16-bit tile that holds such values goes a token at a time
            bool apart = false;
            if constexpr (!I8) {
                if (edge && q.rows > 1) {
                    bool odd = false;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int np = 0; np < NP; ++np) {
                            uint32_t x[4][NW];
                            v_words(mt, np, x);
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
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        uint32_t x[4][NW];
                        v_words(mt, np, x);
#pragma unroll
                        for (int w = 0; w < NW; ++w) {
                            constexpr int MW = I8 ? 2 : 1;   // m tiles of a word
                            uint32_t va[MW][4];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t xa = x[2 * h][w], xb = x[2 * h + 1][w];
                                if constexpr (I8) {
                                    widen4(__byte_perm(xa, xb, 0x5140), va[0][2 * h], va[0][2 * h + 1]);
                                    widen4(__byte_perm(xa, xb, 0x7362), va[MW - 1][2 * h], va[MW - 1][2 * h + 1]);
                                } else {
                                    va[0][2 * h] = __byte_perm(xa, xb, 0x5410);
                                    va[0][2 * h + 1] = __byte_perm(xa, xb, 0x7632);
                                }
                            }
#pragma unroll
                            for (int k = 0; k < MW; ++k) {
                                const int mo_i = (np * NW + w) * MW + k;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    mma_16816<BF16>(o[mo_i][nt], va[k][0], va[k][1], va[k][2], va[k][3], ph[mt][nt][0], ph[mt][nt][1]);
                                    if constexpr (SPLIT)
                                        mma_16816<BF16>(o[mo_i][nt], va[k][0], va[k][1], va[k][2], va[k][3], pl[mt][nt][0], pl[mt][nt][1]);
                                }
                            }
                        }
                    }
            } else if constexpr (!I8) {
                for (int t = 0; t < q.rows; ++t) {
                    const int hi_p = q.length - q.rows + t - p0, lo_p = a.x.window > 0 ? hi_p - a.x.window + 1 : -(1 << 30);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        uint32_t keep[2];   // the halves of positions 2 tig, 2 tig + 1 (and + 8) that token t sees
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int p = 16 * mt + 2 * tig + 8 * h;
                            keep[h] = (p >= lo_p && p <= hi_p ? 0xffffu : 0u) | (p + 1 >= lo_p && p + 1 <= hi_p ? 0xffff0000u : 0u);
                        }
#pragma unroll
                        for (int np = 0; np < NP; ++np) {
                            uint32_t x[4][NW];
                            v_words(mt, np, x);
#pragma unroll
                            for (int w = 0; w < NW; ++w) {
                                uint32_t va[4];
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    va[2 * h] = __byte_perm(x[2 * h][w], x[2 * h + 1][w], 0x5410) & keep[h];
                                    va[2 * h + 1] = __byte_perm(x[2 * h][w], x[2 * h + 1][w], 0x7632) & keep[h];
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma_16816<BF16>(d, va[0], va[1], va[2], va[3], ph[mt][nt][0], ph[mt][nt][1]);
                                    if constexpr (SPLIT) mma_16816<BF16>(d, va[0], va[1], va[2], va[3], pl[mt][nt][0], pl[mt][nt][1]);
#pragma unroll
                                    for (int x4 = 0; x4 < 4; ++x4)
                                        if (lim[nt][x4 & 1] - p0 == hi_p && lim[nt][x4 & 1] >= 0) o[np * NW + w][nt][x4] += d[x4];
                                }
                            }
                        }
                    }
                }
            }
        }
        // a lane summed its positions' weights: the others' of the column are on the lanes with the same tig
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);

        // ---- the segment's end: the position groups joined, then out or to the scratch
        const bool whole = t0 == 0 && t1 == tps;
        const int keep_slot = 2 * cta + (u == begin ? 0 : 1);
        if (!whole && tid == 0)
            a.desc[keep_slot] = make_int4(kPartHeld | (t0 == 0 ? kPartStarts : 0) | (t1 == tps ? kPartEnds : 0), item, q.r0, q.rows);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if constexpr (WR == 1) {
            __syncthreads();   // every warp is through with its ring
            float4 *buf = reinterpret_cast<float4 *>(sm + S::o_ring);   // [group][n tile][m tile][lane]
            if (gid == 0)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) join_s[warp * S::kRows + 8 * nt + 2 * tig + c] = make_float4(m[nt][c], l[nt][c], mo[nt][c], 0.0f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < OM; ++k)
                    buf[((warp * NT + nt) * OM + k) * 32 + lane] = make_float4(o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]);
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float M[2] = {-INFINITY, -INFINITY}, Mo[2] = {-INFINITY, -INFINITY}, Ls[2] = {0.0f, 0.0f}, f[4][2];
                float4 st[4][2];
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        st[w][c] = join_s[w * S::kRows + 8 * nt + 2 * tig + c];
                        M[c] = fmaxf(M[c], st[w][c].x);
                        Mo[c] = fmaxf(Mo[c], st[w][c].z);
                    }
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        Ls[c] += st[w][c].x == -INFINITY ? 0.0f : st[w][c].y * ex2(st[w][c].x - M[c]);
                        f[w][c] = st[w][c].z == -INFINITY ? 0.0f : ex2(st[w][c].z - Mo[c]);
                    }
                const float inv0 = row_factor(M[0], Ls[0], Mo[0]), inv1 = row_factor(M[1], Ls[1], Mo[1]);
                for (int k = 2 * warp; k < OM; k += 8) {
                    float4 v[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        v[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float4 x = buf[((w * NT + nt) * OM + k + h) * 32 + lane];
                            v[h].x += x.x * f[w][0], v[h].y += x.y * f[w][1], v[h].z += x.z * f[w][0], v[h].w += x.w * f[w][1];
                        }
                    }
                    if (whole) {
                        write_out<S>(a, q.r0, q.rows, item, nt, k, v[0], v[1], inv0, inv1);
                    } else {
                        float4 *d = a.part + ((static_cast<int64_t>(keep_slot) * NT + nt) * OM + k) * 32 + lane;
                        d[0] = v[0];
                        d[32] = v[1];
                    }
                }
                if (warp == 0 && gid == 0)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int i = 8 * nt + 2 * tig + c;
                        if (whole) write_lse<S>(a, q.r0, q.rows, item, i, M[c], Ls[c]);
                        else a.stats[static_cast<int64_t>(keep_slot) * S::kRows + i] = make_float4(M[c], Ls[c], Mo[c], 0.0f);
                    }
            }
        } else if (busy) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = wr * NT + nt;
                const float inv0 = row_factor(m[nt][0], l[nt][0], mo[nt][0]), inv1 = row_factor(m[nt][1], l[nt][1], mo[nt][1]);
#pragma unroll
                for (int k = 0; k < OM; k += 2) {
                    const float4 v0 = make_float4(o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]);
                    const float4 v1 = make_float4(o[k + 1][nt][0], o[k + 1][nt][1], o[k + 1][nt][2], o[k + 1][nt][3]);
                    if (whole) {
                        write_out<S>(a, q.r0, q.rows, item, n, k, v0, v1, inv0, inv1);
                    } else {
                        float4 *d = a.part + ((static_cast<int64_t>(keep_slot) * S::NTT + n) * OM + k) * 32 + lane;
                        d[0] = v0;
                        d[32] = v1;
                    }
                }
                if (gid == 0)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int i = 8 * n + 2 * tig + c;
                        if (whole) write_lse<S>(a, q.r0, q.rows, item, i, m[nt][c], l[nt][c]);
                        else a.stats[static_cast<int64_t>(keep_slot) * S::kRows + i] = make_float4(m[nt][c], l[nt][c], mo[nt][c], 0.0f);
                    }
            }
        }
        u += n_tiles;
        if (u - base == static_cast<int64_t>(tps) * a.kv.n_kv_heads * nrb) {
            base = u;
            ++seq;
        }
    }
}

// The parts of each item that was cut, joined. Main CTA c cuts an item when its share starts inside it; the item's first
// cut stands for it: its parts are main CTA c-1's last, then the first of c, c+1, .. up to the one that ends it. CTA
// (i, y) finds the i-th such c among the descriptors (all of them, in one round of loads) and joins the y-th pair of m
// tiles of an n tile: a warp takes every 8th part, eight in flight, then the warps' sums are joined in shared memory.
constexpr int kJoinThreads = 256;

template <typename S>
__global__ void __launch_bounds__(kJoinThreads) k_paged_attn_join(PagedAttnArgs a, int grid) {
    constexpr int OM = S::OM, W = kJoinThreads / 32;
    __shared__ uint32_t s_cut[kPagedMaxGrid / 32], s_end[kPagedMaxGrid / 32];
    __shared__ float4 s_stat[W][2][4], s_v[W][2][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tig = lane & 3, gid = lane >> 2;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    for (int c0 = 0; c0 < grid; c0 += kJoinThreads) {
        const int c = c0 + tid;
        int here = 0, prev = 0;
        if (c < grid) {
            here = a.desc[2 * c].x;
            if (c > 0) prev = a.desc[2 * c - 1].x, prev = prev & kPartHeld ? prev : a.desc[2 * c - 2].x;
        }
        const uint32_t cut = __ballot_sync(0xffffffffu, (here & kPartHeld) && !(here & kPartStarts) && (prev & kPartStarts) && !(prev & kPartEnds));
        const uint32_t end = __ballot_sync(0xffffffffu, c < grid && (here & kPartEnds));
        if (lane == 0) s_cut[c >> 5] = cut, s_end[c >> 5] = end;
    }
    __syncthreads();
    const int words = (grid + 31) / 32;
    int c = -1, left = blockIdx.x;
    for (int w = 0; w < words; ++w) {
        uint32_t bits = s_cut[w];
        const int n = __popc(bits);
        if (left >= n) {
            left -= n;
            continue;
        }
        for (; left > 0; --left) bits &= bits - 1;
        c = 32 * w + __ffs(bits) - 1;
        break;
    }
    if (c < 0) return;
    int last = c >> 5;   // the CTA that ends the item
    uint32_t ends = s_end[last] & (0xffffffffu << (c & 31));
    while (ends == 0 && last + 1 < words) ends = s_end[++last];
    last = ends ? 32 * last + __ffs(ends) - 1 : grid - 1;
    const int n = last - c + 2;
    const int4 item = a.desc[2 * c];
    const int slot0 = 2 * c - 1 - ((a.desc[2 * c - 1].x & kPartHeld) ? 0 : 1);
    auto slot = [&](int k) { return static_cast<int64_t>(k == 0 ? slot0 : 2 * (c + k - 1)); };
    const int nt = blockIdx.y / (OM / 2), k2 = blockIdx.y % (OM / 2) * 2;
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = item.w * G, nrb = (R + S::kRows - 1) / S::kRows;
    if (item.y % nrb * S::kRows + 8 * nt >= R) return;
    constexpr int B = 8;   // parts whose loads are in flight together
    float M[2] = {-INFINITY, -INFINITY}, Mo[2] = {-INFINITY, -INFINITY}, L[2] = {0.0f, 0.0f};
    float4 v[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    // parts or warps b = 0 .. n-1 of (stats of the lane's two rows, values of two m tiles) into M, Mo, L, v
    auto take = [&](const float4 (&st)[B][2], const float4 (&x)[B][2]) {
        float f0[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float mn = M[h], on = Mo[h];
#pragma unroll
            for (int b = 0; b < B; ++b) mn = fmaxf(mn, st[b][h].x), on = fmaxf(on, st[b][h].z);
            L[h] *= M[h] == -INFINITY ? 0.0f : ex2(M[h] - mn);
            f0[h] = Mo[h] == -INFINITY ? 0.0f : ex2(Mo[h] - on);
            M[h] = mn;
            Mo[h] = on;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h].x *= f0[0], v[h].y *= f0[1], v[h].z *= f0[0], v[h].w *= f0[1];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                L[h] += st[b][h].x == -INFINITY ? 0.0f : st[b][h].y * ex2(st[b][h].x - M[h]);
                f[h] = st[b][h].z == -INFINITY ? 0.0f : ex2(st[b][h].z - Mo[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) v[h].x += x[b][h].x * f[0], v[h].y += x[b][h].y * f[1], v[h].z += x[b][h].z * f[0], v[h].w += x[b][h].w * f[1];
        }
    };
    float4 st[B][2], x[B][2];
    for (int k0 = warp; k0 < n; k0 += W * B) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const bool in = k0 + b * W < n;
            const int64_t at = slot(in ? k0 + b * W : 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                st[b][h] = in ? a.stats[at * S::kRows + 8 * nt + 2 * tig + h] : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                x[b][h] = in ? a.part[((at * S::NTT + nt) * OM + k2 + h) * 32 + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        take(st, x);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        s_v[warp][h][lane] = v[h];
        if (gid == 0) s_stat[warp][h][tig] = make_float4(M[h], L[h], Mo[h], 0.0f);
    }
    __syncthreads();
    if (warp != 0) return;
    static_assert(W == B, "the warps' sums are one batch");
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) st[b][h] = s_stat[b][h][tig], x[b][h] = s_v[b][h][lane];
#pragma unroll
    for (int h = 0; h < 2; ++h) M[h] = Mo[h] = -INFINITY, L[h] = 0.0f, v[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    take(st, x);
    write_out<S>(a, item.z, item.w, item.y, nt, k2, v[0], v[1], row_factor(M[0], L[0], Mo[0]), row_factor(M[1], L[1], Mo[1]));
    if (k2 == 0 && gid == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) write_lse<S>(a, item.z, item.w, item.y, 8 * nt + 2 * tig + h, M[h], L[h]);
}

}  // namespace gcu
