// paged_attn.cuh - attention of each sequence's newest rows over its pages (flash decoding over a paged cache).
//
// An item is one (sequence, key head, block of query rows): the sequence's T rows times the G query heads that share the key
// head, R = T * G rows in blocks of 8 (k_paged_attn), 16 or 40 (k_paged_attn_rows, paged_attn_rows.cuh). Items are cut into
// tiles of positions and the tiles of all items, laid end to end with a few tiles' time for each item's beginning, are dealt
// out evenly to two CTAs an SM (each finds its share by a scan over the lengths on the device: whatever the lengths, every
// CTA has the same work). What a CTA holds of an item that it does not finish goes to the scratch and k_paged_attn_join adds
// the parts up. The copies run ahead of the products across tiles and items alike, so memory is not left idle while an item
// ends and the next begins.
//
// Both products run on the tensor cores (mma.sync, float sums) with the cache as the 16-row operand and the query rows as the
// 8-column one, so that one token's few rows fill the instruction: S^T = K Q^T, then O^T = V^T P^T. K's fragments come by
// ldmatrix as they lie; V's by rows, positions interleaved by byte permutation (the order of dims in O^T is free): no staging
// of transposed or widened rows. int8 keys are multiplied as they are (m16n8k32, integer sums); int8 values are widened to
// f16 in registers (exact).
//
// Arithmetic: over an int8 cache a query row is its largest value times (65536 a + 256 b + c) / (127 * 65536) with int8 a, b,
// c: every value to 2^-24 of the row's largest, each sum of products exact. Over a 16-bit cache queries are in the cache's
// type (f16, and floats in any: scaled by a power of two per row); float activations, and f16 ones over bf16, are held as a sum
// of such numbers: two f16 (22 bits) or three bf16 (24 bits; two would leave an error of 4e-6, three times a float product's).
// Weights are held in two numbers of the product's 16-bit type, f16 over int8 (three bf16 for float activations over bf16): one
// would add as much error as rounding the output to that type does, and turn one in eleven of bf16 outputs over int8 to the
// neighbouring number (two: one in a thousand; the second number costs 2% there, up to 9% where the products weigh).
// int8 rows' value scales go into the weight's exponent: w = 2^(s + log2 vs - m'), with a maximum m' of its own, so that
// rows of any scale keep their bits. Scores, sums, maxima and outputs are float.
//
// Measured, main kernel and join (8 query rows a key head): 64 ragged conversations of up to 8192 positions over an int8
// cache of 2 heads of 256 (278 MB) 62 us, each further 278 MB 40 us (7 TB/s); 2 x 131072 positions of bf16 73 us (5.2
// TB/s); 128 of up to 1000 in f16, 8 heads of 128, 69 us (items of four tiles: their beginnings and ends); one conversation
// of 8192 positions 16 us (latency: the scan and the first copies 4.7, a tile 2.5, the join 5).
#pragma once

#include <utility>

#include "paged.cuh"
#include "paged_attn_plan.hpp"

namespace gcu {

struct PagedAttnArgs {
    gcuda_paged_kv kv;
    gcuda_paged_batch b;
    gcuda_attn_rows x;
    uint32_t *status;
    uint32_t page_mul;   // p / page_size = (p * page_mul) >> page_shift for p < 2^31
    int page_shift;
    int4 *cut;       // [grid] the item that CTA c began and did not finish: {2 parts + the slot of c's own, item, first row, rows}
    float4 *stats;   // [grid][2][kRows] {m, l, m', -} of each row
    float4 *part;    // [grid][2][n tile][m tile][lane]
};

constexpr int kPagedAttnThreads = 128;
// The maximum that a row's weights are relative to follows the true one only when that is kSlack (in bits) above it: with
// many rows some maximum grows in nearly every tile, and following each costs a reduction and a rescaling of the outputs
// (32 verify batches of 5 rows: 125 us with every growth followed). f16 weights start at up to 2^kWeightBias, so they
// reach 2^14 at most, and the smallest kept is 2^-30 of the largest.
constexpr float kSlack = 8.0f, kWeightBias = 6.0f;

// What the kernels' shapes share. NT: n tiles (8 query rows each) of an item; ES, RB: bytes of a value, of a row
template <int HD_, int CACHE_, bool SPLIT_, int NT_>
struct PagedBase {
    static constexpr int HD = HD_, CACHE = CACHE_, NT = NT_, kRows = 8 * NT;
    static constexpr bool SPLIT = SPLIT_, I8 = CACHE == GCUDA_I8, BF16 = CACHE == GCUDA_BF16;
    static constexpr int ES = I8 ? 1 : 2, RB = HD * ES, OM = HD / 16;
    static constexpr bool THREE = SPLIT && BF16;                 // floats as three numbers
    static constexpr int PN = THREE ? 3 : 2;                     // numbers of a weight
    // the queries' fragments: int8 three digits a value in k steps of 32 dims, else one to three numbers in k steps of 16
    static constexpr int kQ = I8 ? HD / 32 * NT * 32 * 24 : HD / 16 * NT * 32 * 8 * (THREE ? 3 : SPLIT ? 2 : 1);
    static constexpr int kQTwo = I8 ? HD / 32 * NT * 32 * 16 : THREE ? HD / 16 * NT * 32 * 16 : 0;   // (where the third ones start)
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
__device__ __forceinline__ void mma_s8_16832(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 65536 a + 256 b + c of sums that were made on top of kBiasBits
__device__ __forceinline__ float digits_sum(int32_t a, int32_t b, int32_t c) {
    return fmaf(fmaf(unbias(a), 256.0f, unbias(b)), 256.0f, unbias(c));
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
// N neighbouring values (2, 4 or 8); wide loads where they are aligned
template <int N>
__device__ __forceinline__ void load_act(float (&v)[N], const void *p, int type, int64_t i) {
    if (type == GCUDA_F32) {
        const float *f = static_cast<const float *>(p) + i;
        if constexpr (N >= 4) {
            if ((reinterpret_cast<uintptr_t>(f) & 15) == 0) {
#pragma unroll
                for (int k = 0; k < N; k += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(f + k);
                    v[k] = x.x, v[k + 1] = x.y, v[k + 2] = x.z, v[k + 3] = x.w;
                }
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = f[k];
        return;
    }
    const uint16_t *h = static_cast<const uint16_t *>(p) + i;
    uint32_t w[N / 2];
    if ((reinterpret_cast<uintptr_t>(h) & (2 * N - 1)) == 0) {
        if constexpr (N == 8) {
            const uint4 x = *reinterpret_cast<const uint4 *>(h);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else if constexpr (N == 4) {
            const uint2 x = *reinterpret_cast<const uint2 *>(h);
            w[0] = x.x, w[1] = x.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t *>(h);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 2) w[k / 2] = h[k] | static_cast<uint32_t>(h[k + 1]) << 16;
    }
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const float2 x = type == GCUDA_BF16 ? unpack2<true>(w[k / 2]) : unpack2<false>(w[k / 2]);
        v[k] = x.x, v[k + 1] = x.y;
    }
}
__device__ __forceinline__ void store_act2(void *p, int type, int64_t i, float x, float y) {
    if (type == GCUDA_F32) static_cast<float *>(p)[i] = x, static_cast<float *>(p)[i + 1] = y;
    else if (type == GCUDA_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x), static_cast<__nv_bfloat16 *>(p)[i + 1] = __float2bfloat16_rn(y);
    else static_cast<__half *>(p)[i] = __float2half_rn(x), static_cast<__half *>(p)[i + 1] = __float2half_rn(y);
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

// One row block's finished values of m tiles m, m + 1 (mostly four neighbouring dims) of the rows 2 tig, 2 tig + 1 of an n
// tile
template <typename S>
__device__ __forceinline__ void write_out(const PagedAttnArgs &a, int r0, int rows, int item, int nt, int m, const float4 &x,
                                          const float4 &y, float inv0, float inv1) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = rows * G, nrb = (R + S::kRows - 1) / S::kRows;
    const int kh = item / nrb, rb = item % nrb, d = S::dim(m, gid), d2 = S::dim(m + 1, gid);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int r = rb * S::kRows + 8 * nt + 2 * tig + c;
        if (r >= R) continue;
        const float inv = c ? inv1 : inv0;
        const int64_t at = static_cast<int64_t>(r0 + r / G) * a.x.out_stride + static_cast<int64_t>(kh * G + r % G) * S::HD;
        const float4 v = c ? make_float4(x.y * inv, x.w * inv, y.y * inv, y.w * inv) : make_float4(x.x * inv, x.z * inv, y.x * inv, y.z * inv);
        if (d2 == d + 2) {
            store_act4(a.x.out, a.x.type, at + d, v);
        } else {
            store_act2(a.x.out, a.x.type, at + d, v.x, v.y);
            store_act2(a.x.out, a.x.type, at + d2, v.z, v.w);
        }
    }
}
// the same of one m tile (two dims)
template <typename S>
__device__ __forceinline__ void write_one(const PagedAttnArgs &a, int r0, int rows, int item, int nt, int m, const float4 &x,
                                          float inv0, float inv1) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = rows * G, nrb = (R + S::kRows - 1) / S::kRows;
    const int kh = item / nrb, rb = item % nrb;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int r = rb * S::kRows + 8 * nt + 2 * tig + c;
        if (r >= R) continue;
        const int64_t at = static_cast<int64_t>(r0 + r / G) * a.x.out_stride + static_cast<int64_t>(kh * G + r % G) * S::HD + S::dim(m, gid);
        store_act2(a.x.out, a.x.type, at, c ? x.y * inv1 : x.x * inv0, c ? x.w * inv1 : x.z * inv0);
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

// a / b of numbers >= 0: in 32 bits where they fit (a 64-bit division takes some 400 cycles, and four of them stand between
// a CTA's start and its first copy)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// The positions [lo, hi) that a sequence's rows see between them, and its tiles a (key head, row block)
template <typename S>
__device__ __forceinline__ int seq_tiles(const PagedAttnArgs &a, const SeqRows &q, int &lo) {
    lo = a.x.window > 0 ? max(0, q.length - q.rows + 1 - a.x.window) : 0;
    return max(1, (q.length - lo + S::CT - 1) / S::CT);
}
// a sequence's share of the work: for each of its items the beginning's cost and the tiles
template <typename S>
__device__ __forceinline__ int64_t seq_cost(const PagedAttnArgs &a, const SeqRows &q) {
    if (q.rows == 0) return 0;
    int lo;
    const int64_t t = S::kItemCost + seq_tiles<S>(a, q, lo);
    return t * a.kv.n_kv_heads * ((q.rows * (a.x.n_heads / a.kv.n_kv_heads) + S::kRows - 1) / S::kRows);
}

// f(kind) for the kinds first, first + 1, ..
template <int first = 0, typename F, int... e>
__device__ __forceinline__ void for_kinds(F &&f, std::integer_sequence<int, e...>) {
    (f(std::integral_constant<int, first + e>{}), ...);
}

struct PagedSegment {   // what a CTA does of one item (48 bytes)
    int r0, rows, length;
    int lo, tps;        // the item's first position and tiles
    int item, t0, n;    // the item within its sequence; this CTA's tiles
    int parts;          // the CTAs that share the item, where it begins here and ends elsewhere (else 0)
    int no;             // how many segments came before it in this CTA
    int kh, rb;         // its key head, its block of rows
};

// A CTA's share of the work and the way through it. A warp walks for itself (all alike): look() gives the next tile and
// the page of this lane's position in it; the segments it opens wait in shared memory until the products reach them, and
// so does what only the opening of the next one needs (it would cost the products some thirty registers). The following
// sequence's plan is loaded a sequence ahead.
struct PagedTile {
    int page;    // of this lane's position (-2: it has none)
    int in_page; // its place there
    int p0;      // the warp's first position in the tile (-1: no tile)
    int kh;
};
struct PagedWalkShared {
    int64_t sum[4], base;
    int seq;
    struct Warp {
        int64_t total, ctas, u, end, base;
        SeqRows sq, sq_next;
        int seq;
    } warp[4];
};

template <typename S>
struct PagedWalk {
    const PagedAttnArgs &a;
    PagedWalkShared &sh;
    PagedSegment *segs;      // this warp's [kSegs]
    const int *pages;        // the segment being looked up: its pages,
    int p0, n, length, kh;   // next tile's position for this warp, tiles left
    int opened;
    bool more;               // work is left behind that segment

    __device__ __forceinline__ SeqRows load(int s) const {
        return s < a.b.n_seq ? seq_rows(a.b, a.kv.page_size, s, a.status) : SeqRows{0, 0, 0};
    }
    // This CTA's share [u, end) of all work: each thread sums a run of sequences, then a scan over the threads. False:
    // nothing for this CTA.
    __device__ __forceinline__ bool start() {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
        const int run = (a.b.n_seq + kPagedAttnThreads - 1) / kPagedAttnThreads;
        const int s_lo = min(tid * run, a.b.n_seq), s_hi = min(s_lo + run, a.b.n_seq);
        int64_t mine = 0;
        for (int s = s_lo; s < s_hi; ++s) mine += seq_cost<S>(a, load(s));
        int64_t before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) sh.sum[warp] = before;
        __syncthreads();
        before -= mine;
        int64_t total = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < warp) before += sh.sum[w];
            total += sh.sum[w];
        }
        const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
        if (cta >= ctas) return false;
        const int64_t u = quotient(total * cta, ctas);
        if (before <= u && u < before + mine) {
            int64_t b = before;
            int s = s_lo;
            for (; s < s_hi; ++s) {
                const int64_t c = seq_cost<S>(a, load(s));
                if (u < b + c) break;
                b += c;
            }
            sh.seq = s;
            sh.base = b;
        }
        __syncthreads();
        if (lane == 0) sh.warp[warp] = {total, ctas, u, quotient(total * (cta + 1), ctas), sh.base, load(sh.seq), load(sh.seq + 1), sh.seq};
        __syncwarp();
        n = opened = 0;
        more = true;
        return true;
    }
    __device__ __forceinline__ void open() {   // the next segment with tiles (none left: n 0)
        const int G = a.x.n_heads / a.kv.n_kv_heads, warp = threadIdx.x >> 5;
        PagedWalkShared::Warp w = sh.warp[warp];
        while (n == 0 && w.u < w.end) {
            if (w.sq.rows > 0) {
                PagedSegment g;
                g.r0 = w.sq.r0, g.rows = w.sq.rows, g.length = w.sq.length;
                g.tps = seq_tiles<S>(a, w.sq, g.lo);
                const int nrb = (g.rows * G + S::kRows - 1) / S::kRows, per = S::kItemCost + g.tps;
                const int64_t off = w.u - w.base;
                g.item = static_cast<int>(quotient(off, per));
                const int o = static_cast<int>(off - static_cast<int64_t>(g.item) * per), m = static_cast<int>(min(static_cast<int64_t>(per - o), w.end - w.u));
                g.t0 = max(0, o - S::kItemCost);
                g.n = max(0, o + m - S::kItemCost) - g.t0;
                // (the CTA that holds the item's last tile, by the shares' own division)
                g.parts = g.t0 == 0 && g.n < g.tps ? static_cast<int>(quotient((w.u - o + per) * w.ctas - 1, w.total)) - static_cast<int>(blockIdx.x) + 1 : 0;
                g.no = opened;
                g.kh = g.item / nrb;
                g.rb = g.item % nrb;
                if (g.n > 0) {
                    n = g.n;
                    p0 = g.lo + g.t0 * S::CT + warp * S::TP;
                    length = g.length;
                    kh = g.kh;
                    pages = a.b.pages + w.seq * a.b.pages_stride;
                    if ((threadIdx.x & 31) == 0) segs[opened % S::kSegs] = g;
                    ++opened;
                }
                w.u += m;
                if (w.u - w.base < static_cast<int64_t>(per) * a.kv.n_kv_heads * nrb) continue;
                w.base = w.u;
            }
            ++w.seq;
            w.sq = w.sq_next;
            w.sq_next = load(w.seq + 1);
        }
        more = w.u < w.end;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) sh.warp[warp] = w;
        __syncwarp();
    }
    __device__ __forceinline__ PagedTile look() {
        if (n == 0) {
            if (!more) return PagedTile{-2, 0, -1, 0};
            open();
            if (n == 0) return PagedTile{-2, 0, -1, 0};
        }
        const int lane = threadIdx.x & 31, p = p0 + lane, k = static_cast<int>((static_cast<uint64_t>(p) * a.page_mul) >> a.page_shift);
        PagedTile t{-2, p - k * a.kv.page_size, p0, kh};
        if (lane < S::TP && p < length) t.page = pages[k];
        p0 += S::CT;
        --n;
        return t;
    }
};

// Where the 16-byte pieces of a tile's rows lie in shared memory: rows of RE bytes, a row's pieces swapped so that the
// fragment loads of K (8 rows x one piece) and of V (every second row x 2 pieces) meet no bank twice. A warp's k-th copy
// takes PR rows; its place is the first one's, some bits of it flipped (flip), and k times PR rows on.
template <int RE, bool V>
struct PagedPieces {
    static constexpr int CH = RE / 16, PR = 32 / CH;   // pieces of a row; rows of a copy
    static __host__ __device__ constexpr int turn(int p) {
        return V ? (RE == 64 ? (p >> 1 & 1) << 1 : (p >> 1 & 3) << 1) : (RE == 64 ? p >> 1 & 3 : p & 7);
    }
    static __device__ __forceinline__ uint32_t first(int lane) { return lane / CH * RE + (lane % CH ^ turn(lane / CH)) * 16; }
    static __host__ __device__ constexpr uint32_t flip(int k) { return turn(k * PR) << 4; }   // (the lane's own row bits are in first())
};
// K's fragments of 16 positions (rows of RE bytes at `rows`) and one k step (32 bytes of each): a0 .. a3
template <int RE>
struct KeyFragments {
    uint32_t at;   // this lane's row and piece of k step 0
    __device__ __forceinline__ explicit KeyFragments(const uint8_t *rows) {
        const int lane = threadIdx.x & 31, p = (lane & 7) + (lane & 8);
        at = smem_addr(rows) + p * RE + ((lane >> 4) ^ PagedPieces<RE, false>::turn(p)) * 16;
    }
    __device__ __forceinline__ uint4 operator()(int ks) const {   // (a row starts on a multiple of its size: the step's bits flip)
        uint4 r;
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at ^ (ks << 5)) : "memory");
        return r;
    }
};
// The copies of N * PR rows (16-byte aligned to 256 bytes of shared memory at dst) of one page, or of any pages: `place`
// the value offset of lane p's row (rows first_p ..), ok a bit for each that is there.
template <int RE, bool V, int N, int ES>
__device__ __forceinline__ void copy_rows(uint32_t dst, const uint8_t *src, int64_t pos_stride, int64_t place, uint32_t ok, bool one_page, int first_p) {
    using P = PagedPieces<RE, V>;
    const int lane = threadIdx.x & 31, rl = lane / P::CH, c = lane % P::CH;
    const uint32_t to = dst + P::first(lane);
    if (one_page) {
        const int64_t step = pos_stride * ES;
        const uint8_t *from = src + __shfl_sync(0xffffffffu, place, first_p) * ES + rl * step + c * 16;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            copy16((to ^ P::flip(k)) + k * P::PR * RE, from, 16);
            from += step * P::PR;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int p = first_p + k * P::PR + rl;
        const int64_t x = __shfl_sync(0xffffffffu, place, p);
        copy16((to ^ P::flip(k)) + k * P::PR * RE, src + x * ES + c * 16, (ok >> p & 1) ? 16 : 0);
    }
}

// The segment's queries as fragments (b0, b1) [k step][n tile][lane] and the rows' column factors: warp w takes rows w,
// w + 4, ..; a lane HD / 32 neighbouring dims; up to five rows' loads in flight.
template <typename S>
__device__ __forceinline__ void build_queries(const PagedAttnArgs &a, const PagedSegment &g, uint8_t *sm_q, float *col) {
    constexpr bool I8 = S::I8, BF16 = S::BF16, SPLIT = S::SPLIT;
    constexpr int HD = S::HD, N = HD / 32, B = S::kRows / 4 < 5 ? S::kRows / 4 : 5;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.x.n_heads / a.kv.n_kv_heads, R = g.rows * G;
    uint2 *q_one = reinterpret_cast<uint2 *>(sm_q + S::kQTwo);   // (the third numbers, or the only ones)
    uint4 *q_two = reinterpret_cast<uint4 *>(sm_q);              // two numbers a value (SPLIT, and int8's first digits)
    for (int i0 = warp; i0 < S::kRows; i0 += 4 * B) {
        float vs[B][N];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int r = g.rb * S::kRows + i0 + 4 * b;
#pragma unroll
            for (int k = 0; k < N; ++k) vs[b][k] = 0.0f;
            if (r < R) load_act(vs[b], a.x.q, a.x.type, static_cast<int64_t>(g.r0 + r / G) * a.x.q_stride + static_cast<int64_t>(g.kh * G + r % G) * a.x.q_head_stride + lane * N);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int i = i0 + 4 * b;
            float (&v)[N] = vs[b], top = 0.0f;
            const int nt = i >> 3, row = i & 7;
            if constexpr (I8) {
#pragma unroll
                for (int k = 0; k < N; ++k) top = max_nan(top, fabsf(v[k]));
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, x));
                // (the nearest integer n to 127 * 65536 v / top; the bytes of n + 0x808080, their top bits flipped, are its
                // signed digits. Rows so small that the quotient or the factor has no normal float: times a power of two)
                float down = 1.0f;
                if (top < 0x1p-60f) {
                    top *= 0x1p60f;
                    down = 0x1p-60f;
#pragma unroll
                    for (int k = 0; k < N; ++k) v[k] *= 0x1p60f;
                }
                const float inv = top > 0.0f ? 8323072.0f / top : 0.0f;
                if (lane == 0) col[i] = a.x.scale * 1.44269504088896341f * down * (top * (1.0f / 8323072.0f));
                uint32_t n[N];
#pragma unroll
                for (int k = 0; k < N; ++k) n[k] = static_cast<uint32_t>(__float2int_rn(v[k] * inv)) + 0x808080u;
                constexpr int W = N < 4 ? N : 4;   // neighbouring dims stored together
#pragma unroll
                for (int k = 0; k < N; k += W) {
                    const int d = lane * N + k, ks = d / 32, t = d % 16 / 4, half = d % 32 / 16, f = (ks * S::NT + nt) * 32 + row * 4 + t;
                    uint32_t *const at3[3] = {reinterpret_cast<uint32_t *>(q_two + f) + half, reinterpret_cast<uint32_t *>(q_two + f) + 2 + half,
                                              reinterpret_cast<uint32_t *>(q_one + f) + half};
#pragma unroll
                    for (int y = 0; y < 3; ++y) {
                        const uint32_t byte = 2 - y, pick = byte | (byte + 4) << 4;
                        const uint32_t lo = __byte_perm(n[k], n[k + 1], pick);
                        if constexpr (W == 4) *at3[y] = __byte_perm(lo, __byte_perm(n[k + 2], n[k + 3], pick), 0x5410) ^ 0x80808080u;
                        else reinterpret_cast<uint16_t *>(at3[y])[d % 4 / 2] = static_cast<uint16_t>(lo ^ 0x8080u);
                    }
                }
            } else {
                int ex = 0;
                if constexpr (!BF16 || SPLIT) {   // (bf16 queries over bf16 keep their bits as they are)
#pragma unroll
                    for (int k = 0; k < N; ++k) top = fmaxf(top, fabsf(v[k]));
                    top = warp_max(top);
                    // 2^-ex brings the largest to [1, 2); zeros, infinities: as they are
                    ex = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
#pragma unroll
                    for (int k = 0; k < N; ++k) v[k] = scalbnf(v[k], -ex);
                }
                if (lane == 0) col[i] = scalbnf(a.x.scale * 1.44269504088896341f, ex);
#pragma unroll
                for (int k = 0; k < N; k += 2) {
                    const int d = lane * N + k, ks = d / 16, t = d % 8 / 2, half = d % 16 / 8;
                    const int f = (ks * S::NT + nt) * 32 + row * 4 + t;
                    const uint32_t hi = pack2<BF16>(v[k], v[k + 1]);
                    if constexpr (SPLIT) {
                        const float2 h = unpack2<BF16>(hi);
                        reinterpret_cast<uint32_t *>(q_two + f)[half] = hi;
                        const float x = v[k] - h.x, y = v[k + 1] - h.y;
                        const uint32_t mid = pack2<BF16>(x, y);
                        reinterpret_cast<uint32_t *>(q_two + f)[2 + half] = mid;
                        if constexpr (S::THREE) {
                            const float2 m = unpack2<BF16>(mid);
                            reinterpret_cast<uint32_t *>(q_one + f)[half] = pack2<BF16>(x - m.x, y - m.y);
                        }
                    } else {
                        reinterpret_cast<uint32_t *>(q_one + f)[half] = hi;
                    }
                }
            }
        }
    }
}

// Shapes of k_paged_attn: 8 query rows, each warp with positions of its own. An entry of the ring is K's or V's rows of ME m
// tiles (16 positions each), at most 256 bytes of a row; a tile is EPO entries of K, then as many of V.
template <int HD_, int CACHE_, bool SPLIT_>
struct PagedShape : PagedBase<HD_, CACHE_, SPLIT_, 1> {
    using B = PagedBase<HD_, CACHE_, SPLIT_, 1>;
    using B::RB, B::I8, B::OM, B::ES, B::kRows;
    static constexpr int RE = RB < 256 ? RB : 256, PARTS = RB / RE;
    static constexpr int MT = 2, TP = 16 * MT;                    // m tiles, positions of a warp's tile
    static constexpr int ME = RB < 256 ? 2 : 1, EM = MT / ME, EPO = EM * PARTS;
    static constexpr int CT = 4 * TP;                             // positions of a CTA's tile
    // an item's beginning and end cost about what 128 KB of rows do (5 us; with half of it the CTAs with two items finish
    // 2.4 us after those with one)
    static constexpr int kItemCost = 131072 / (2 * CT * RB) > 0 ? 131072 / (2 * CT * RB) : 1;
    static constexpr int kEntry = 16 * ME * RE;
    static constexpr int kRing = 16 * 1024;                       // bytes of a warp's ring
    static constexpr int E = kRing / kEntry < 12 ? kRing / kEntry : 12;
    static constexpr int TS = E / (2 * EPO) + 2;                  // tiles whose scales and valid bits are kept
    static constexpr int kScale = (I8 ? 2 * TP * 4 : 0) + 16;
    static constexpr int kSegs = E / (2 * EPO) + 5;               // segments looked up, not yet done
    static constexpr int o_ring = 0, o_q = o_ring + 4 * E * kEntry, o_scale = o_q + B::kQ;
    static constexpr int o_col = o_scale + 4 * TS * kScale;       // [kRows] column factor
    static constexpr int o_seg = o_col + kRows * 4;               // [warp][kSegs]
    static constexpr int o_stat = o_seg + 4 * kSegs * 48;         // [warp][kRows] m, l, m'
    static constexpr int o_join = o_stat + 4 * kRows * 16;        // [warp][m tile][lane] O
    static constexpr int kSmem = o_join + 4 * OM * 32 * 16;
    static_assert(E >= 3, "two entries in flight");
    // the dims of m tile m's rows gid and gid + 8 (the first of the two neighbours): a lane's 8th of a row is taken in
    // pieces of at most 16 bytes, 8 pieces side by side
    static __device__ __forceinline__ int dim(int m, int gid) {
        constexpr int PB = RB / 8 < 16 ? RB / 8 : 16, DPP = PB / ES;
        return 2 * m / DPP * 8 * DPP + gid * DPP + 2 * m % DPP;
    }
};

// Eight query rows or fewer: each of the four warps takes positions of its own, keeps a running maximum, sum and output
// over them and meets the others only at an item's end.
template <typename S>
__global__ void __launch_bounds__(kPagedAttnThreads, 2) k_paged_attn(PagedAttnArgs a) {
    constexpr int NT = 1, TP = S::TP, MT = S::MT, RE = S::RE, E = S::E, OM = S::OM, PARTS = S::PARTS, ME = S::ME, EPO = S::EPO;
    constexpr bool I8 = S::I8, BF16 = S::BF16, SPLIT = S::SPLIT;
    extern __shared__ __align__(1024) uint8_t sm[];   // (a row of the ring starts on a multiple of its size)
    __shared__ PagedWalkShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.x.n_heads / a.kv.n_kv_heads, cta = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) a.cut[cta] = make_int4(0, 0, 0, 0);
    PagedWalk<S> walk{a, sh, reinterpret_cast<PagedSegment *>(sm + S::o_seg) + warp * S::kSegs};
    if (!walk.start()) return;

    // the queries' fragments (b0, b1) [k step][n tile][lane]; two numbers a value (SPLIT, and int8's a, b): uint4
    uint2 *q_one = reinterpret_cast<uint2 *>(sm + S::o_q + S::kQTwo);   // (int8: c)
    uint4 *q_two = reinterpret_cast<uint4 *>(sm + S::o_q);
    float *col_s = reinterpret_cast<float *>(sm + S::o_col);
    uint8_t *ring = sm + S::o_ring + warp * E * S::kEntry;
    uint8_t *scales = sm + S::o_scale + warp * S::TS * S::kScale;
    const uint32_t ring_a = smem_addr(ring), scales_a = smem_addr(scales);

    PagedTile ahead0 = walk.look(), ahead1 = walk.look();

    // ---- the copies: entry by entry through the tiles looked up. The kind of an entry (0 .. EPO-1: K's, then V's) is known
    // where it is issued: it follows from the kind that is waited for there.
    int in_slot = 0, in_tile = 0;   // the ring slot; the tile's place among the scales
    bool in_any = true, one_page = false;
    int64_t place = 0;    // value offset of this lane's position
    uint32_t ok = 0;      // the tile's positions that are on a page
    auto issue = [&](auto kind_) {
        constexpr int kind = decltype(kind_)::value % (2 * EPO);
        if (kind == 0 && in_any) {
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
                // positions one after the other on one page: their rows are pos_stride apart
                one_page = ok == 0xffffffffu && __shfl_sync(0xffffffffu, t.in_page, 0) + TP <= a.kv.page_size;
                const uint32_t d = scales_a + in_tile * S::kScale;
                if (lane == 0) *reinterpret_cast<uint32_t *>(scales + in_tile * S::kScale) = ok;
                if constexpr (I8) {
                    const int64_t sp = there ? t.page * a.kv.scale_page_stride + t.in_page * a.kv.scale_pos_stride + t.kh * a.kv.scale_head_stride : 0;
                    copy4(d + 16 + lane * 4, a.kv.k_scale + sp, there ? 4 : 0);
                    copy4(d + 16 + (TP + lane) * 4, a.kv.v_scale + sp, there ? 4 : 0);
                }
            }
        }
        if (in_any) {
            constexpr bool is_v = kind >= EPO;
            constexpr int first_p = kind % EPO / PARTS * 16 * ME, part = kind % PARTS;
            const uint8_t *src = static_cast<const uint8_t *>(is_v ? a.kv.v : a.kv.k) + part * RE;
            copy_rows<RE, is_v, 16 * ME * (RE / 16) / 32, S::ES>(ring_a + in_slot * S::kEntry, src, a.kv.pos_stride, place, ok, one_page, first_p);
        }
        in_slot = in_slot + 1 == E ? 0 : in_slot + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    in_tile = S::TS - 1;
    for_kinds(issue, std::make_integer_sequence<int, E - 1>{});
    __syncwarp();   // (the first segments are written)

    int slot = 0, tile_at = 0;   // the products' place in the ring and among the scales
    auto next_entry = [&](auto kind_) {   // the entry at `slot`, of this kind, has landed; the one before it is free for a copy
        asm volatile("cp.async.wait_group %0;" ::"n"(E - 2) : "memory");
        __syncwarp();
        issue(std::integral_constant<int, decltype(kind_)::value + E - 1>{});
        const uint8_t *ent = ring + slot * S::kEntry;
        slot = slot + 1 == E ? 0 : slot + 1;
        return ent;
    };

    for (int done = 0; done < walk.opened; ++done) {
        const PagedSegment g = walk.segs[done % S::kSegs];
        const int R = g.rows * G;
        build_queries<S>(a, g, sm + S::o_q, col_s);
        __syncthreads();

        // ---- this lane's columns: rows 2 tig, 2 tig + 1 of each of the warp's n tiles
        float col[NT][2], m[NT][2], mo[NT][2], l[NT][2];
        int lim[NT][2];   // the last position that the row sees (-1: none, or no such row)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int i = 8 * nt + 2 * tig + c, r = g.rb * S::kRows + i;
                col[nt][c] = col_s[i];
                lim[nt][c] = r < R ? g.length - g.rows + r / G : -1;
                m[nt][c] = mo[nt][c] = -INFINITY;
                l[nt][c] = 0.0f;
            }
        // rows of this block: all see [all_lo, all_hi]
        const int t_first = g.rb * S::kRows / G, t_last = (min(R, (g.rb + 1) * S::kRows) - 1) / G;
        const int all_hi = g.length - g.rows + t_first;
        const int all_lo = a.x.window > 0 ? g.length - g.rows + t_last + 1 - a.x.window : 0;
        float o[OM][NT][4];
#pragma unroll
        for (int k = 0; k < OM; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[k][nt][c] = 0.0f;

        for (int i = 0; i < g.n; ++i) {
            const int p0 = g.lo + (g.t0 + i) * S::CT + warp * TP;
            constexpr int PN = S::PN;
            uint32_t pw[PN][MT][NT][2];   // the weights as fragments (b0, b1), and what is left of them
            bool edge;
            {
                // ---- S^T = K Q^T
                float s[MT][NT][4];
                auto k_entry = [&](auto kind_) {
                    constexpr int kind = decltype(kind_)::value, m0 = kind / PARTS * ME;
                    [[maybe_unused]] constexpr int part = kind % PARTS;
                    const uint8_t *ent = next_entry(kind_);
                    auto keys = [&](int mt, int ks) { return KeyFragments<RE>(ent + 16 * mt * RE)(ks); };
                    if constexpr (I8) {
                        // sums on top of 1.5 * 2^23, whose float neighbours are the integers: |sum| <= 127^2 HD < 2^22
                        int32_t acc[ME][NT][3][4];
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int y = 0; y < 3; ++y)
#pragma unroll
                                    for (int c = 0; c < 4; ++c) acc[mt][nt][y][c] = static_cast<int32_t>(kBiasBits);
#pragma unroll
                        for (int ks = 0; ks < RE / 32; ++ks)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const int f = (ks * NT + nt) * 32 + lane;
                                const uint4 ab = q_two[f];
                                const uint2 cc = q_one[f];
#pragma unroll
                                for (int mt = 0; mt < ME; ++mt) {
                                    const uint4 k = keys(mt, ks);
                                    mma_s8_16832(acc[mt][nt][0], k.x, k.y, k.z, k.w, ab.x, ab.y);
                                    mma_s8_16832(acc[mt][nt][1], k.x, k.y, k.z, k.w, ab.z, ab.w);
                                    mma_s8_16832(acc[mt][nt][2], k.x, k.y, k.z, k.w, cc.x, cc.y);
                                }
                            }
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c) s[m0 + mt][nt][c] = digits_sum(acc[mt][nt][0][c], acc[mt][nt][1][c], acc[mt][nt][2][c]);
                    } else {
                        float hi[ME][NT][4], lo[ME][NT][4];
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c) hi[mt][nt][c] = part ? s[m0 + mt][nt][c] : 0.0f, lo[mt][nt][c] = 0.0f;
#pragma unroll
                        for (int ks = 0; ks < RE / 32; ++ks)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const int f = ((part * (RE / 32) + ks) * NT + nt) * 32 + lane;
                                const uint4 b2 = SPLIT ? q_two[f] : make_uint4(0, 0, 0, 0);
                                const uint2 b = SPLIT ? make_uint2(b2.x, b2.y) : q_one[f];
#pragma unroll
                                for (int mt = 0; mt < ME; ++mt) {
                                    const uint4 k = keys(mt, ks);
                                    mma_16816<BF16>(hi[mt][nt], k.x, k.y, k.z, k.w, b.x, b.y);
                                    if constexpr (SPLIT) mma_16816<BF16>(lo[mt][nt], k.x, k.y, k.z, k.w, b2.z, b2.w);
                                    if constexpr (S::THREE) mma_16816<BF16>(lo[mt][nt], k.x, k.y, k.z, k.w, q_one[f].x, q_one[f].y);
                                }
                            }
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c) s[m0 + mt][nt][c] = SPLIT ? hi[mt][nt][c] + lo[mt][nt][c] : hi[mt][nt][c];
                    }
                };
                for_kinds(k_entry, std::make_integer_sequence<int, EPO>{});
                // ---- scores in bits, masks, running maxima
                const uint8_t *sc = scales + tile_at * S::kScale;
                tile_at = tile_at + 1 == S::TS ? 0 : tile_at + 1;
                const uint32_t bits = *reinterpret_cast<const uint32_t *>(sc);
                const float *sv = reinterpret_cast<const float *>(sc + 16);
                edge = p0 < all_lo || p0 + TP - 1 > all_hi;
                const bool masked = edge || bits != 0xffffffffu;
                // int8: lv = log2 vs. An unseen scale may be anything: -inf + lv is then no number, which the maxima pass over;
                // the weight of such a score (a bit of hidden) is set to 0
                float lv[MT][2];
                uint32_t hidden = 0;
                bool strange = false;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int p = 16 * mt + 8 * h + gid;
                        float ks = 1.0f;
                        lv[mt][h] = 0.0f;
                        if constexpr (I8) {
                            ks = sv[p];
                            lv[mt][h] = lg2(sv[TP + p]);
                            strange = strange || !(lv[mt][h] < INFINITY);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float &v = s[mt][nt][2 * h + c];
                                v *= col[nt][c] * ks;
                                if (masked) {
                                    const int gp = p0 + p;
                                    if (gp > lim[nt][c] || !(bits >> p & 1) || (a.x.window > 0 && gp <= lim[nt][c] - a.x.window)) {
                                        v = -INFINITY;
                                        hidden |= 1u << ((mt * NT + nt) * 4 + 2 * h + c);
                                    }
                                }
                            }
                    }
                strange = I8 && masked && __any_sync(0xffffffffu, strange);
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
                                if constexpr (I8) topo[c] = fmaxf(topo[c], s[mt][nt][2 * h + c] + lv[mt][h]);
                            }
                    // (far seldom: the reduction over the positions' lanes and the rescaling only then)
                    const bool grows = top[0] > m[nt][0] + kSlack || top[1] > m[nt][1] + kSlack ||
                                       (I8 && (topo[0] > mo[nt][0] + (kWeightBias + kSlack) || topo[1] > mo[nt][1] + (kWeightBias + kSlack)));
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
                                w[x] = ex2(s[mt][nt][x] + lv[mt][x >> 1] - oz);
                                if (strange && (hidden >> ((mt * NT + nt) * 4 + x) & 1)) w[x] = 0.0f;
                            } else {
                                w[x] = ex2(s[mt][nt][x] - oz);
                                l[nt][c] += BF16 ? w[x] : w[x] * 0.015625f;   // 2^-kWeightBias
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float x = w[2 * h], y = w[2 * h + 1];
#pragma unroll
                            for (int n = 0; n < PN; ++n) {
                                const uint32_t part = pack2<BF16>(x, y);
                                pw[n][mt][nt][h] = move_trans(part);
                                const float2 b = unpack2<BF16>(part);
                                x -= b.x, y -= b.y;
                            }
                        }
                    }
                }
            }
            // ---- O^T += V^T P^T
            auto v_entry = [&](auto kind_) {
                constexpr int m0 = (decltype(kind_)::value - EPO) / PARTS * ME, part = decltype(kind_)::value % PARTS;
                const uint8_t *ent = next_entry(kind_);
                constexpr int PB = RE / 8 < 16 ? RE / 8 : 16, NP = RE / 8 / PB, NW = PB / 4;
                constexpr int MW = I8 ? 2 : 1;   // m tiles of a word
                auto v_words = [&](int mt, int np, uint32_t (&x)[4][NW]) {   // positions 2 tig, + 1, + 8, + 9
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int p = 16 * mt + 2 * tig + (k & 1) + 8 * (k >> 1);
                        const uint8_t *row = ent + p * RE;
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
                // a row must not be touched by values that it does not see, and zero times an infinity is not zero: at
                // the edges of what the rows see a 16-bit tile that holds such values goes a token at a time (the same
                // sums in the same order: bit for bit what finite values there give)
                bool apart = false;
                if constexpr (!I8) {
                    if (edge && g.rows > 1) {
                        bool odd = false;
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt)
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
                    for (int mt = 0; mt < ME; ++mt)
#pragma unroll
                        for (int np = 0; np < NP; ++np) {
                            uint32_t x[4][NW];
                            v_words(mt, np, x);
#pragma unroll
                            for (int w = 0; w < NW; ++w) {
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
                                for (int n = 0; n < PN; ++n)
#pragma unroll
                                    for (int k = 0; k < MW; ++k) {
                                        const int om = ((part * NP + np) * NW + w) * MW + k;
#pragma unroll
                                        for (int nt = 0; nt < NT; ++nt) {
                                            mma_16816<BF16>(o[om][nt], va[k][0], va[k][1], va[k][2], va[k][3], pw[n][m0 + mt][nt][0], pw[n][m0 + mt][nt][1]);
                                        }
                                    }
                            }
                        }
                } else if constexpr (!I8) {
                    for (int t = 0; t < g.rows; ++t) {
                        const int hi_p = g.length - g.rows + t - p0, lo_p = a.x.window > 0 ? hi_p - a.x.window + 1 : -(1 << 30);
#pragma unroll
                        for (int mt = 0; mt < ME; ++mt) {
                            uint32_t keep[2];   // the halves of positions 2 tig, 2 tig + 1 (and + 8) that token t sees
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int p = 16 * (m0 + mt) + 2 * tig + 8 * h;
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
                                        float d[4];
#pragma unroll
                                        for (int x4 = 0; x4 < 4; ++x4) d[x4] = o[(part * NP + np) * NW + w][nt][x4];
#pragma unroll
                                        for (int n = 0; n < PN; ++n)
                                            mma_16816<BF16>(d, va[0], va[1], va[2], va[3], pw[n][m0 + mt][nt][0], pw[n][m0 + mt][nt][1]);
#pragma unroll
                                        for (int x4 = 0; x4 < 4; ++x4)
                                            if (lim[nt][x4 & 1] - p0 == hi_p && lim[nt][x4 & 1] >= 0) o[(part * NP + np) * NW + w][nt][x4] = d[x4];
                                    }
                                }
                            }
                        }
                    }
                }
            };
            for_kinds<EPO>(v_entry, std::make_integer_sequence<int, EPO>{});
        }
        // a lane summed its positions' weights: the others' of the column are on the lanes with the same tig
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);

        // ---- the segment's end: the position groups joined, then out or to the scratch
        const bool whole = g.t0 == 0 && g.n == g.tps;
        const int keep_slot = 2 * cta + (g.no == 0 ? 0 : 1);
        if (g.parts > 0 && tid == 0) a.cut[cta] = make_int4(2 * g.parts + (keep_slot & 1), g.item, g.r0, g.rows);
        float4 *stat = reinterpret_cast<float4 *>(sm + S::o_stat);
        float4 *buf = reinterpret_cast<float4 *>(sm + S::o_join);   // [group][m tile][lane], an n tile at a time
        if (gid == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) stat[warp * S::kRows + 8 * nt + 2 * tig + c] = make_float4(m[nt][c], l[nt][c], mo[nt][c], 0.0f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0) __syncthreads();
#pragma unroll
            for (int k = 0; k < OM; ++k)
                buf[(warp * OM + k) * 32 + lane] = make_float4(o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]);
            __syncthreads();   // (the queries' fragments are free from here, the buffer after the next barrier)
            float M[2] = {-INFINITY, -INFINITY}, Mo[2] = {-INFINITY, -INFINITY}, Ls[2] = {0.0f, 0.0f}, f[4][2];
            float4 st[4][2];
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    st[w][c] = stat[w * S::kRows + 8 * nt + 2 * tig + c];
                    M[c] = fmaxf(M[c], st[w][c].x);
                    Mo[c] = fmaxf(Mo[c], st[w][c].z);
                }
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    // (a sum of 0: nothing seen. One that is no number stays so, though no maximum came with it)
                    Ls[c] += st[w][c].y == 0.0f ? 0.0f : st[w][c].y * ex2(st[w][c].x - M[c]);
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
                        const float4 x = buf[(w * OM + k + h) * 32 + lane];
                        v[h].x += x.x * f[w][0], v[h].y += x.y * f[w][1], v[h].z += x.z * f[w][0], v[h].w += x.w * f[w][1];
                    }
                }
                if (whole) {
                    write_out<S>(a, g.r0, g.rows, g.item, nt, k, v[0], v[1], inv0, inv1);
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
                    if (whole) write_lse<S>(a, g.r0, g.rows, g.item, i, M[c], Ls[c]);
                    else a.stats[static_cast<int64_t>(keep_slot) * S::kRows + i] = make_float4(M[c], Ls[c], Mo[c], 0.0f);
                }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The parts of each item that was cut, joined: CTA (c, y) has the one that main CTA c began, if there is one - its parts
// are c's last and the first of c + 1, c + 2, .. - and a share of its values, `split` warps to a pair of m tiles of an
// n tile: they take every split-th part, B in flight, and join their sums in shared memory.
constexpr int kJoinThreads = 512;   // (split 1: 256 of them)

template <typename S>
__global__ void __launch_bounds__(kJoinThreads, 1) k_paged_attn_join(PagedAttnArgs a, int split, int grid) {
    constexpr int OM = S::OM;
    __shared__ float4 s_stat[kJoinThreads / 32][2][4], s_v[kJoinThreads / 32][2][32];
    __shared__ uint32_t s_cut[kJoinThreads / 32];
    const int W = blockDim.x / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tig = lane & 3, gid = lane >> 2;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    int c = blockIdx.x;
    if (split > 1) {   // (few items: a CTA for each of them, not for each main CTA)
        int left = blockIdx.x;
        c = -1;
        for (int c0 = 0; c0 < grid && c < 0; c0 += blockDim.x) {
            const uint32_t held = __ballot_sync(0xffffffffu, c0 + tid < grid && a.cut[c0 + tid].x != 0);
            if (lane == 0) s_cut[warp] = held;
            __syncthreads();
            for (int w = 0; w < W && c < 0; ++w) {
                uint32_t bits = s_cut[w];
                const int m = __popc(bits);
                if (left < m) {
                    for (; left > 0; --left) bits &= bits - 1;
                    c = c0 + 32 * w + __ffs(bits) - 1;
                } else {
                    left -= m;
                }
            }
            __syncthreads();
        }
        if (c < 0) return;
    }
    const int4 item = a.cut[c];
    const int n = item.x >> 1, unit = blockIdx.y * (W / split) + warp / split, sub = warp % split;
    if (n == 0) return;
    auto slot = [&](int k) { return static_cast<int64_t>(2 * (c + k) + (k == 0 ? item.x & 1 : 0)); };
    const int nt = unit / (OM / 2), k2 = unit % (OM / 2) * 2;
    const int G = a.x.n_heads / a.kv.n_kv_heads, R = item.w * G, nrb = (R + S::kRows - 1) / S::kRows;
    const bool live = nt < S::NT && item.y % nrb * S::kRows + 8 * nt < R;
    constexpr int B = 4;   // parts whose loads are in flight together
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
                L[h] += st[b][h].y == 0.0f ? 0.0f : st[b][h].y * ex2(st[b][h].x - M[h]);   // (as at a segment's end)
                f[h] = st[b][h].z == -INFINITY ? 0.0f : ex2(st[b][h].z - Mo[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) v[h].x += x[b][h].x * f[0], v[h].y += x[b][h].y * f[1], v[h].z += x[b][h].z * f[0], v[h].w += x[b][h].w * f[1];
        }
    };
    float4 st[B][2], x[B][2];
    for (int k0 = live ? sub : n; k0 < n; k0 += split * B) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const bool in = k0 + b * split < n;
            const int64_t at = slot(in ? k0 + b * split : 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                st[b][h] = in ? a.stats[at * S::kRows + 8 * nt + 2 * tig + h] : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                x[b][h] = in ? a.part[((at * S::NT + nt) * OM + k2 + h) * 32 + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        take(st, x);
    }
    if (split > 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s_v[warp][h][lane] = v[h];
            if (gid == 0) s_stat[warp][h][tig] = make_float4(M[h], L[h], Mo[h], 0.0f);
        }
        __syncthreads();
        if (sub != 0) return;
#pragma unroll
        for (int h = 0; h < 2; ++h) M[h] = Mo[h] = -INFINITY, L[h] = 0.0f, v[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int b0 = 0; b0 < split; b0 += B) {   // (split a multiple of B)
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) st[b][h] = s_stat[warp + b0 + b][h][tig], x[b][h] = s_v[warp + b0 + b][h][lane];
            take(st, x);
        }
    }
    if (!live) return;
    write_out<S>(a, item.z, item.w, item.y, nt, k2, v[0], v[1], row_factor(M[0], L[0], Mo[0]), row_factor(M[1], L[1], Mo[1]));
    if (k2 == 0 && gid == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) write_lse<S>(a, item.z, item.w, item.y, 8 * nt + 2 * tig + h, M[h], L[h]);
}

}  // namespace gcu
