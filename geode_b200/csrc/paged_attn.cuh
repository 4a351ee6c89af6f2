// paged_attn.cuh - attention of each sequence's newest rows over its pages.
#pragma once

#include "paged.cuh"

namespace gcu {

struct PagedAttnArgs {
    gcuda_paged_kv kv;
    gcuda_paged_batch b;
    gcuda_attn_rows x;
    uint32_t *status;
};

constexpr int kPagedAttnThreads = 128;

// One CTA per (row, head), its warps' positions interleaved; a lane holds dims lane + 32 i. Running maximum and sum
// per warp, joined at the end.
template <int HD, typename TA, int CACHE>
__global__ void __launch_bounds__(kPagedAttnThreads) k_paged_attn(PagedAttnArgs a) {
    constexpr int W = kPagedAttnThreads / 32, N = HD / 32;
    __shared__ int s_seq;
    __shared__ float s_o[W][HD], s_m[W], s_l[W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x, head = blockIdx.y;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    for (int s = tid; s < a.b.n_seq; s += kPagedAttnThreads)
        if (a.b.row_start[s] <= row && row < a.b.row_start[s + 1]) atomicMax(&s_seq, s);
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) return;
    const SeqRows r = seq_rows(a.b, a.kv.page_size, seq, a.status);
    if (row - r.r0 >= r.rows) return;
    const int end = r.length - r.rows + (row - r.r0) + 1;   // the row sees [begin, end)
    const int begin = a.x.window > 0 ? max(0, end - a.x.window) : 0;
    const int kh = head / (a.x.n_heads / a.kv.n_kv_heads);
    float q[N], o[N], m = -INFINITY, l = 0.0f;
    const TA *src = static_cast<const TA *>(a.x.q) + row * a.x.q_stride + head * a.x.q_head_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = to_float(src[lane + 32 * i]), o[i] = 0.0f;
    for (int p = begin + warp; p < end; p += W) {
        const int page = a.b.pages[seq * a.b.pages_stride + p / a.kv.page_size];
        if (page < 0 || page >= a.kv.n_pages) {
            if (lane == 0) atomicOr(a.status, kErrBadShape);
            continue;
        }
        const int ip = p % a.kv.page_size;
        const int64_t at = page * a.kv.page_stride + ip * a.kv.pos_stride + kh * a.kv.head_stride;
        float ks = 1.0f, vs = 1.0f, k[N], v[N];
        if constexpr (CACHE == GCUDA_I8) {
            const int64_t sa = page * a.kv.scale_page_stride + ip * a.kv.scale_pos_stride + kh * a.kv.scale_head_stride;
            ks = a.kv.k_scale[sa];
            vs = a.kv.v_scale[sa];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                k[i] = static_cast<const int8_t *>(a.kv.k)[at + lane + 32 * i];
                v[i] = static_cast<const int8_t *>(a.kv.v)[at + lane + 32 * i];
            }
        } else {
            using TC = std::conditional_t<CACHE == GCUDA_BF16, __nv_bfloat16, __half>;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                k[i] = to_float(static_cast<const TC *>(a.kv.k)[at + lane + 32 * i]);
                v[i] = to_float(static_cast<const TC *>(a.kv.v)[at + lane + 32 * i]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
        s = warp_sum(s) * ks * a.x.scale;
        const float mn = fmaxf(m, s);
        const float f = m == -INFINITY ? 0.0f : expf(m - mn), e = s == -INFINITY ? 0.0f : expf(s - mn);
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * f + e * vs * v[i];
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s_o[warp][lane + 32 * i] = o[i];
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    __syncthreads();
    float M = -INFINITY, Lsum = 0.0f;
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_m[w]);
    float f[W];
    for (int w = 0; w < W; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.0f : expf(s_m[w] - M);
        Lsum += s_l[w] * f[w];
    }
    TA *dst = static_cast<TA *>(a.x.out) + row * a.x.out_stride + head * HD;
    for (int d = tid; d < HD; d += kPagedAttnThreads) {
        float acc = 0.0f;
        for (int w = 0; w < W; ++w) acc += s_o[w][d] * f[w];
        dst[d] = from_float<TA>(Lsum > 0.0f ? acc / Lsum : Lsum == 0.0f ? 0.0f : Lsum);
    }
    if (tid == 0 && a.x.lse) a.x.lse[static_cast<int64_t>(row) * a.x.n_heads + head] = Lsum == 0.0f ? -INFINITY : M + logf(Lsum);
}

}  // namespace gcu
