// paged.cuh - a step's rows over a paged KV cache: what the append and attention kernels share (value types, the
// plan's checks on the device, addresses of a position's rows), and the append kernel.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/geode_cuda.h"
#include "common.cuh"

namespace gcu {

// ---------------------------------------------------------------------------------------------- value types ----
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// ---------------------------------------------------------------------------------------------- the plan ----
// Sequence s of the step as the device finds it: its rows [r0, r0 + rows) and its cache's length. A sequence whose
// rows or length are out of range has rows 0 (left out) and raises the status word.
struct SeqRows {
    int r0, rows, length;
};
__device__ __forceinline__ SeqRows seq_rows(const gcuda_paged_batch &b, int page_size, int s, uint32_t *status) {
    SeqRows q{b.row_start[s], 0, b.length[s]};
    const int r1 = b.row_start[s + 1];
    if (q.r0 < 0 || r1 < q.r0 || r1 > b.n_rows || r1 - q.r0 > b.max_rows || q.length < 0 ||
        q.length > static_cast<int64_t>(b.max_pages) * page_size) {
        atomicOr(status, kErrBadShape);
        q.length = 0;
        return q;
    }
    q.rows = r1 - q.r0;
    return q;
}

// ---------------------------------------------------------------------------------------------- append ----
// One CTA per row: the row's sequence is found by all threads at once (row_start is read in one round of loads, no
// search down a tree), the rotary cosines and sines of its position are taken once for all heads, then a warp per head
// vector. Angles are position * inv_freq in 64 bits (at position 10^6 a 32-bit angle is off by 0.03). Queries and keys
// for a 16-bit cache go through float; keys for the int8 cache through double up to the rounding to float, so that
// their codes are those of the definition (a float rounding moves one code in about 10^5).
struct AppendArgs {
    gcuda_paged_kv kv;
    gcuda_paged_batch b;
    gcuda_append_rows x;
    uint32_t *status;
};

constexpr int kAppendThreads = 256;

__device__ __forceinline__ float max_nan(float a, float b) {   // (a NaN among the values stays one)
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Norm (w: NULL off) and rotation of the HD values a warp holds (lane + 32 i), through its staging row st.
template <int HD, typename T>
__device__ __forceinline__ void norm_rotate(T (&v)[HD / 32], const float *w, float eps, int half, const double2 *trig, T *st) {
    const int lane = threadIdx.x & 31;
    if (w) {
        T ss = 0;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) ss += v[i] * v[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T inv = T(1) / sqrt(ss / T(HD) + T(eps));
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) v[i] = v[i] * inv * (T(1) + T(w[lane + 32 * i]));
    }
    if (half == 0) return;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) st[lane + 32 * i] = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const int d = lane + 32 * i;
        if (d < half) v[i] = v[i] * T(trig[d].x) - st[d + half] * T(trig[d].y);
        else if (d < 2 * half) v[i] = v[i] * T(trig[d - half].x) + st[d - half] * T(trig[d - half].y);
    }
    __syncwarp();
}

template <int HD, typename TA, int CACHE>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(AppendArgs a) {
    __shared__ double2 trig[HD / 2];
    __shared__ double stage[kAppendThreads / 32][HD];
    __shared__ int s_seq;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    for (int s = tid; s < a.b.n_seq; s += kAppendThreads)
        if (a.b.row_start[s] <= row && row < a.b.row_start[s + 1]) atomicMax(&s_seq, s);
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) return;
    const SeqRows q = seq_rows(a.b, a.kv.page_size, seq, a.status);
    if (row - q.r0 >= q.rows) return;
    const int pos = q.length - q.rows + (row - q.r0);
    if (pos < 0) {
        if (tid == 0) atomicOr(a.status, kErrBadShape);
        return;
    }
    const int half = a.x.rope_dim / 2;
    for (int i = tid; i < half; i += kAppendThreads) {
        double sn, cs;
        sincos(static_cast<double>(pos) * static_cast<double>(a.x.inv_freq[i]), &sn, &cs);
        trig[i] = make_double2(cs, sn);
    }
    const int page = a.b.pages[seq * a.b.pages_stride + pos / a.kv.page_size];
    const bool stored = page >= 0 && page < a.kv.n_pages;
    if (!stored && tid == 0) atomicOr(a.status, kErrBadShape);
    __syncthreads();
    const int nh = a.x.n_heads, nkv = a.kv.n_kv_heads, in_page = pos % a.kv.page_size;
    for (int item = warp; item < nh + 2 * nkv; item += kAppendThreads / 32) {
        if (item < nh) {
            const TA *src = static_cast<const TA *>(a.x.q) + row * a.x.q_stride + item * a.x.q_head_stride;
            TA *dst = static_cast<TA *>(a.x.q_out) + row * a.x.q_out_stride + item * HD;
            float v[HD / 32];
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) v[i] = to_float(src[lane + 32 * i]);
            norm_rotate<HD, float>(v, a.x.q_norm, a.x.eps, half, trig, reinterpret_cast<float *>(stage[warp]));
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) dst[lane + 32 * i] = from_float<TA>(v[i]);
            continue;
        }
        if (!stored) continue;
        const bool is_k = item < nh + nkv;
        const int h = is_k ? item - nh : item - nh - nkv;
        const TA *src = is_k ? static_cast<const TA *>(a.x.k) + row * a.x.k_stride + h * HD
                             : static_cast<const TA *>(a.x.v) + row * a.x.v_stride + h * HD;
        float v[HD / 32];
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) v[i] = to_float(src[lane + 32 * i]);
        if (is_k) {
            if constexpr (CACHE == GCUDA_I8) {
                double d[HD / 32];
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) d[i] = v[i];
                norm_rotate<HD, double>(d, a.x.k_norm, a.x.eps, half, trig, stage[warp]);
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) v[i] = static_cast<float>(d[i]);
            } else {
                norm_rotate<HD, float>(v, a.x.k_norm, a.x.eps, half, trig, reinterpret_cast<float *>(stage[warp]));
            }
        }
        const int64_t at = page * a.kv.page_stride + in_page * a.kv.pos_stride + h * a.kv.head_stride;
        void *base = is_k ? a.kv.k : a.kv.v;
        if constexpr (CACHE == GCUDA_I8) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) top = max_nan(top, fabsf(v[i]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            int8_t *dst = static_cast<int8_t *>(base) + at;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
                dst[lane + 32 * i] = top > 0.0f ? static_cast<int8_t>(__double2int_rn(static_cast<double>(v[i]) * 127.0 / static_cast<double>(top)))
                                                : static_cast<int8_t>(0);
            if (lane == 0)
                (is_k ? a.kv.k_scale : a.kv.v_scale)[page * a.kv.scale_page_stride + in_page * a.kv.scale_pos_stride +
                                                     h * a.kv.scale_head_stride] =
                    static_cast<float>(static_cast<double>(top) / 127.0);
        } else {
            using TC = std::conditional_t<CACHE == GCUDA_BF16, __nv_bfloat16, __half>;
            TC *dst = static_cast<TC *>(base) + at;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) dst[lane + 32 * i] = from_float<TC>(v[i]);
        }
    }
}

}  // namespace gcu
