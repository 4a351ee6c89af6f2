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
// One or more warps to a row, each on its own (no barrier): a head vector is 8 values to a lane, so a warp's turn is 1, 2 or
// 4 vectors of one kind (queries, keys, values), and a lane has the same dims of every head of its row, so that the norm's
// weights and the rotary cosines and sines stay in registers. The 8 are 4 neighbours and the 4 that these rotate with
// (8 neighbours where nothing rotates), so a rotation needs no other lane. The turns' rows come through a ring in
// shared memory, the first of them asked for before anything else; then the row's sequence is found (one round of loads
// over up to 256 row_start entries), its length and page read and the angles taken. Angles are position * inv_freq in 64
// bits (at position 10^6 a 32-bit angle is off by 0.03), reduced to a turn there. Queries and keys for a 16-bit cache go
// through float; keys for the int8 cache through double up to the rounding to float, so that their codes are those of the
// definition (a float rounding moves one code in about 10^5).
//
// What bounds it: for few rows the chain row -> sequence -> length -> page -> angle (8 us for one row, 16 us for 1280 rows of
// 16/2 heads of 256 to int8, 3.0 TB/s); for prompts instruction issue (9645 bf16 rows of 32/8 heads of 128: 56 us, 4.2 TB/s;
// 6151 f16 rows to int8: 47 us, 2.6 TB/s). One CTA per row with barriers between those steps: 24, 90 and 90 us.
struct AppendArgs {
    gcuda_paged_kv kv;
    gcuda_paged_batch b;
    gcuda_append_rows x;
    int warps;                       // of a row
    bool vec_q, vec_k, vec_v, vec_o; // loads and stores of these rows by 4 values
    uint32_t *status;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendAhead = 4;   // turns whose copies to shared memory are in flight
// (float rows of 256, every dimension rotated by an odd half: ring, angles and staging)
constexpr int kAppendMaxShared = kAppendThreads * kAppendAhead * 32 + kAppendWarps * 128 * 16 + kAppendThreads * 8 * 8;

__device__ __forceinline__ float max_nan(float a, float b) {   // (a NaN among the values stays one)
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The nearest integers to 127 y / top, the even one of two, as bytes: by a float product where that is sure (it is within
// 10^-4 of the quotient; added to 1.5 * 2^23 its low bits are the integer), next to a half by comparing 2 * 127 |y| with
// (2 k + 1) top, both exact in double. Rows of values so small that 127 / top has no float (below 2^-121) are scaled by a
// power of two first, which is exact: y is theirs afterwards.
__device__ __forceinline__ uint2 codes_of(float (&y)[8], float top) {
    if (top < 0x1p-100f) {
        top *= 0x1p100f;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= 0x1p100f;
    }
    const float inv = top > 0.0f ? 127.0f / top : 0.0f;
    uint32_t w[2] = {0, 0}, near = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = __fmul_rn(y[i], inv), m = __fadd_rn(c, kBiasF);
        if (fabsf(c - __fsub_rn(m, kBiasF)) > 0.499f) near |= 1u << i;
        w[i / 4] |= (__float_as_uint(m) & 0xffu) << (8 * (i % 4));
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (near >> i & 1) {
                const double k = floor(static_cast<double>(__fmul_rn(fabsf(y[i]), inv)));
                const double a = 254.0 * static_cast<double>(fabsf(y[i])), h = (2.0 * k + 1.0) * static_cast<double>(top);
                const int n = static_cast<int>(k), r = a > h ? n + 1 : a < h ? n : n + (n & 1);
                w[i / 4] = (w[i / 4] & ~(0xffu << (8 * (i % 4)))) | static_cast<uint32_t>((y[i] < 0.0f ? -r : r) & 0xff) << (8 * (i % 4));
            }
    }
    return make_uint2(w[0], w[1]);
}

// 1 / sqrt(mean x^2 + eps) of a vector of HD, 8 values to a lane
template <int HD>
__device__ __forceinline__ float head_factor(const float (&v)[8], float eps) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrtf(ss * (1.0f / HD) + eps);
}
template <int HD>
__device__ __forceinline__ double head_factor(const double (&v)[8], double eps) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(v[i], v[i], ss);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrt(ss * (1.0 / HD) + eps);
}

// Rotation where half is no multiple of 4: through st, a vector's HD values of shared memory; a lane's values lie at `at`
template <typename T, typename T2>
__device__ __forceinline__ void rotate_odd(T (&v)[8], int at, int half, const T2 *trig, T *st) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) st[at + i] = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = at + i;
        if (d < half) v[i] = v[i] * T(trig[d].x) - st[d + half] * T(trig[d].y);
        else if (d < 2 * half) v[i] = v[i] * T(trig[d - half].x) + st[d - half] * T(trig[d - half].y);
    }
}

// The last sequence s with row_start[s] <= row (a warp's lanes alike), -1: none. Rounds of 32 probes while more than 256
// are left, then all of these.
__device__ __forceinline__ int find_sequence(const gcuda_paged_batch &b, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.n_seq;   // the answer is among [lo, lo + n), or there is none
    while (n > 256) {
        const int gap = (n + 31) / 32, s = lo + lane * gap;
        const uint32_t le = __ballot_sync(0xffffffffu, lane * gap < n && b.row_start[min(s, b.n_seq)] <= row);
        const int k = le ? 31 - __clz(le) : 0;
        n = min(gap, n - k * gap);
        lo += k * gap;
    }
    int found = -1;
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lane + 32 * i < n ? b.row_start[lo + lane + 32 * i] : 0x7fffffff;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t le = __ballot_sync(0xffffffffu, v[i] <= row);
        if (le) found = lo + 32 * i + 31 - __clz(le);
    }
    return found;
}

template <int HD, typename TA, int CACHE>
__global__ void __launch_bounds__(kAppendThreads, 4) k_paged_append(AppendArgs a) {
    constexpr int LV = HD / 8, VW = 32 / LV;   // lanes of a vector, vectors of a turn
    constexpr bool I8 = CACHE == GCUDA_I8;
    using Trig = std::conditional_t<I8, double2, float2>;
    using Wide = std::conditional_t<I8, double, float>;
    extern __shared__ __align__(16) uint8_t append_sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LV, j = lane % LV;
    const int64_t work = static_cast<int64_t>(blockIdx.x) * kAppendWarps + warp;
    const int row = static_cast<int>(work / a.warps), first = static_cast<int>(work % a.warps);
    const int nh = a.x.n_heads, nkv = a.kv.n_kv_heads, half = a.x.rope_dim / 2;
    const int tq = (nh + VW - 1) / VW, tk = (nkv + VW - 1) / VW, turns = tq + 2 * tk;
    if (row >= a.b.n_rows) return;
    // the lane's dims: at[0] .. + 3 and at[1] .. + 3, which rotate with each other on the first half / 4 lanes
    const bool paired = half % 4 == 0, rotates = paired && j < half / 4;
    const int at0 = !paired ? 8 * j : rotates ? 4 * j : 8 * j, at1 = rotates ? half + 4 * j : at0 + 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    constexpr int CB = 4 * sizeof(TA);   // bytes of 4 values
    struct __align__(16) Raw {
        TA v[8];
    };
    Raw *ring = reinterpret_cast<Raw *>(append_sm) + (warp * kAppendAhead) * 32 + lane;   // [turn][lane]: a lane's own
    const TA *src_q = static_cast<const TA *>(a.x.q) + row * a.x.q_stride, *src_k = static_cast<const TA *>(a.x.k) + row * a.x.k_stride,
             *src_v = static_cast<const TA *>(a.x.v) + row * a.x.v_stride;
    auto fetch = [&](int turn, int slot) {
        if (turn < turns) {
            const TA *src;
            bool vec, in;
            if (turn < tq) {
                const int h = turn * VW + sub;
                in = h < nh, vec = a.vec_q;
                src = src_q + h * a.x.q_head_stride;
            } else {
                const bool k = turn < tq + tk;
                const int h = (turn - (k ? tq : tq + tk)) * VW + sub;
                in = h < nkv, vec = k ? a.vec_k : a.vec_v;
                src = (k ? src_k : src_v) + h * HD;
            }
            Raw *dst = ring + slot * 32;
            if (!in) {
                *dst = Raw{};
            } else if (vec) {
                if constexpr (CB == 16) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst->v)), "l"(src + at0) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst->v + 4)), "l"(src + at1) : "memory");
                } else {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst->v)), "l"(src + at0) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst->v + 4)), "l"(src + at1) : "memory");
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) dst->v[i] = src[at0 + i], dst->v[4 + i] = src[at1 + i];
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kAppendAhead - 1; ++i) fetch(first + i * a.warps, i);

    // the row's place
    const int seq = find_sequence(a.b, row);
    int pos = -1, page = -1;
    if (seq >= 0) {
        const SeqRows q = seq_rows(a.b, a.kv.page_size, seq, a.status);
        if (row - q.r0 < q.rows) {
            pos = q.length - q.rows + (row - q.r0);
            if (pos >= 0) page = a.b.pages[seq * a.b.pages_stride + pos / a.kv.page_size];
            if ((page < 0 || page >= a.kv.n_pages) && lane == 0) atomicOr(a.status, kErrBadShape);
        }
    }
    const bool stored = page >= 0 && page < a.kv.n_pages;
    const int in_page = pos >= 0 ? pos % a.kv.page_size : 0;
    Trig *trig = reinterpret_cast<Trig *>(append_sm + kAppendWarps * kAppendAhead * 32 * sizeof(Raw)) + warp * half;
    Wide *st = reinterpret_cast<Wide *>(append_sm + kAppendWarps * (kAppendAhead * 32 * sizeof(Raw) + half * sizeof(Trig))) + (warp * VW + sub) * HD;   // (odd halves only)
    for (int i = lane; i < half && pos >= 0; i += 32) {
        const double angle = static_cast<double>(pos) * static_cast<double>(a.x.inv_freq[i]);
        if constexpr (I8) {
            double sn, cs;
            sincos(angle, &sn, &cs);
            trig[i] = make_double2(cs, sn);
        } else {
            const double t = angle * 0.15915494309189534;   // in turns
            float sn, cs;
            sincospif(2.0f * static_cast<float>(t - rint(t)), &sn, &cs);
            trig[i] = make_float2(cs, sn);
        }
    }
    __syncwarp();
    if (pos < 0) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        return;
    }
    // queries: lo' = lo A - hi B, hi' = hi C + lo D with the norm's weights in the factors
    float fa[4], fb[4], fc[4], fd[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Trig t = rotates ? trig[4 * j + i] : Trig{1, 0};
        const float c = static_cast<float>(t.x), n = static_cast<float>(t.y);
        const float wl = a.x.q_norm ? 1.0f + a.x.q_norm[at0 + i] : 1.0f, wh = a.x.q_norm ? 1.0f + a.x.q_norm[at1 + i] : 1.0f;
        fa[i] = wl * c, fb[i] = wh * n, fc[i] = wh * c, fd[i] = wl * n;
    }
    // keys: the norm, then the rotation, in T
    auto key = [&](auto (&v)[8]) {
        using T = std::remove_reference_t<decltype(v[0])>;
        if (a.x.k_norm) {
            const T f = head_factor<HD>(v, static_cast<T>(a.x.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * f * (T(1) + static_cast<T>(a.x.k_norm[(i < 4 ? at0 : at1 - 4) + i]));
        }
        if (rotates)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T c = static_cast<T>(trig[4 * j + i].x), n = static_cast<T>(trig[4 * j + i].y), lo = v[i], hi = v[4 + i];
                v[i] = lo * c - hi * n;
                v[4 + i] = hi * c + lo * n;
            }
        if (!paired) rotate_odd<T>(v, at0, half, trig, reinterpret_cast<T *>(st));
    };
    // a lane's 8 values as two groups of 4 (dst: the vector's start)
    auto put = [&](auto *dst, const auto (&y)[8], bool vec) {
        using Group = std::conditional_t<sizeof(y[0]) == 4, uint4, std::conditional_t<sizeof(y[0]) == 2, uint2, uint32_t>>;
        if (vec) {
            *reinterpret_cast<Group *>(dst + at0) = *reinterpret_cast<const Group *>(y);
            *reinterpret_cast<Group *>(dst + at1) = *reinterpret_cast<const Group *>(y + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[at0 + i] = y[i], dst[at1 + i] = y[4 + i];
        }
    };
    const int64_t place = stored ? page * a.kv.page_stride + in_page * a.kv.pos_stride : 0;
    const int64_t place_s = stored ? page * a.kv.scale_page_stride + in_page * a.kv.scale_pos_stride : 0;
    TA *out = static_cast<TA *>(a.x.q_out) + row * a.x.q_out_stride;
    int slot = 0;
#pragma unroll 1
    for (int turn = first; turn < turns; turn += a.warps) {
        fetch(turn + (kAppendAhead - 1) * a.warps, slot == 0 ? kAppendAhead - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAppendAhead - 1) : "memory");   // (a lane reads what it copied)
        float v[8];
        {
            const Raw r = ring[slot * 32];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float(r.v[i]);
        }
        slot = slot + 1 == kAppendAhead ? 0 : slot + 1;
        if (turn < tq) {
            const int h = turn * VW + sub;
            const float f = a.x.q_norm ? head_factor<HD>(v, a.x.eps) : 1.0f;
            alignas(16) TA y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = v[i], hi = v[4 + i];
                v[i] = f * (rotates ? fmaf(lo, fa[i], -(hi * fb[i])) : lo * fa[i]);   // (an infinity stays one where nothing rotates)
                v[4 + i] = f * (rotates ? fmaf(hi, fc[i], lo * fd[i]) : hi * fc[i]);
            }
            if (!paired) rotate_odd<float>(v, at0, half, trig, reinterpret_cast<float *>(st));
            if (h >= nh) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = from_float<TA>(v[i]);
            put(out + h * HD, y, a.vec_o);
            continue;
        }
        if (!stored) continue;
        const bool is_k = turn < tq + tk;
        const int h = (turn - (is_k ? tq : tq + tk)) * VW + sub;
        if (is_k) {
            if constexpr (I8) {
                double y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = v[i];
                key(y);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(y[i]);
            } else {
                key(v);
            }
        }
        const int64_t to = place + h * a.kv.head_stride;
        void *base = is_k ? a.kv.k : a.kv.v;
        if constexpr (I8) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
#pragma unroll
            for (int o = LV / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (h >= nkv) continue;
            const uint2 codes = codes_of(v, top);
            *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(base) + to + at0) = codes.x;
            *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(base) + to + at1) = codes.y;
            if (lane % LV == 0)
                (is_k ? a.kv.k_scale : a.kv.v_scale)[place_s + h * a.kv.scale_head_stride] =
                    static_cast<float>(static_cast<double>(top) / 127.0);
        } else {
            using TC = std::conditional_t<CACHE == GCUDA_BF16, __nv_bfloat16, __half>;
            if (h >= nkv) continue;
            alignas(16) TC y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = from_float<TC>(v[i]);
            put(static_cast<TC *>(base) + to, y, true);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace gcu
