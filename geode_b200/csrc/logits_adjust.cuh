// logits_adjust.cuh - penalties, biases and grammar masks on the logits of many sequences' rows.
#pragma once

#include "paged.cuh"

namespace gcu {

struct AdjustArgs {
    gcuda_logit_rules r;
    const void *in;
    void *out;
    int S, k, V, slice, slices;
    int64_t in_stride, out_stride;
    uint32_t *status;
};

constexpr int kAdjustThreads = 256;

// One CTA per (sequence, slice of the vocabulary): the slice's token counts and last bias entries are gathered once in
// shared memory (integers: the order of the atomics does not matter) for all k+1 rows; draft i-1 is counted in front of
// row i. Then one pass over each row's slice.
template <typename T>
__global__ void __launch_bounds__(kAdjustThreads) k_logits_adjust(AdjustArgs a) {
    extern __shared__ int adjust_sm[];
    int *count = adjust_sm, *entry = adjust_sm + a.slice;   // occurrences, 1 + the last bias entry
    const int tid = threadIdx.x, s = blockIdx.x / a.slices, v0 = (blockIdx.x % a.slices) * a.slice;
    const int nv = min(a.slice, a.V - v0), rows = a.k + 1;
    const gcuda_logit_rules &r = a.r;
    for (int i = tid; i < 2 * a.slice; i += kAdjustThreads) adjust_sm[i] = 0;
    __syncthreads();
    auto checked = [&](int n, int64_t most) {
        if (n >= 0 && n <= most) return n;
        if (tid == 0) atomicOr(a.status, kErrBadShape);
        return n < 0 ? 0 : static_cast<int>(most);
    };
    if (r.history) {
        const int n = checked(r.history_len[s], r.history_stride);
        for (int i = tid; i < n; i += kAdjustThreads) {
            const int t = r.history[s * r.history_stride + i];
            if (t >= a.V) atomicOr(a.status, kErrBadToken);
            else if (t >= v0 && t - v0 < nv) atomicAdd(&count[t - v0], 1);
        }
    }
    if (r.bias_id) {
        const int n = checked(r.bias_len[s], r.bias_stride);
        for (int i = tid; i < n; i += kAdjustThreads) {
            const int t = r.bias_id[s * r.bias_stride + i];
            if (t >= a.V) atomicOr(a.status, kErrBadToken);
            else if (t >= v0 && t - v0 < nv) atomicMax(&entry[t - v0], i + 1);
        }
    }
    const float rep = r.repetition ? r.repetition[s] : 1.0f, fr = r.frequency ? r.frequency[s] : 0.0f,
                pr = r.presence ? r.presence[s] : 0.0f;
    for (int i = 0; i < rows; ++i) {
        __syncthreads();
        if (i > 0 && r.drafts && tid == 0) {
            const int t = r.drafts[static_cast<int64_t>(s) * a.k + i - 1];
            if (t >= a.V) atomicOr(a.status, kErrBadToken);
            else if (t >= v0 && t - v0 < nv) ++count[t - v0];
        }
        __syncthreads();
        const int64_t row = static_cast<int64_t>(s) * rows + i;
        const uint32_t *mask = nullptr;
        if (r.mask) {
            const int64_t m = r.mask_row ? r.mask_row[row] : row;
            if (m >= r.n_masks) {
                if (tid == 0) atomicOr(a.status, kErrBadShape);
            } else if (m >= 0) {
                mask = r.mask + m * r.mask_stride;
            }
        }
        const T *in = static_cast<const T *>(a.in) + row * a.in_stride + v0;
        T *out = static_cast<T *>(a.out) + row * a.out_stride + v0;
        for (int j = tid; j < nv; j += kAdjustThreads) {
            float x = to_float(in[j]);
            if (entry[j]) x = __fadd_rn(x, r.bias[s * r.bias_stride + entry[j] - 1]);
            if (const int c = count[j]) {
                x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                x = __fsub_rn(__fsub_rn(x, __fmul_rn(fr, static_cast<float>(c))), pr);
            }
            if (mask && !((mask[(v0 + j) >> 5] >> ((v0 + j) & 31)) & 1u)) x = -INFINITY;
            out[j] = from_float<T>(x);
        }
    }
}

}  // namespace gcu
