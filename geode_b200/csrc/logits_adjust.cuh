// logits_adjust.cuh - penalties, biases and grammar masks on the logits of many sequences' rows.
//
// Nearly every logit is only copied (or becomes -inf), so the kernel is a copy with a bit per token that says whether a
// rule touches it. One CTA per (sequence, slice of the vocabulary): the sequence's lists are gone through once for all
// its k+1 rows, the tokens of the slice counted in shared memory (integer atomics: their order does not matter, and of
// an id's bias entries the largest index wins). Then each row's slice is one round of 16-byte loads and stores, the next
// row's loads in flight while one is finished, the first row's and the lists' while the counts are cleared.
//
// Measured: 64 x 5 rows of 248320 floats (641 MB) 130 us, 4.9 TB/s: 3904 slices in six to seven turns of four CTAs an SM, each
// with its walk through the lists before the first store; 100 rows of 50257 bf16 (21 MB) 15.6 us, 1300 slices in one and a half
// turns, each a chain lists -> atomics -> row; one row of 248320 floats 7.0 us, the same chain. A value at a time with 8 bytes of
// counts read for each: 449, 25 and 13 us.
#pragma once

#include "paged.cuh"

namespace gcu {

struct AdjustArgs {
    gcuda_logit_rules r;
    const void *in;
    void *out;
    int S, k, V, slices;
    int64_t in_stride, out_stride;
    uint32_t *status;
};

constexpr int kAdjustThreads = 256;

template <typename T, int U>
struct AdjustShape {
    static constexpr int VN = 16 / sizeof(T);                    // logits of a 16-byte load
    static constexpr int slice = U * kAdjustThreads * VN;        // tokens of a CTA: U loads a thread
    static constexpr int words = slice / 32 + 4;                 // (more for fields across a word's end, and whole 16 bytes)
    static constexpr int smem = (words + 2 * slice) * 4;
};

// bits [at, at + n) of a bit array, n <= 8
__device__ __forceinline__ uint32_t bit_field(const uint32_t *w, int at, int n) {
    return __funnelshift_r(w[at >> 5], w[(at >> 5) + 1], at & 31) & ((1u << n) - 1u);
}

template <typename T, int U>
__global__ void __launch_bounds__(kAdjustThreads, U == 2 ? 6 : 4) k_logits_adjust(AdjustArgs a) {
    using P = AdjustShape<T, U>;
    constexpr int VN = P::VN, NT = kAdjustThreads;
    extern __shared__ __align__(16) uint32_t adjust_sm[];
    uint32_t *touched = adjust_sm;                               // a bit per token of the slice
    int *count = reinterpret_cast<int *>(touched + P::words), *entry = count + P::slice;   // occurrences; 1 + the last bias entry
    const int tid = threadIdx.x, s = blockIdx.x / a.slices, v0 = (blockIdx.x % a.slices) * P::slice;
    const int nv = min(P::slice, a.V - v0), rows = a.k + 1;
    const gcuda_logit_rules &r = a.r;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    // a row's slice: a head up to the first 16-byte boundary of both buffers, the body of whole loads, a tail
    struct Row {
        const T *in;
        T *out;
        int head, body;   // tokens of the head; loads of the body
    };
    auto row_at = [&](int i) {
        const int64_t row = static_cast<int64_t>(s) * rows + i;
        Row q{static_cast<const T *>(a.in) + row * a.in_stride + v0, static_cast<T *>(a.out) + row * a.out_stride + v0, nv, 0};
        const uintptr_t x = reinterpret_cast<uintptr_t>(q.in), y = reinterpret_cast<uintptr_t>(q.out);
        if (((x ^ y) & 15) == 0) {   // (else: a value at a time)
            q.head = min(nv, static_cast<int>((16 - (x & 15)) % 16 / sizeof(T)));
            q.body = (nv - q.head) / VN;
        }
        return q;
    };
    constexpr uint32_t kAll = (1u << VN) - 1u;
    auto mask_of = [&](int i) -> int {   // the row's mask (negative: none)
        if (!r.mask || i >= rows) return -1;
        const int64_t at = static_cast<int64_t>(s) * rows + i;
        return r.mask_row ? r.mask_row[at] : static_cast<int>(at);
    };
    auto mask_words = [&](int m) { return m >= 0 && m < r.n_masks ? r.mask + m * r.mask_stride : nullptr; };
    uint4 next[U];
    auto fetch = [&](const Row &q) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (tid + u * NT < q.body) next[u] = __ldcs(reinterpret_cast<const uint4 *>(q.in + q.head) + tid + u * NT);
    };
    Row row = row_at(0);
    fetch(row);
    int mask_next = mask_of(0);   // (a row's mask is looked up a row ahead)
    const float rep = r.repetition ? r.repetition[s] : 1.0f, fr = r.frequency ? r.frequency[s] : 0.0f,
                pr = r.presence ? r.presence[s] : 0.0f;

    auto checked = [&](int n, int64_t most) {
        if (n >= 0 && n <= most) return n;
        if (tid == 0) atomicOr(a.status, kErrBadShape);
        return n < 0 ? 0 : static_cast<int>(most);
    };
    const int nh = r.history ? checked(r.history_len[s], r.history_stride) : 0;
    const int nb = r.bias_id ? checked(r.bias_len[s], r.bias_stride) : 0;
    // the lists' first eight entries a thread, whatever their lengths (another row follows within a stride): one trip to
    // memory. The last row may end with its used entries (columns of a wider array): those only, a second trip.
    const int *hist = r.history + static_cast<int64_t>(s) * r.history_stride, *bid = r.bias_id + static_cast<int64_t>(s) * r.bias_stride;
    auto ahead = [&](const int *list, int64_t stride, int n, int (&t)[8]) {
        const int64_t most = s + 1 < a.S ? stride : n;
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = list && tid + j * NT < most ? list[tid + j * NT] : -1;
    };
    int th[8], tb[8];
    ahead(r.history ? hist : nullptr, r.history_stride, nh, th);
    ahead(r.bias_id ? bid : nullptr, r.bias_stride, nb, tb);
    for (int i = tid; i < P::smem / 16; i += NT) reinterpret_cast<uint4 *>(adjust_sm)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    // f(token in the slice, place in the list)
    auto each = [&](const int *list, int n, int (&t)[8], auto f) {
        for (int i0 = tid; i0 < n; i0 += 8 * NT) {
            if (i0 != tid)
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = i0 + j * NT < n ? list[i0 + j * NT] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i0 + j * NT >= n) continue;
                if (t[j] >= v0 && t[j] - v0 < nv) {
                    atomicOr(&touched[(t[j] - v0) >> 5], 1u << ((t[j] - v0) & 31));
                    f(t[j] - v0, i0 + j * NT);
                } else if (t[j] >= a.V) {
                    atomicOr(a.status, kErrBadToken);
                }
            }
        }
    };
    each(hist, nh, th, [&](int t, int) { atomicAdd(&count[t], 1); });
    each(bid, nb, tb, [&](int t, int i) { atomicMax(&entry[t], i + 1); });
    __syncthreads();

    auto adjusted = [&](float x, int t) {
        if (const int e = entry[t]) x = __fadd_rn(x, r.bias[static_cast<int64_t>(s) * r.bias_stride + e - 1]);
        if (const int c = count[t]) {
            x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            x = __fsub_rn(__fsub_rn(x, __fmul_rn(fr, static_cast<float>(c))), pr);
        }
        return x;
    };
    for (int i = 0; i < rows; ++i) {
        if (i > 0 && r.drafts) {   // draft i - 1 counts from this row on
            const int d = r.drafts[static_cast<int64_t>(s) * a.k + i - 1], t = d - v0;
            if (d >= v0 && t < nv) {
                __syncthreads();
                if (tid == 0) {
                    touched[t >> 5] |= 1u << (t & 31);
                    ++count[t];
                }
                __syncthreads();
            } else if (d >= a.V && tid == 0) {
                atomicOr(a.status, kErrBadToken);
            }
        }
        const uint32_t *mask = mask_words(mask_next);
        if (r.mask && mask_next >= r.n_masks && tid == 0) atomicOr(a.status, kErrBadShape);
        mask_next = mask_of(i + 1);
        const Row q = row;
        uint4 x[U];
        uint32_t allow[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x[u] = next[u];
            allow[u] = kAll;
            const int j = tid + u * NT, t = v0 + q.head + j * VN;
            if (mask && j < q.body) {
                const uint32_t lo = mask[t >> 5], hi = (t & 31) + VN > 32 ? mask[(t >> 5) + 1] : 0u;
                allow[u] = __funnelshift_r(lo, hi, t & 31) & kAll;
            }
        }
        if (i + 1 < rows) {
            row = row_at(i + 1);
            fetch(row);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = tid + u * NT, t = q.head + j * VN;
            if (j >= q.body) continue;
            uint32_t *w = reinterpret_cast<uint32_t *>(&x[u]);
            if (const uint32_t hit = bit_field(touched, t, VN) & allow[u]) {
#pragma unroll
                for (int e = 0; e < VN; ++e)
                    if (hit >> e & 1) {
                        if constexpr (sizeof(T) == 4) {
                            w[e] = __float_as_uint(adjusted(__uint_as_float(w[e]), t + e));
                        } else {
                            const uint16_t b = static_cast<uint16_t>(w[e / 2] >> 16 * (e % 2));
                            const T y = from_float<T>(adjusted(to_float(reinterpret_cast<const T &>(b)), t + e));
                            const uint32_t c = reinterpret_cast<const uint16_t &>(y);
                            w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | c << 16 : (w[e / 2] & 0xffff0000u) | c;
                        }
                    }
            }
            if (allow[u] != kAll) {
#pragma unroll
                for (int e = 0; e < VN; ++e)
                    if (!(allow[u] >> e & 1)) {
                        if constexpr (sizeof(T) == 4) {
                            w[e] = 0xff800000u;
                        } else {
                            const T y = from_float<T>(-INFINITY);
                            const uint32_t c = reinterpret_cast<const uint16_t &>(y);
                            w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | c << 16 : (w[e / 2] & 0xffff0000u) | c;
                        }
                    }
            }
            __stcs(reinterpret_cast<uint4 *>(q.out + q.head) + j, x[u]);
        }
        // head and tail (the whole slice where the buffers' rows are aligned differently)
        const int ends = nv - q.body * VN;
        for (int e = tid; e < ends; e += NT) {
            const int t = e < q.head ? e : e + q.body * VN;
            T y = q.in[t];
            if (touched[t >> 5] >> (t & 31) & 1) y = from_float<T>(adjusted(to_float(y), t));
            if (mask && !(mask[(v0 + t) >> 5] >> ((v0 + t) & 31) & 1)) y = from_float<T>(-INFINITY);
            q.out[t] = y;
        }
    }
}

}  // namespace gcu
