// batch.cu - the operators for many conversations at once (gcuda_op_paged_append, gcuda_op_paged_attn,
// gcuda_op_logits_adjust): argument checks and launches. A translation unit of its own.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/geode_cuda.h"
#include "device.hpp"
#include "logits_adjust.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_attn_plan.hpp"

using namespace gcu;

namespace {

bool activation(int type) { return type == GCUDA_F32 || type == GCUDA_BF16 || type == GCUDA_F16; }
bool misaligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
size_t value_bytes(int type) { return type == GCUDA_F32 ? 4 : type == GCUDA_I8 ? 1 : 2; }
template <typename... P>
bool words(const P *...p) { return !(misaligned(p, 4) || ...); }   // (32-bit values; NULL passes)

// Whether n rows of two buffers, `width` values `stride` apart, share no value: apart as a whole, or columns of the same
// rows (the parts of a fused q | k | v row).
struct RowSpan {
    const void *p;
    int64_t stride, width;
};
bool apart(const RowSpan &a, const RowSpan &b, int64_t n, int64_t bytes) {
    auto low = [&](const RowSpan &r) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(r.p)) + std::min<int64_t>(0, (n - 1) * r.stride) * bytes; };
    auto high = [&](const RowSpan &r) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(r.p)) + (std::max<int64_t>(0, (n - 1) * r.stride) + r.width) * bytes; };
    if (high(a) <= low(b) || high(b) <= low(a)) return true;
    const int64_t step = (a.stride < 0 ? -a.stride : a.stride) * bytes;
    if (a.stride != b.stride || step == 0) return false;
    const int64_t d = ((static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.p))) % step + step) % step;
    return d >= a.width * bytes && d + b.width * bytes <= step;
}
// query rows, whose heads lie head_stride apart
RowSpan query_rows(const void *q, int type, int64_t stride, int64_t head_stride, int n_heads, int head_dim) {
    const int64_t over = (n_heads - 1) * head_stride;
    return {static_cast<const uint8_t *>(q) + std::min<int64_t>(0, over) * static_cast<int64_t>(value_bytes(type)), stride, (over < 0 ? -over : over) + head_dim};
}

// Whether a stretch of memory meets any of n rows of `width` bytes, `step` bytes apart.
struct Stretch {
    const void *p;
    int64_t bytes;   // (nothing at NULL)
};
bool meets(const Stretch &a, const void *rows, int64_t step, int64_t width, int64_t n) {
    if (!a.p) return false;
    __int128 base = reinterpret_cast<uintptr_t>(rows), w = width, d = step;
    const __int128 lo = reinterpret_cast<uintptr_t>(a.p), hi = lo + a.bytes;
    if (d < 0) base += (n - 1) * d, d = -d;
    if (d == 0 || n == 1) return base < hi && lo < base + w;
    const __int128 first = lo - w < base ? 0 : (lo - w - base) / d + 1, end = hi <= base ? 0 : (hi - base + d - 1) / d;   // rows that end behind lo; that begin before hi
    return first < (end < n ? end : n);
}
// rows that are written: none over another
bool rows_apart(const RowSpan &r, int64_t n) { return n == 1 || (r.stride < 0 ? -r.stride : r.stride) >= r.width; }

// The geometry alone (what the scratch's size follows from); then with the pointers
bool good_geometry(const gcuda_paged_kv *kv, const gcuda_paged_batch *b) {
    return kv && b && (kv->type == GCUDA_I8 || kv->type == GCUDA_BF16 || kv->type == GCUDA_F16) && kv->n_pages >= 1 &&
           kv->page_size >= 1 && kv->n_kv_heads >= 1 && kv->n_kv_heads <= 1024 &&
           (kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256) && b->n_seq >= 1 && b->n_rows >= 1 &&
           b->n_seq <= (1 << 30) && b->n_rows <= (1 << 30) &&
           b->max_rows >= 1 && b->max_pages >= 1 && b->pages_stride >= 0 &&
           static_cast<int64_t>(b->max_pages) * kv->page_size <= (1ll << 30);
}
bool good_cache(const gcuda_paged_kv *kv, const gcuda_paged_batch *b) {
    if (!good_geometry(kv, b) || !kv->k || !kv->v || !b->row_start || !b->length || !b->pages) return false;
    if ((kv->type == GCUDA_I8) != (kv->k_scale != nullptr) || (kv->type == GCUDA_I8) != (kv->v_scale != nullptr)) return false;
    if (!words(kv->k_scale, kv->v_scale, b->row_start, b->length, b->pages)) return false;
    const int64_t unit = 16 / static_cast<int64_t>(value_bytes(kv->type));
    return !misaligned(kv->k, 16) && !misaligned(kv->v, 16) && kv->page_stride % unit == 0 && kv->pos_stride % unit == 0 &&
           kv->head_stride % unit == 0 && kv->page_stride >= 0 && kv->pos_stride >= 0 && kv->head_stride >= 0;
}

// f(activation type, cache type) for the call's types
template <int CACHE, typename F>
int by_activation(int act, F f) {
    if (act == GCUDA_F32) return f(float{}, std::integral_constant<int, CACHE>{});
    if (act == GCUDA_BF16) return f(__nv_bfloat16{}, std::integral_constant<int, CACHE>{});
    return f(__half{}, std::integral_constant<int, CACHE>{});
}
template <typename F>
int by_types(int act, int cache, F f) {
    if (cache == GCUDA_I8) return by_activation<GCUDA_I8>(act, f);
    if (cache == GCUDA_BF16) return by_activation<GCUDA_BF16>(act, f);
    return by_activation<GCUDA_F16>(act, f);
}
template <typename F>
int by_dim(int hd, F f) {
    if (hd == 64) return f(std::integral_constant<int, 64>{});
    if (hd == 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}
int launched(cudaError_t e) { return e == cudaSuccess ? GCUDA_OK : GCUDA_E_CUDA; }

template <typename T, int U>
int launch_adjust_slices(AdjustArgs a, cudaStream_t st) {
    using P = AdjustShape<T, U>;
    a.slices = (a.V + P::slice - 1) / P::slice;
    if (static_cast<int64_t>(a.S) * a.slices > 0x7fffffff) return GCUDA_E_ARG;
    if (!shared_opt_in<k_logits_adjust<T, U>>(P::smem)) return GCUDA_E_CUDA;
    return launched(launch_ex(k_logits_adjust<T, U>, dim3(a.S * a.slices), dim3(kAdjustThreads), P::smem, st, true, a));
}
// Slices of 4096 tokens (33 KB of counts; four CTAs an SM for floats, six for 16 bits) where they make two CTAs an SM or more, of
// one load a thread otherwise. With one, two and four loads a thread: 64 x 5 rows of 248320 floats 234, 131 and 130 us, of bf16
// 134, 94 and 145; 100 rows of 50257 bf16 21.4, 15.7 and 19.0; one row of 248320 floats (61 slices of 4096) 10.7, 11.0 and 12.2.
template <typename T>
int launch_adjust(const AdjustArgs &a, cudaStream_t st) {
    constexpr int U = sizeof(T) == 4 ? 4 : 2;
    const int64_t wide = static_cast<int64_t>(a.S) * ((a.V + AdjustShape<T, U>::slice - 1) / AdjustShape<T, U>::slice);
    return wide >= 2 * sm_count() ? launch_adjust_slices<T, U>(a, st) : launch_adjust_slices<T, 1>(a, st);
}

}  // namespace

extern "C" {

int gcuda_op_paged_append(const gcuda_paged_kv *kv, const gcuda_paged_batch *b, const gcuda_append_rows *x, void *stream) {
    if (!good_cache(kv, b) || !x || !activation(x->type) || !x->k || !x->v || x->n_heads < 0 || x->n_heads > 1024 ||
        (x->n_heads > 0) != (x->q != nullptr) || (x->n_heads > 0) != (x->q_out != nullptr) || x->rope_dim < 0 ||
        x->rope_dim % 2 || x->rope_dim > kv->head_dim || (x->rope_dim > 0 && !x->inv_freq) || !(x->eps >= 0.0f) ||
        (x->q && x->q == x->q_out && (x->q_stride != x->q_out_stride || x->q_head_stride != kv->head_dim)))
        return GCUDA_E_ARG;
    const size_t es = value_bytes(x->type);
    if (misaligned(x->q, es) || misaligned(x->k, es) || misaligned(x->v, es) || misaligned(x->q_out, es) ||
        !words(x->q_norm, x->k_norm, x->inv_freq))
        return GCUDA_E_ARG;
    if (x->q) {   // q_out is q itself or apart from all that is read
        const int64_t kv_width = static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim;
        const RowSpan out{x->q_out, x->q_out_stride, static_cast<int64_t>(x->n_heads) * kv->head_dim};
        if ((x->q != x->q_out && !apart(query_rows(x->q, x->type, x->q_stride, x->q_head_stride, x->n_heads, kv->head_dim), out, b->n_rows, es)) ||
            !apart({x->k, x->k_stride, kv_width}, out, b->n_rows, es) || !apart({x->v, x->v_stride, kv_width}, out, b->n_rows, es) ||
            !rows_apart(out, b->n_rows))
            return GCUDA_E_ARG;
    }
    if (const int rc = on_current_device(kv->k, kv->v, kv->k_scale, kv->v_scale, b->row_start, b->length, b->pages, x->q, x->k, x->v, x->q_out,
                                         x->q_norm, x->k_norm, x->rope_dim > 0 ? x->inv_freq : nullptr))
        return rc;
    // A row's warps: one where the rows alone make three CTAs an SM, else more, up to a turn for every warp. For one warp a row,
    // and warps for three, four and nine CTAs an SM: 1280 rows to int8 22, 16.0, 19.6 and 22 us, 1000 prompt rows 12.4, 10.0,
    // 10.6 and 12.5, 320 rows 15.4, 10.3, 10 and 10.4, 9645 prompt rows 56 (57 with nine)
    const int per_turn = 256 / kv->head_dim;   // vectors
    const int turns = (x->n_heads + per_turn - 1) / per_turn + 2 * ((kv->n_kv_heads + per_turn - 1) / per_turn);
    const int warps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(turns, (3ll * kAppendWarps * sm_count() + b->n_rows - 1) / b->n_rows)));
    const int64_t grid = (static_cast<int64_t>(b->n_rows) * warps + kAppendWarps - 1) / kAppendWarps;
    if (grid > 0x7fffffff) return GCUDA_E_ARG;
    const int half = x->rope_dim / 2;
    const size_t word = kv->type == GCUDA_I8 ? 8 : 4;   // the angles' and the odd halves' staging values
    const size_t smem = kAppendThreads * kAppendAhead * 8 * value_bytes(x->type) + kAppendWarps * half * 2 * word +
                        (half % 4 ? kAppendThreads * 8 * word : 0);
    auto vec = [&](const void *p, int64_t stride, int64_t head_stride) {
        return p && !misaligned(p, 4 * es) && stride % 4 == 0 && head_stride % 4 == 0;
    };
    AppendArgs a{*kv, *b, *x, warps, vec(x->q, x->q_stride, x->q_head_stride), vec(x->k, x->k_stride, 0),
                 vec(x->v, x->v_stride, 0), vec(x->q_out, x->q_out_stride, 0), device_status()};
    if (!a.status) return GCUDA_E_CUDA;
    return by_types(x->type, kv->type, [&](auto act, auto cache) {
        return by_dim(kv->head_dim, [&](auto hd) {
            if (!shared_opt_in<k_paged_append<hd(), decltype(act), cache()>>(kAppendMaxShared)) return static_cast<int>(GCUDA_E_CUDA);
            return launched(launch_ex(k_paged_append<hd(), decltype(act), cache()>, dim3(static_cast<unsigned>(grid)), dim3(kAppendThreads), smem,
                                      static_cast<cudaStream_t>(stream), true, a));
        });
    });
}

size_t gcuda_op_paged_attn_work_bytes(const gcuda_paged_kv *kv, const gcuda_paged_batch *b, int n_heads) {
    if (!good_geometry(kv, b) || b->max_rows > kMaxTok || n_heads < 1 || n_heads > 1024 || n_heads % kv->n_kv_heads) return 0;
    return plan_paged_attn(*kv, *b, n_heads).total;
}

int gcuda_op_paged_attn(const gcuda_paged_kv *kv, const gcuda_paged_batch *b, const gcuda_attn_rows *x, void *d_work,
                        size_t work_bytes, void *stream) {
    if (!good_cache(kv, b) || !x || !activation(x->type) || !x->q || !x->out || !d_work || misaligned(d_work, 256) ||
        x->window < 0)
        return GCUDA_E_ARG;
    const size_t need = gcuda_op_paged_attn_work_bytes(kv, b, x->n_heads);
    if (need == 0 || work_bytes < need) return GCUDA_E_ARG;
    const size_t es = value_bytes(x->type);
    if (misaligned(x->q, es) || misaligned(x->out, es) || !words(x->lse)) return GCUDA_E_ARG;
    // out and lse apart from each other and from q
    const RowSpan q = query_rows(x->q, x->type, x->q_stride, x->q_head_stride, x->n_heads, kv->head_dim),
                  out{x->out, x->out_stride, static_cast<int64_t>(x->n_heads) * kv->head_dim};
    if (!apart(q, out, b->n_rows, es) || !rows_apart(out, b->n_rows)) return GCUDA_E_ARG;
    for (const RowSpan &r : {q, out})
        if (meets({x->lse, static_cast<int64_t>(b->n_rows) * x->n_heads * 4}, r.p, r.stride * static_cast<int64_t>(es), r.width * static_cast<int64_t>(es), b->n_rows))
            return GCUDA_E_ARG;
    if (const int rc = on_current_device(kv->k, kv->v, kv->k_scale, kv->v_scale, b->row_start, b->length, b->pages, x->q, x->out, x->lse, d_work))
        return rc;
    const PagedAttnPlan p = plan_paged_attn(*kv, *b, x->n_heads);
    uint8_t *w = static_cast<uint8_t *>(d_work);
    // p / page_size by a multiplication, exact for p < 2^31: with 2^l >= page_size the multiplier is less than
    // page_size / 2^(31 + l) too large, which p < 2^31 does not carry over the next integer
    int l = 0;
    while ((1ll << l) < kv->page_size) ++l;
    const uint64_t d = static_cast<uint64_t>(kv->page_size);
    const uint32_t mul = static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d);
    PagedAttnArgs a{*kv, *b, *x, device_status(), mul, 31 + l, reinterpret_cast<int4 *>(w + p.cut),
                          reinterpret_cast<float4 *>(w + p.stats), reinterpret_cast<float4 *>(w + p.part)};
    if (a.x.window >= 1 << 30) a.x.window = 0;   // (no sequence is longer: all positions; the differences stay in 32 bits)
    if (!a.status) return GCUDA_E_CUDA;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kv->type == GCUDA_I8) return launch_paged_attn_i8(a, p, st);
    if (kv->type == GCUDA_BF16) return launch_paged_attn_bf16(a, p, st);
    return launch_paged_attn_f16(a, p, st);
}

int gcuda_op_logits_adjust(const gcuda_logit_rules *r, const void *d_in, void *d_out, int type, int S, int k, int V,
                           int64_t in_stride, int64_t out_stride, void *stream) {
    if (!r || !d_in || !d_out || !activation(type) || S < 1 || S > (1 << 20) || k < 0 || k > 64 || V < 1 || V > (1 << 30) || in_stride < V ||
        out_stride < V)
        return GCUDA_E_ARG;
    const int64_t rows = static_cast<int64_t>(S) * (k + 1);
    if ((r->history != nullptr) != (r->history_len != nullptr) || (r->bias_id != nullptr) != (r->bias != nullptr) ||
        (r->bias_id != nullptr) != (r->bias_len != nullptr) || (r->drafts && k == 0) || r->history_stride < 0 ||
        r->bias_stride < 0 || r->history_stride > (1 << 30) || r->bias_stride > (1 << 30) || (r->mask_row && !r->mask) ||
        (r->mask && (r->n_masks < 1 || r->mask_stride < (V + 31) / 32 || (!r->mask_row && r->n_masks < rows))))
        return GCUDA_E_ARG;
    if (misaligned(d_in, value_bytes(type)) || misaligned(d_out, value_bytes(type)) ||
        !words(r->history, r->history_len, r->drafts, r->repetition, r->frequency, r->presence, r->bias_id, r->bias, r->bias_len, r->mask, r->mask_row))
        return GCUDA_E_ARG;
    // in place row for row, or apart
    const char *i0 = static_cast<const char *>(d_in), *o0 = static_cast<const char *>(d_out);
    const int64_t es = static_cast<int64_t>(value_bytes(type)), ib = ((rows - 1) * in_stride + V) * es,
                  ob = ((rows - 1) * out_stride + V) * es;
    if (i0 == o0 ? in_stride != out_stride : (i0 < o0 + ob && o0 < i0 + ib)) return GCUDA_E_ARG;
    // (of the lists' last rows the first entry: how many are used is on the device, and the rows may be columns of a wider array)
    const int64_t n = S, lists = ((n - 1) * r->history_stride + 1) * 4, biases = ((n - 1) * r->bias_stride + 1) * 4;
    for (const Stretch &a : {Stretch{r->history, lists}, Stretch{r->history_len, n * 4}, Stretch{r->drafts, n * k * 4}, Stretch{r->repetition, n * 4},
                             Stretch{r->frequency, n * 4}, Stretch{r->presence, n * 4}, Stretch{r->bias_id, biases}, Stretch{r->bias, biases},
                             Stretch{r->bias_len, n * 4}, Stretch{r->mask, r->mask ? ((r->n_masks - 1) * r->mask_stride + (V + 31) / 32) * 4 : 0},
                             Stretch{r->mask_row, rows * 4}})
        if (meets(a, d_out, out_stride * es, V * es, rows)) return GCUDA_E_ARG;
    if (const int rc = on_current_device(d_in, d_out, r->history, r->history_len, r->drafts, r->repetition, r->frequency, r->presence, r->bias_id,
                                         r->bias, r->bias_len, r->mask, r->mask_row))
        return rc;
    AdjustArgs a{*r, d_in, d_out, S, k, V, 0, in_stride, out_stride, device_status()};
    if (!a.status) return GCUDA_E_CUDA;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == GCUDA_F32) return launch_adjust<float>(a, st);
    if (type == GCUDA_BF16) return launch_adjust<__nv_bfloat16>(a, st);
    return launch_adjust<__half>(a, st);
}

}  // extern "C"
