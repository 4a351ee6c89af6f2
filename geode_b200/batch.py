"""The descriptors of libgeode_cuda.so's operators for many conversations at once (include/geode_cuda.h): a paged KV cache,
a step's rows over it, and the rules applied to its logits. Pointers are device addresses (a tensor's data_ptr()),
strides count values; a program fills a descriptor where it allocates the buffers and passes it by reference:

    kv = PagedKV(k=..., v=..., type=I8, ...)
    rc = cuda_lib().gcuda_op_paged_append(C.byref(kv), C.byref(step), C.byref(rows), stream)
"""
from __future__ import annotations

import ctypes as C

F32, BF16, F16, I8 = 0, 1, 2, 3   # GCUDA_F32, GCUDA_BF16, GCUDA_F16, GCUDA_I8

_vp, _i32, _i64, _f32 = C.c_void_p, C.c_int, C.c_int64, C.c_float


class PagedKV(C.Structure):
    """gcuda_paged_kv: the cache."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp)] + \
               [(n, _i32) for n in ("type", "n_pages", "page_size", "n_kv_heads", "head_dim")] + \
               [(n, _i64) for n in ("page_stride", "pos_stride", "head_stride", "scale_page_stride", "scale_pos_stride",
                                    "scale_head_stride")]


class PagedBatch(C.Structure):
    """gcuda_paged_batch: the step's rows and their sequences' pages."""
    _fields_ = [(n, _i32) for n in ("n_seq", "n_rows", "max_rows", "max_pages")] + \
               [(n, _vp) for n in ("row_start", "length", "pages")] + [("pages_stride", _i64)]


class AppendRows(C.Structure):
    """gcuda_append_rows: what gcuda_op_paged_append takes and where the queries go."""
    _fields_ = [("type", _i32), ("n_heads", _i32), ("rope_dim", _i32), ("eps", _f32)] + \
               [(n, _vp) for n in ("q", "k", "v", "q_out")] + \
               [(n, _i64) for n in ("q_stride", "q_head_stride", "k_stride", "v_stride", "q_out_stride")] + \
               [(n, _vp) for n in ("q_norm", "k_norm", "inv_freq")]


class AttnRows(C.Structure):
    """gcuda_attn_rows: the queries of gcuda_op_paged_attn and its outputs."""
    _fields_ = [("type", _i32), ("n_heads", _i32), ("window", _i32), ("scale", _f32), ("q", _vp), ("out", _vp), ("lse", _vp),
                ("q_stride", _i64), ("q_head_stride", _i64), ("out_stride", _i64)]


class LogitRules(C.Structure):
    """gcuda_logit_rules: biases, penalties and masks of gcuda_op_logits_adjust."""
    _fields_ = [("history", _vp), ("history_len", _vp), ("history_stride", _i64), ("drafts", _vp), ("repetition", _vp),
                ("frequency", _vp), ("presence", _vp), ("bias_id", _vp), ("bias", _vp), ("bias_len", _vp),
                ("bias_stride", _i64), ("mask", _vp), ("mask_row", _vp), ("n_masks", _i32), ("mask_stride", _i64)]
