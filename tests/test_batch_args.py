"""The refusals of the operators for many conversations at once: every bad argument is an error before anything is
launched, so they are checked without a GPU (the pointers are never followed)."""
import ctypes as C
import subprocess

import pytest
import torch

from geode_b200 import batch as gb
from geode_b200 import CUDA_SO, cuda_lib

E_ARG = -1
P = 1 << 20   # an aligned address


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, type=gb.I8, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64,
             page_stride=16 * 128, pos_stride=128, head_stride=64, scale_page_stride=32, scale_pos_stride=2, scale_head_stride=1)
    return gb.PagedKV(**{**d, **kw})


def batch(**kw):
    d = dict(n_seq=1, n_rows=1, max_rows=1, max_pages=4, row_start=P, length=P, pages=P, pages_stride=4)
    return gb.PagedBatch(**{**d, **kw})


def rows(**kw):
    d = dict(type=gb.F32, n_heads=4, rope_dim=32, eps=1e-6, q=P, k=P, v=P, q_out=2 * P, q_stride=256, q_head_stride=64,
             k_stride=128, v_stride=128, q_out_stride=256, inv_freq=P)
    return gb.AppendRows(**{**d, **kw})


def attn(**kw):
    d = dict(type=gb.F32, n_heads=4, window=0, scale=0.1, q=P, out=1 << 40, lse=None, q_stride=256, q_head_stride=64, out_stride=256)
    return gb.AttnRows(**{**d, **kw})


def by(x):
    return None if x is None else C.byref(x)


BAD_CACHE = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(type=gb.F32), dict(type=9),
             dict(type=gb.F16), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(n_kv_heads=2000),
             dict(head_dim=96), dict(head_dim=512), dict(k=P + 8), dict(v=P + 1), dict(page_stride=16 * 128 + 8),
             dict(pos_stride=120), dict(head_stride=8), dict(pos_stride=-128),
             dict(k_scale=P + 2), dict(v_scale=P + 1)]
BAD_BATCH = [dict(n_seq=0), dict(n_rows=0), dict(max_rows=0), dict(max_pages=0), dict(row_start=None), dict(length=None),
             dict(pages=None), dict(pages_stride=-1), dict(n_seq=(1 << 30) + 1), dict(n_rows=(1 << 30) + 1),
             dict(row_start=P + 2), dict(length=P + 1), dict(pages=P + 3)]
BAD_ROWS = [dict(type=gb.I8), dict(type=7), dict(n_heads=-1), dict(n_heads=5000), dict(k=None), dict(v=None), dict(q=None),
            dict(q_out=None), dict(n_heads=0), dict(rope_dim=31), dict(rope_dim=66), dict(rope_dim=-2), dict(inv_freq=None),
            dict(eps=-1.0), dict(eps=float("nan")), dict(q_out=P, q_out_stride=512), dict(q_out=P, q_head_stride=128),
            dict(q=P + 2), dict(k=P + 1), dict(v=P + 3), dict(q_out=2 * P + 2), dict(q_norm=P + 2), dict(k_norm=P + 1),
            dict(inv_freq=P + 2), dict(q_out=P + 4), dict(q_out=P - 4), dict(k=2 * P + 1020), dict(v=2 * P - 508)]
BAD_ATTN = [dict(type=gb.I8), dict(n_heads=0), dict(n_heads=3), dict(n_heads=2000), dict(window=-1), dict(q=None), dict(out=None),
            dict(q=P + 1), dict(out=P + 2 + (1 << 30)), dict(lse=P + 2), dict(out=P), dict(out=P + 1020), dict(out=P - 1020)]


def test_library_loads_without_a_driver():
    """The driver's library is looked up where a call needs it, never linked: a machine without a GPU has none."""
    needed = subprocess.run(["readelf", "-d", CUDA_SO], capture_output=True, text=True, check=True).stdout
    assert "libcudart" in needed and "libcuda.so" not in needed


def ids(d):
    return ",".join(f"{k}={v}" for k, v in d.items())


@pytest.mark.parametrize("bad", BAD_CACHE, ids=ids)
def test_cache_refused(bad):
    L = cuda_lib()
    assert L.gcuda_op_paged_append(by(cache(**bad)), by(batch()), by(rows()), None) == E_ARG
    assert L.gcuda_op_paged_attn(by(cache(**bad)), by(batch()), by(attn()), P, 1 << 40, None) == E_ARG


@pytest.mark.parametrize("bad", BAD_BATCH, ids=ids)
def test_batch_refused(bad):
    L = cuda_lib()
    assert L.gcuda_op_paged_append(by(cache()), by(batch(**bad)), by(rows()), None) == E_ARG
    assert L.gcuda_op_paged_attn(by(cache()), by(batch(**bad)), by(attn()), P, 1 << 40, None) == E_ARG


@pytest.mark.parametrize("bad", BAD_ROWS, ids=ids)
def test_append_refused(bad):
    assert cuda_lib().gcuda_op_paged_append(by(cache()), by(batch()), by(rows(**bad)), None) == E_ARG


@pytest.mark.parametrize("bad", BAD_ATTN, ids=ids)
def test_attn_refused(bad):
    assert cuda_lib().gcuda_op_paged_attn(by(cache()), by(batch()), by(attn(**bad)), P, 1 << 40, None) == E_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are followed where there is a device")
def test_good_calls_pass_the_checks():
    """What the refusals start from, and rows side by side in one buffer (q | k | v, with and without other rows
    between): not refused, but without a device they go no further."""
    L = cuda_lib()
    E_CUDA = L.gcuda_op_logits_adjust(C.byref(gb.LogitRules()), P, 1 << 40, gb.F32, 1, 0, 8, 8, 8, None)
    assert E_CUDA not in (0, E_ARG)
    many = batch(n_rows=5, max_rows=5)
    for r in (rows(), rows(q_out=P, k=P + 1024, v=P + 1536, q_stride=512, k_stride=512, v_stride=512, q_out_stride=512),
              rows(q_out=P + 4 * 1024, k=P + 1024, v=P + 1536, q_stride=2048, k_stride=2048, v_stride=2048, q_out_stride=2048),
              rows(n_heads=0, q=None, q_out=None), rows(q_stride=0)):
        assert L.gcuda_op_paged_append(by(cache()), by(many), by(r), None) == E_CUDA
    for a in (attn(), attn(out=P + 1024, q_stride=512, out_stride=512), attn(out=P - 1024, q_stride=512, out_stride=512), attn(q_stride=0)):
        assert L.gcuda_op_paged_attn(by(cache()), by(many), by(a), P, 1 << 40, None) == E_CUDA
    for a in (attn(out=P + 1024, q_stride=512, out_stride=520), attn(out=P + 1020, q_stride=512, out_stride=512),
              attn(out=P + 1028, q_stride=512, out_stride=512)):
        assert L.gcuda_op_paged_attn(by(cache()), by(many), by(a), P, 1 << 40, None) == E_ARG


def test_attn_scratch_and_rows_refused():
    L = cuda_lib()
    need = L.gcuda_op_paged_attn_work_bytes(by(cache()), by(batch()), 4)
    assert need > 0
    for work, size in ((None, need), (P + 16, need), (P, need - 1)):
        assert L.gcuda_op_paged_attn(by(cache()), by(batch()), by(attn()), work, size, None) == E_ARG
    assert L.gcuda_op_paged_attn_work_bytes(by(cache()), by(batch(max_rows=9)), 4) == 0
    assert L.gcuda_op_paged_attn(by(cache()), by(batch(max_rows=9, n_rows=9)), by(attn()), P, 1 << 40, None) == E_ARG
    for heads in (0, 3, -2, 4000):
        assert L.gcuda_op_paged_attn_work_bytes(by(cache()), by(batch()), heads) == 0
    for null in range(3):
        a = [by(cache()), by(batch()), by(attn())]
        a[null] = None
        assert L.gcuda_op_paged_attn(*a, P, 1 << 40, None) == E_ARG
        a = [by(cache()), by(batch()), by(rows())]
        a[null] = None
        assert L.gcuda_op_paged_append(*a, None) == E_ARG


def test_adjust_refused():
    L = cuda_lib()
    good = dict(history=P, history_len=P, history_stride=4, drafts=P, repetition=P, bias_id=P, bias=P, bias_len=P,
                bias_stride=4, mask=P, mask_row=P, n_masks=1, mask_stride=4)
    far = 1 << 40

    def call(rules=None, d_in=P, d_out=far, type=gb.F32, S=2, k=2, V=100, si=100, so=100):
        r = gb.LogitRules(**{**good, **(rules or {})})
        return L.gcuda_op_logits_adjust(C.byref(r), d_in, d_out, type, S, k, V, si, so, None)

    bad = [dict(rules=x) for x in (dict(history=None), dict(history_len=None), dict(bias=None), dict(bias_id=None),
                                   dict(bias_len=None), dict(history_stride=-1), dict(bias_stride=-1), dict(mask=None),
                                   dict(n_masks=0), dict(mask_stride=3), dict(mask_row=None, n_masks=5))]
    bad += [dict(d_in=None), dict(d_out=None), dict(type=gb.I8), dict(type=-1), dict(S=0), dict(k=-1), dict(k=65), dict(V=0),
            dict(si=99), dict(so=99), dict(S=1 << 21), dict(k=0), dict(d_out=P, so=104), dict(d_out=P + 400),
            dict(d_out=P - 400), dict(d_in=P + 2), dict(d_out=far + 1)]
    bad += [dict(rules={n: P + 2}) for n in ("history", "history_len", "drafts", "repetition", "frequency", "presence", "bias_id",
                                            "bias", "bias_len", "mask", "mask_row")]
    bad += [dict(rules={n: (1 << 30) + 1}) for n in ("history_stride", "bias_stride")]
    assert torch.cuda.is_available() or call() not in (0, E_ARG)
    for b in bad:
        assert call(**b) == E_ARG, b
    assert L.gcuda_op_logits_adjust(None, P, far, gb.F32, 1, 0, 8, 8, 8, None) == E_ARG
