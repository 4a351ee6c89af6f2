"""Refusals of the operators for many conversations at once where what is written lies over itself or over what is read;
beside each the nearest call that is not refused (without a device it goes no further, with another error)."""
import ctypes as C

import pytest
import torch

from geode_b200 import batch as gb
from geode_b200 import cuda_lib
from test_batch_args import E_ARG, P, attn, batch, by, cache, rows

FAR = 1 << 40


@pytest.fixture(scope="module")
def good():
    """What a call gives that passes the checks: on a machine without a device the device's error, where there is one these
    addresses are refused."""
    rc = cuda_lib().gcuda_op_logits_adjust(C.byref(gb.LogitRules()), P, FAR, gb.F32, 1, 0, 8, 8, 8, None)
    assert rc not in (0, E_ARG) or torch.cuda.is_available()
    return rc


many = dict(n_rows=5, max_rows=5)


# 4 heads of 64 float values: rows of 1024 bytes
@pytest.mark.parametrize("d,refused", [(dict(q_out_stride=255), True), (dict(q_out_stride=-255), True), (dict(q_out_stride=0), True),
                                       (dict(q_out_stride=256), False), (dict(q_out_stride=-256, q_out=FAR), False), (dict(q_out_stride=300), False),
                                       (dict(q_out=P, q_stride=0, q_out_stride=0), True)])
def test_append_rows_over_each_other(good, d, refused):
    L = cuda_lib()
    d = {**dict(q_out=FAR, k=P + (1 << 30), v=P + (1 << 31)), **d}
    assert L.gcuda_op_paged_append(by(cache()), by(batch(**many)), by(rows(**d)), None) == (E_ARG if refused else good)
    if d["q_out"] == FAR:   # one row lies over no other
        assert L.gcuda_op_paged_append(by(cache()), by(batch()), by(rows(**d)), None) == good


LSE = [(dict(out_stride=255), True), (dict(out_stride=0), True), (dict(out_stride=-256), False), (dict(out_stride=257), False),
       # lse: 5 x 4 floats, 80 bytes
       (dict(lse=FAR), True), (dict(lse=FAR + 5 * 1024 - 4), True), (dict(lse=FAR + 5 * 1024), False), (dict(lse=FAR - 76), True),
       (dict(lse=FAR - 80), False), (dict(lse=P), True), (dict(lse=P + 5 * 1024 - 4), True), (dict(lse=P + 5 * 1024), False), (dict(lse=P - 80), False),
       (dict(lse=P - 79 + 3), True),
       # in the gap between out's rows, and over its ends
       (dict(out_stride=276, lse=FAR + 1024), False), (dict(out_stride=275, lse=FAR + 1024), True), (dict(out_stride=276, lse=FAR + 1020), True),
       (dict(out_stride=276, lse=FAR + 3 * 1104 + 1024), False), (dict(out_stride=-276, lse=FAR - 80), False), (dict(out_stride=-276, lse=FAR - 84), True),
       (dict(out_stride=-276, lse=FAR - 4 * 1104 - 80), False), (dict(out_stride=-276, lse=FAR - 4 * 1104 - 76), True),
       (dict(q_stride=0, lse=P + 1020), True), (dict(q_stride=0, lse=P + 1024), False)]


@pytest.mark.parametrize("d,refused", LSE, ids=str)
def test_attn_outputs_over_rows(good, d, refused):
    L = cuda_lib()
    rc = L.gcuda_op_paged_attn(by(cache()), by(batch(**many)), by(attn(**{**dict(out=FAR), **d})), P, 1 << 40, None)
    assert rc == (E_ARG if refused else good)


@pytest.mark.parametrize("name,bytes_", [("history", (7 + 1) * 4), ("history_len", 8), ("drafts", 2 * 2 * 4), ("repetition", 8), ("frequency", 8), ("presence", 8),
                                         ("bias_id", (5 + 1) * 4), ("bias", (5 + 1) * 4), ("bias_len", 8), ("mask", (2 * 6 + 4) * 4), ("mask_row", 6 * 4)])
def test_adjust_output_over_its_rules(good, name, bytes_):
    """(Of the lists' last rows the first entry counts: where their used entries end is not known on the host.)"""
    L = cuda_lib()
    S, k, V = 2, 2, 100
    d = dict(history=P, history_len=P, history_stride=7, drafts=P, repetition=P, frequency=P, presence=P, bias_id=P, bias=P, bias_len=P,
             bias_stride=5, mask=P, mask_row=P, n_masks=3, mask_stride=6)
    for at, refused in ((FAR, True), (FAR - bytes_, False), (FAR - bytes_ + 4, True), (FAR + (5 * 120 + 100) * 4, False), (FAR + (5 * 120 + 99) * 4, True),
                        (FAR + 400, bytes_ > 80), (FAR + 404, bytes_ > 76), (FAR + 396, True)):   # (the gap between two rows: 80 bytes)
        rc = L.gcuda_op_logits_adjust(C.byref(gb.LogitRules(**{**d, name: at})), P, FAR, gb.F32, S, k, V, V, 120, None)
        assert rc == (E_ARG if refused else good), (at - FAR, refused)
