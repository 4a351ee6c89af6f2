"""The operators for many conversations at once where their sizes and values leave the ordinary: CTAs with several tiles and
several items, warps with several turns, wide vocabularies and long lists, values next to the types' ends, rows that are no
numbers, unseen values in every shape of the attention, plans that are wrong in part, memory elsewhere."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from geode_b200 import batch as gb  # noqa: E402
from geode_b200 import cuda_lib  # noqa: E402
import batch_helpers as bh  # noqa: E402
from batch_helpers import CODE, HALF_STEP, TORCH, Plan, ref  # noqa: E402
from test_batch_gpu import append_inputs, attn_inputs, check_adjust, check_append, check_attn, run_attn, rules_for, stream  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return cuda_lib()


@pytest.fixture(autouse=True)
def status_clear(L):
    torch.cuda.synchronize()
    L.gcuda_op_status(1)
    yield
    torch.cuda.synchronize()
    assert L.gcuda_op_status(1) == 0   # (a test that raises flags clears them itself)


class LongPlan(Plan):
    """A plan whose sequences are long or many: their values by one gather each."""

    def values(self, s, which, upto):
        P = self.page
        pos = torch.arange(upto)
        page = torch.from_numpy(self.table_host[s].astype(np.int64))[pos // P]
        x = self.view[page.to(self.device), which, (pos % P).to(self.device)].cpu().double()
        if self.scale_view is not None:
            x = x * self.scale_view[page.to(self.device), which, (pos % P).to(self.device)].cpu().double()[..., None]
        return x


# ------------------------------------------------------------------------------------------- tiny values ----
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [0, 2])
def test_append_tiny_rows(L, act, heads):
    """int8 rows whose largest value is next to the smallest normal number, or below it: the definition's codes, zeros among
    them."""
    tops = [1e-30, 1e-36, 3.7e-37, 1e-37, 1.3e-38, 1e-39, 1e-40, 1e-44]
    n = len(tops)
    plan = Plan([n], [n + 3], 4, 1, 64, "i8", seed=1)
    before, scales = plan.randomize(2)
    x = append_inputs(plan, act, heads, 0, False, 3)
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(n, 64, generator=g, dtype=torch.float64)
    rows[:, ::7] = 0.0
    rows /= rows.abs().amax(1, keepdim=True)
    rows = (rows * torch.tensor(tops, dtype=torch.float64)[:, None]).to(TORCH[act])
    x["v"][:n] = rows.cuda()
    x["k"][:n, :64] = -rows.cuda()
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    check_append(plan, x, act, heads, False, before, scales)


@pytest.mark.parametrize("cache", ["i8", "bf16", "f16"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 5])
def test_attend_tiny_queries(L, act, cache, tokens):
    """Queries far below 1 under a softmax scale that makes up for it."""
    plan = Plan([tokens, 1], [70, 9], 16, 2, 64, cache, seed=2)
    plan.randomize(3)
    x = attn_inputs(L, plan, act, 16, 4, q_scale=3e-37, scale=4e35)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 16)


# ---------------------------------------------------------------------------------------- rows of no numbers ----
@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "i8"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("tokens,heads", [(1, 8), (5, 8), (2, 1), (2, 8)])
@pytest.mark.parametrize("length", [5, 6001])
def test_attend_nan_query(L, act, cache, tokens, heads, length):
    """A query that is no number gives none, neither out nor lse, whether its item is cut or not; the others' bits stay."""
    plan = LongPlan([tokens, 1], [length, 40], 16, 1, 64, cache, seed=3)
    plan.randomize(4)
    x = attn_inputs(L, plan, act, heads, 5)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    out, lse = x["out"].clone(), x["lse"].clone()
    row, head = tokens - 1, heads // 2
    x["q"][row, head, 17] = math.nan
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    assert torch.isnan(x["out"][row, head].float()).all() and torch.isnan(x["lse"][row, head])
    x["out"][row, head], x["lse"][row, head] = out[row, head], lse[row, head]
    assert torch.equal(x["out"], out) and torch.equal(x["lse"], lse)


@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("length", [1, 33, 6001])
def test_attend_nan_key(L, act, cache, tokens, length):
    """A key that is no number, alone in its warp's positions: out and lse of the rows that see it are no numbers."""
    length = max(length, tokens)
    plan = LongPlan([tokens], [length], 16, 1, 64, cache, seed=5)
    plan.randomize(6)
    x = attn_inputs(L, plan, act, 8, 7)
    p = length - tokens   # (every row sees it)
    at = (int(plan.table_host[0, p // 16]), 0, p % 16)
    if cache == "i8":
        plan.scale_view[at] = math.nan
    else:
        plan.view[at] = math.nan
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    assert torch.isnan(x["out"].float()).all() and torch.isnan(x["lse"]).all()


# ------------------------------------------------------------------------------------------------- the device ----
def host_address(keep):
    """An address of ordinary host memory, 256-byte aligned."""
    a = np.zeros(1 << 16, np.uint8)
    keep.append(a)
    return (a.ctypes.data + 255) // 256 * 256


def test_every_buffer_elsewhere_is_refused(L):
    """Each array that a kernel would follow, as host memory: refused before anything is launched."""
    keep = []
    plan = Plan([2], [5], 16, 2, 64, "i8")
    x = attn_inputs(L, plan, "f32", 4, 1)
    y = append_inputs(plan, "f32", 4, 64, True, 1)

    def swapped(d, name, f):
        was = getattr(d, name)
        setattr(d, name, host_address(keep))
        rc = f()
        setattr(d, name, was)
        return rc

    attend = lambda: run_attn(L, plan, x)  # noqa: E731
    append = lambda: L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(y["desc"]), stream())  # noqa: E731
    for name in ("k", "v", "k_scale", "v_scale"):
        assert swapped(plan.kv, name, attend) == -1 and swapped(plan.kv, name, append) == -1, name
    for name in ("row_start", "length", "pages"):
        assert swapped(plan.batch, name, attend) == -1 and swapped(plan.batch, name, append) == -1, name
    for name in ("q", "out", "lse"):
        assert swapped(x["desc"], name, attend) == -1, name
    for name in ("q", "k", "v", "q_out", "q_norm", "k_norm", "inv_freq"):
        assert swapped(y["desc"], name, append) == -1, name
    work = host_address(keep)
    assert L.gcuda_op_paged_attn(ref(plan.kv), ref(plan.batch), ref(x["desc"]), work, x["need"], stream()) == -1
    h, t, r = rules_for(2, 2, 500, 3)
    src, dst = torch.zeros(6, 500, device="cuda"), torch.zeros(6, 500, device="cuda")
    adjust = lambda a, b: L.gcuda_op_logits_adjust(ref(r), a, b, gb.F32, 2, 2, 500, 500, 500, stream())  # noqa: E731
    for name in ("history", "history_len", "drafts", "repetition", "frequency", "presence", "bias_id", "bias", "bias_len", "mask", "mask_row"):
        assert swapped(r, name, lambda: adjust(src.data_ptr(), dst.data_ptr())) == -1, name
    assert adjust(host_address(keep), dst.data_ptr()) == -1 and adjust(src.data_ptr(), host_address(keep)) == -1
    assert attend() == 0 and append() == 0 and adjust(src.data_ptr(), dst.data_ptr()) == 0
    torch.cuda.synchronize()


def test_page_locked_and_managed_memory_is_taken(L):
    """Host memory that the device can follow: a plan may lie there, and the outputs in managed memory."""
    plan = Plan([2], [5], 16, 2, 64, "bf16")
    plan.randomize(1)
    x = attn_inputs(L, plan, "bf16", 4, 1)
    pinned = [t.cpu().pin_memory() for t in (plan.row_start, plan.length, plan.table)]
    plan.batch.row_start, plan.batch.length, plan.batch.pages = (t.data_ptr() for t in pinned)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, "bf16", 4)
    p = C.c_void_p()
    assert L.cudaMallocManaged(C.byref(p), C.c_size_t(4096), 1) == 0   # (of the runtime that the library is linked with)
    x["desc"].lse = p.value
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    lse = np.ctypeslib.as_array(C.cast(p, C.POINTER(C.c_float)), (2, 4)).copy()
    assert L.cudaFree(p) == 0
    assert np.array_equal(lse, x["lse"].cpu().numpy())


THREADS = """
import sys, threading
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import batch_helpers as bh
from geode_b200 import batch as gb, cuda_lib
from test_batch_gpu import append_inputs, attn_inputs, run_attn, check_attn
L = cuda_lib()
plan = bh.Plan([1, 2], [40, 70], 16, 2, 64, "i8")
plan.randomize(1)
x = attn_inputs(L, plan, "f32", 4, 2)
y = append_inputs(plan, "f32", 4, 32, True, 1)
src, dst = torch.randn(2, 100, device="cuda"), torch.zeros(2, 100, device="cuda")
r = gb.LogitRules()
st = torch.cuda.current_stream().cuda_stream
torch.cuda.synchronize()
rc = []
def call(which):
    if which == 0: rc.append(run_attn(L, plan, x, st))
    if which == 1: rc.append(L.gcuda_op_paged_append(bh.ref(plan.kv), bh.ref(plan.batch), bh.ref(y["desc"]), st))
    if which == 2: rc.append(L.gcuda_op_logits_adjust(bh.ref(r), src.data_ptr(), dst.data_ptr(), gb.F32, 2, 0, 100, 100, 100, st))
for which in (0, 1, 2):
    t = threading.Thread(target=call, args=(which,))
    t.start(); t.join()
torch.cuda.synchronize()
assert rc == [0, 0, 0], rc
assert torch.equal(src, dst)
print("threads")
"""


def test_first_call_of_a_thread(L):
    """A thread's first call into CUDA may be one of these."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = THREADS.format(root=os.path.dirname(here), tests=here)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "threads" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------------------------------------- wrong plans ----
def left_out(plan, bad):
    """The plan as the operators see it: the bad sequences own nothing."""
    for s in bad:
        plan.rows[s] = 0


BAD_PLANS = [
    # lengths, row_start (None: as it should be), the sequences that are left out
    ([49, 17, 9], None, [0]), ([5, -3, 9], None, [1]), ([5, 17, 2**31 - 1], None, [2]), ([-2**31, 17, 33], None, [0, 2]),
    ([5, 17, 9], [0, 9, 2, 3], [0, 1]), ([5, 17, 9], [-2, 1, 2, 3], [0]), ([5, 17, 9], [0, 1, 2, 99], [2]),
    ([5, 17, 9], [0, 1, 2, 4], [2]), ([5, 17, 9], [2**31 - 1, 1, 2, 3], [0]), ([5, 17, 9], [0, 2, 2, 3], [0, 1]),
]


@pytest.mark.parametrize("lengths,starts,bad", BAD_PLANS, ids=str)
@pytest.mark.parametrize("cache", ["i8", "bf16"])
def test_wrong_plans(L, lengths, starts, bad, cache):
    """Sequences whose rows or lengths are out of range are left out whole, flagged, and the others served: rows, cache and
    outputs exactly."""
    plan = Plan([1, 1, 1], [5, 17, 9], 16, 2, 64, cache, seed=2)
    plan.batch.n_rows = 3
    before, scales = plan.randomize(3)
    plan.length.copy_(torch.tensor(lengths, dtype=torch.int32))
    if starts:
        plan.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        plan.start_host = np.array(starts, np.int32)
    left_out(plan, bad)
    act = "f32" if cache == "i8" else "bf16"
    y = attn_inputs(L, plan, act, 4, 5)
    assert run_attn(L, plan, y) == 0
    torch.cuda.synchronize()
    assert L.gcuda_op_status(1) == 2
    check_attn(plan, y, act, 4)      # (rows of no good sequence: as they were)
    x = append_inputs(plan, act, 2, 32, True, 4)
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    assert L.gcuda_op_status(1) in (0, 2)   # (a bad sequence that no row falls to is not met)
    check_append(plan, x, act, 2, True, before, scales)
    owned = {int(plan.start_host[s]) for s in range(3) if plan.rows[s]}
    for row in range(3):
        assert (x["q_out"][row] == 77.0).all() == (row not in owned)


# ---------------------------------------------------------------------------------------------- unseen values ----
@pytest.mark.parametrize("heads,tokens", [(1, 4), (1, 8), (2, 4), (4, 4), (8, 5), (16, 4)])   # rows an item: 4, 8, 8, 16, 40, 64
@pytest.mark.parametrize("act,cache", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16"), ("bf16", "i8"), ("f32", "i8")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_unseen_values_in_every_shape(L, heads, tokens, act, cache, dim, bad):
    """The newest position, which only the last row sees, and (under a window) the oldest one, which only the first row
    sees: whatever they hold, the other rows' bits stay."""
    for window in (0, 21):
        plan = LongPlan([tokens, tokens], [130 + tokens, tokens], 16, 1, dim, cache, seed=8)
        plan.randomize(9)
        x = attn_inputs(L, plan, act, heads, 10, window=window)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        clean, clean_lse = x["out"].clone(), x["lse"].clone()
        check_attn(plan, x, act, heads)
        places = [(0, plan.lengths[0] - 1, tokens - 1), (1, plan.lengths[1] - 1, 2 * tokens - 1)]
        if window:
            places.append((0, plan.lengths[0] - tokens + 1 - window, 0))
        for which in (0, 1):   # keys, values
            target = plan.scale_view if cache == "i8" else plan.view
            kept = target.clone()
            touched = set()
            for s, p, row in places:
                target[int(plan.table_host[s, p // 16]), which, p % 16] = bad
                touched.add(row)
            assert run_attn(L, plan, x) == 0
            torch.cuda.synchronize()
            target.copy_(kept)
            # (a key's scale of inf makes scores of -inf, weights of 0, as well as inf: nothing to say about the rows that see it)
            either = which == 0 and cache == "i8" and bad == math.inf
            for row in range(2 * tokens):
                if row not in touched:
                    assert torch.equal(x["out"][row], clean[row]) and torch.equal(x["lse"][row], clean_lse[row]), (window, which, row)
                elif not either:
                    assert not torch.isfinite(x["out"][row].float()).any(), (window, which, row)
