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


# --------------------------------------------------------------------------------------------------- weights ----
@pytest.mark.parametrize("act,cache", [("f16", "i8"), ("f16", "f16"), ("bf16", "i8"), ("bf16", "f16")])
@pytest.mark.parametrize("tokens", [1, 2, 5])
@pytest.mark.parametrize("dim", [64, 256])
def test_attend_16_bit_weights(L, act, cache, tokens, dim):
    """16-bit activations: what the weights are rounded to is finer than the output's own rounding (values that cancel show
    it). The bound is check_attn's with weights of two f16 numbers: each to 2^-22."""
    plan = LongPlan([tokens] * 6, [tokens + 1, tokens + 2, 40, 200, 70, 1000], 16, 2, dim, cache, seed=7)
    plan.randomize(8)
    if cache == "f16":   # neighbours that nearly cancel
        for s in range(6):
            for p in range(0, plan.lengths[s] - 1, 2):
                a, b = ((int(plan.table_host[s, q // 16]), 1, q % 16) for q in (p, p + 1))
                plan.view[b] = -plan.view[a] * 0.75
    x = attn_inputs(L, plan, act, 16, 9, q_scale=0.3)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    out = x["out"].cpu().double()
    scale = float(x["desc"].scale)
    for s, n in enumerate(plan.rows):
        keys, values = plan.values(s, 0, plan.lengths[s]), plan.values(s, 1, plan.lengths[s])
        for i in range(n):
            row, end = int(plan.start_host[s]) + i, plan.lengths[s] - n + i + 1
            q = x["q"][row].cpu().double()
            o, _, size, mag = bh.attend(q, keys[:end], values[:end], scale)
            ds = mag * (dim + 10) * 2.0**-24 + 2.0**-21 * q.abs().amax(-1) * keys[:end].abs().sum(-1).amax() * abs(scale)
            tol = size * (2 * ds[:, None] + 2.0**-21 + (end + 40) * 2.0**-24) + HALF_STEP[act] * 1.01 * o.abs() + 2.0**-25
            assert ((out[row] - o).abs() <= tol).all(), (s, i, float(((out[row] - o).abs() / tol).max()))


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


# ----------------------------------------------------------------------------------------- many tiles, many items ----
@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "i8"), ("f16", "i8"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("tokens", [1, 2, 5])   # of 8 query heads a key head: 8, 16 and 40 rows
@pytest.mark.parametrize("dim", [64, 256])
def test_many_items_a_cta(L, act, cache, tokens, dim):
    """128 ragged sequences of two key heads: 256 items of several tiles each, more than the CTAs: a CTA goes from tile to
    tile and from item to item, and items are cut between CTAs."""
    rng = np.random.default_rng(dim + tokens)
    n = 128
    rows = [int(v) for v in rng.integers(1, tokens + 1, n)]
    lengths = [max(r, int(v)) for r, v in zip(rows, rng.integers(1, 1500 if dim == 64 else 700, n))]
    plan = LongPlan(rows, lengths, 32, 2, dim, cache, seed=dim, max_rows=tokens)
    plan.randomize(11)
    x = attn_inputs(L, plan, act, 16, 12, q_scale=2.0)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 16)
    again = x["out"].clone(), x["lse"].clone()
    for _ in range(4):   # the same bits run after run, whatever the scratch held
        x["work"].random_(0, 256)
        x["out"].fill_(3.0)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        assert torch.equal(again[0], x["out"]) and torch.equal(again[1], x["lse"])


@pytest.mark.parametrize("act,cache,tokens,dim", [("f32", "i8", 1, 128), ("f32", "i8", 5, 128), ("bf16", "bf16", 1, 128), ("bf16", "bf16", 3, 64),
                                                  ("f16", "f16", 5, 128), ("f16", "f16", 1, 64)])
def test_many_tiles_a_cta(L, act, cache, tokens, dim):
    """One sequence of 100000 positions with scores that climb: a CTA's running maxima are carried, and grow, from tile to
    tile."""
    n = 100_000
    plan = LongPlan([tokens], [n], 64, 1, dim, cache, seed=5)
    plan.randomize(6)
    x = attn_inputs(L, plan, act, 8, 7)
    # a direction that all queries share, along which the keys grow with the position
    P = plan.page
    u = torch.zeros(dim)
    u[:8] = 1.0
    climb = torch.linspace(0, 1, n)
    pos = torch.arange(n)
    page = torch.from_numpy(plan.table_host[0].astype(np.int64))[pos // P]
    if cache == "i8":
        codes = plan.view[page.cuda(), 0, (pos % P).cuda()]
        codes[:, 0] = (codes[:, 0].float() * 0.3 + (90 * climb[:, None] * u).cuda()).round().clamp(-127, 127).to(torch.int8)
        plan.view[page.cuda(), 0, (pos % P).cuda()] = codes
    else:
        k = plan.view[page.cuda(), 0, (pos % P).cuda()].float()
        k[:, 0] += (4 * climb[:, None] * u).cuda()
        plan.view[page.cuda(), 0, (pos % P).cuda()] = k.to(plan.view.dtype)
    x["q"][..., :8] += 6.0
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 8)


# ------------------------------------------------------------------------------------------- many turns a warp ----
@pytest.mark.parametrize("act,cache,heads,nkv,dim,rope,norm", [("bf16", "bf16", 16, 4, 128, 128, False), ("f16", "i8", 32, 4, 128, 128, True),
                                                             ("f32", "i8", 16, 2, 256, 64, True), ("f32", "f16", 24, 3, 64, 36, True),
                                                             ("bf16", "i8", 9, 5, 256, 256, False)])
def test_append_many_turns(L, act, cache, heads, nkv, dim, rope, norm):
    """Prompts: more rows than warps, so that a warp goes through all of a row's turns and its ring is used over and over;
    every row against the definition."""
    rows, lengths = [1500, 1, 2300], [1500, 90, 4001]
    plan = Plan(rows, lengths, 32, nkv, dim, cache, seed=1, spare=3)
    plan.randomize(2)
    before, scales = plan.view.clone(), None if plan.scale_view is None else plan.scale_view.clone()
    x = append_inputs(plan, act, heads, rope, norm, 3)
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    N = sum(rows)
    pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lengths)])
    page = torch.cat([torch.from_numpy(plan.table_host[s].astype(np.int64))[torch.arange(n - r, n) // 32] for s, (r, n) in enumerate(zip(rows, lengths))])
    angle = pos.double()[:, None, None] * x["freq"].cpu().double()
    h = rope // 2

    def vectors(v, w):   # [row][head][dim] in 64 bits
        v = v.double()
        if norm:
            v = v / (v.square().mean(-1, keepdim=True) + float(np.float32(1e-6))).sqrt() * (1.0 + w.cpu().double())
        a, b = v[..., :h], v[..., h:2 * h]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), v[..., 2 * h:]], -1)

    def size(y):   # a rotation's two products of values up to the pair's size
        p = y.abs().clone()
        p[..., :h] = 2 * torch.hypot(y[..., :h], y[..., h:2 * h])
        p[..., h:2 * h] = p[..., :h]
        return p

    arithmetic = ((dim + 5) / 2 + 12) * 2.0**-24
    q = vectors(x["q"][:N, :, :dim].cpu(), x["qn"])
    got = x["q_out"].cpu().double()
    assert ((got[:N] - q).abs() <= arithmetic * size(q) + HALF_STEP[act] * 1.01 * q.abs() + 1e-7 * HALF_STEP[act]).all()
    assert (got[N:] == 77.0).all()
    k = vectors(x["k"][:N, :nkv * dim].cpu().view(N, nkv, dim), x["kn"])
    v = x["v"][:N].cpu().double().view(N, nkv, dim)
    at = (page.cuda(), slice(None), (pos % 32).cuda())
    held = plan.view[at].cpu()
    for which, y in ((0, k), (1, v)):
        if cache == "i8":
            y = y.float().double()
            top = y.abs().amax(-1, keepdim=True)
            codes = torch.round(y * 127.0 / top).to(torch.int8)   # (to even)
            # the definition in 64 bits rounds to float first; this one's own 64-bit roundings may tip a value there
            off = held[:, which] != codes
            assert off.float().mean() <= 1e-6 and (held[:, which].int() - codes.int()).abs().max() <= 1
            got_scale = plan.scale_view[at].cpu()[:, which]
            want_scale = (top[..., 0] / 127.0).float()
            assert ((got_scale - want_scale).abs() <= want_scale * 2.0**-23).all()
        else:
            tol = arithmetic * size(y) if which == 0 else torch.zeros_like(y)
            assert ((held[:, which].double() - y).abs() <= tol + HALF_STEP[cache] * 1.01 * y.abs() + 2.0**-25).all()
    # the rest of the cache as it was
    plan.view[at] = before[at]
    assert torch.equal(plan.view.nan_to_num(-1) if cache != "i8" else plan.view, before.nan_to_num(-1) if cache != "i8" else before)
    if scales is not None:
        plan.scale_view[at] = scales[at]
        assert torch.equal(plan.scale_view.nan_to_num(-1), scales.nan_to_num(-1))


# ------------------------------------------------------------------------------ wide vocabularies, long lists ----
@pytest.mark.parametrize("act,S,k,V", [("f32", 24, 1, 50257), ("bf16", 30, 0, 50257), ("f16", 30, 2, 50001), ("f32", 5, 4, 248320)])
@pytest.mark.parametrize("layout", ["apart", "in place", "strided"])
def test_adjust_wide(L, act, S, k, V, layout):
    """Enough slices of 4096 tokens for every SM (the kernels of large batches), lists longer than a thread's first eight
    entries, tokens all over the vocabulary."""
    rows, history, biases = S * (k + 1), 5000, 2300
    h, t, r = rules_for(S, k, V, 5, history, biases, True, True)
    rng = np.random.default_rng(6)
    # words of all sizes, the same ones over and over
    h["history"][:] = np.minimum(V - 1, (np.float64(V + 1) ** rng.random((S, history)) - 1)).astype(np.int32)
    h["history"][:, 1] = -1
    h["bias_id"][:] = rng.integers(0, V, (S, biases))
    h["bias_id"][:, -40:] = h["bias_id"][:, :40]   # entries of one id far apart
    h["drafts"][:] = rng.integers(0, V, h["drafts"].shape)
    h["history_len"][:] = rng.integers(4000, history + 1, S)
    h["bias_len"][:] = biases
    h["history_len"][0], h["bias_len"][0] = 2048, 2049
    for n in ("history", "bias_id", "drafts", "history_len", "bias_len"):
        t[n].copy_(torch.from_numpy(h[n]))
    g = torch.Generator().manual_seed(7)
    x = (4 * torch.randn(rows, V, generator=g)).to(TORCH[act])
    pad_in, pad_out = (5, 3) if layout == "strided" else (0, 0)
    src = torch.full((rows, V + pad_in), 9.0, dtype=TORCH[act], device="cuda")
    src[:, :V] = x.cuda()
    dst = src if layout == "in place" else torch.full((rows, V + pad_out), 7.0, dtype=TORCH[act], device="cuda")
    assert L.gcuda_op_logits_adjust(ref(r), src.data_ptr(), dst.data_ptr(), CODE[act], S, k, V, src.stride(0), dst.stride(0), stream()) == 0
    torch.cuda.synchronize()
    got = dst.cpu()
    assert (got[:, V:] == 7.0).all()
    check_adjust(x, got[:, :V], act, S, k, V, h, history, biases, True, True, (True, True, True))


def test_adjust_lists_in_a_wider_array(L):
    """Lists that are the last columns of a wider array (an answer's tokens behind its prompt's): the other columns, and what is
    behind the used entries, do not count; the last row ends with its used entries."""
    S, k, V = 3, 1, 700
    h, t, r = rules_for(S, k, V, 11, history=25, biases=9)
    wide = {}
    for name, skip, width in (("history", 2000, 2025), ("bias_id", 7, 16), ("bias", 7, 16)):
        w = torch.full((S, width), V + 5 if name != "bias" else 3.0, dtype=t[name].dtype, device="cuda")
        n = h["history_len" if name == "history" else "bias_len"]
        for s in range(S):
            w[s, skip:skip + int(n[s])] = t[name][s, :int(n[s])]
        wide[name] = w.flatten()[:(S - 1) * width + skip + int(n[S - 1])].clone()
        setattr(r, name, wide[name].data_ptr() + 4 * skip)
    r.history_stride, r.bias_stride = 2025, 16
    x = torch.randn(S * (k + 1), V)
    src, dst = x.cuda(), torch.empty(S * (k + 1), V, device="cuda")
    assert L.gcuda_op_logits_adjust(ref(r), src.data_ptr(), dst.data_ptr(), gb.F32, S, k, V, V, V, stream()) == 0
    torch.cuda.synchronize()
    check_adjust(x, dst.cpu(), "f32", S, k, V, h, 25, 9, True, True, (True, True, True))


ALLOCATORS = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import batch_helpers as bh
from geode_b200 import batch as gb, cuda_lib
from test_batch_gpu import append_inputs, attn_inputs, run_attn, check_attn, rules_for, stream
L = cuda_lib()
plan = bh.Plan([1, 2], [40, 70], 16, 2, 64, "i8")
plan.randomize(1)
x = attn_inputs(L, plan, "f32", 4, 2)
assert run_attn(L, plan, x) == 0
torch.cuda.synchronize()
check_attn(plan, x, "f32", 4)
y = append_inputs(plan, "f32", 4, 32, True, 1)
assert L.gcuda_op_paged_append(bh.ref(plan.kv), bh.ref(plan.batch), bh.ref(y["desc"]), stream()) == 0
h, t, r = rules_for(2, 2, 500, 3)
src, dst = torch.zeros(6, 500, device="cuda"), torch.zeros(6, 500, device="cuda")
assert L.gcuda_op_logits_adjust(bh.ref(r), src.data_ptr(), dst.data_ptr(), gb.F32, 2, 2, 500, 500, 500, stream()) == 0
torch.cuda.synchronize()
print("taken")
"""


@pytest.mark.parametrize("conf", ["expandable_segments:True", "backend:cudaMallocAsync"])
def test_memory_of_other_allocators_is_taken(L, conf):
    """Mapped segments and the stream-ordered pools are the device's memory too."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = ALLOCATORS.format(root=os.path.dirname(here), tests=here)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTORCH_CUDA_ALLOC_CONF": conf})
    assert r.returncode == 0 and "taken" in r.stdout, r.stderr[-2000:]
