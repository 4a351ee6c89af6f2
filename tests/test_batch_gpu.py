"""The operators for many conversations at once on the GPU against their definitions in 64 bits: rows appended to a paged
cache, attention of each sequence's newest rows over its pages, logits adjusted before the acceptance."""
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


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------------------------------------------- append ----
def append_inputs(plan, act, heads, rope, norm, seed, gate=False, theta=1e6, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    N, nkv, hd = plan.n_rows, plan.kv_heads, plan.dim
    x = {}
    wide = 2 * hd if gate else hd
    x["q"] = (scale * torch.randn(N, heads, wide, generator=g)).to(TORCH[act]).cuda()
    x["k"] = (scale * torch.randn(N, nkv * hd + 3, generator=g)).to(TORCH[act]).cuda()   # (rows with a tail)
    x["v"] = (scale * torch.randn(N, nkv * hd, generator=g)).to(TORCH[act]).cuda()
    x["q_out"] = torch.full((N, heads, hd), 77.0, dtype=TORCH[act], device="cuda")
    x["qn"], x["kn"] = 0.2 * torch.randn(hd, generator=g).cuda(), 0.2 * torch.randn(hd, generator=g).cuda()
    x["freq"] = (theta ** (-torch.arange(0, rope, 2, dtype=torch.float64) / max(rope, 1))).float().cuda()
    x["desc"] = gb.AppendRows(type=CODE[act], n_heads=heads, rope_dim=rope, eps=1e-6, q=x["q"].data_ptr() if heads else None,
                              k=x["k"].data_ptr(), v=x["v"].data_ptr(), q_out=x["q_out"].data_ptr() if heads else None,
                              q_stride=x["q"].stride(0), q_head_stride=wide, k_stride=x["k"].stride(0),
                              v_stride=x["v"].stride(0), q_out_stride=x["q_out"].stride(0),
                              q_norm=x["qn"].data_ptr() if norm else None, k_norm=x["kn"].data_ptr() if norm else None,
                              inv_freq=x["freq"].data_ptr() if rope else None)
    return x


def check_append(plan, x, act, heads, norm, before, before_scales):
    """Every stored row by the definition; everything else as it was."""
    nkv, hd = plan.kv_heads, plan.dim
    want, want_s = before.clone(), None if before_scales is None else before_scales.clone()
    freq, qn, kn = x["freq"].cpu().numpy(), x["qn"].cpu().numpy(), x["kn"].cpu().numpy()
    q_want = torch.full(x["q_out"].shape, 77.0, dtype=torch.float64)
    bound = torch.zeros_like(q_want)
    tol = {}
    for row, _, pos, page, off in plan.places():
        for h in range(heads):
            src = x["q"][row, h, :hd].cpu().double().numpy()
            y = bh.norm_rotate(src, pos, qn if norm else None, 1e-6, freq)
            q_want[row, h] = torch.from_numpy(y)
            # float arithmetic: the sum of squares (hd + 5 roundings, halved by the root), six more on the way, the
            # rotation's two products of values up to the pair's size; then the rounding to the type
            pair = np.abs(y).copy()
            r = len(freq)
            if r:
                n = np.hypot(y[:r], y[r:2 * r])
                pair[:r], pair[r:2 * r] = 2 * n, 2 * n
            bound[row, h] = torch.from_numpy(((hd + 5) / 2 + 12) * 2.0**-24 * pair + HALF_STEP[act] * 1.01 * np.abs(y) + 1e-7 * HALF_STEP[act])
        for which in (0, 1):
            for h in range(nkv):
                src = x["kv"[which]][row, h * hd:(h + 1) * hd].cpu().double().numpy()
                y = bh.norm_rotate(src, pos, kn if norm else None, 1e-6, freq) if which == 0 else src
                if plan.cache == "i8":
                    codes, sc = bh.codes_of(y)
                    want[page, which, off, h] = torch.from_numpy(codes)
                    want_s[page, which, off, h] = float(sc)
                else:
                    want[page, which, off, h] = torch.from_numpy(y).float().to(want.dtype)
                    pair = np.abs(y).copy()
                    if which == 0 and len(freq):
                        r = len(freq)
                        pair[:r] = pair[r:2 * r] = 2 * np.hypot(y[:r], y[r:2 * r])
                    tol[page, which, off, h] = ((hd + 5) / 2 + 12) * 2.0**-24 * pair + HALF_STEP[plan.cache] * 1.01 * np.abs(y) + 1e-9
    got = plan.view.cpu()
    if plan.cache == "i8":
        assert torch.equal(got, want)
        assert torch.equal(plan.scale_view.cpu().nan_to_num(-1), want_s.nan_to_num(-1))
    else:
        for at, t in tol.items():
            # (against the unrounded definition: want was rounded, so one more half step)
            d = (got[at].double() - want[at].double()).abs().numpy()
            assert (d <= 2 * t).all(), (at, d.max())
            want[at] = got[at]
        assert torch.equal(got.nan_to_num(-1), want.nan_to_num(-1))   # the other rows untouched
    if heads:
        d = (x["q_out"].cpu().double() - q_want).abs()
        assert (d <= bound).all(), float((d - bound).max())


APPEND = [
    # act, cache, heads, kv heads, dim, rope, norm, page, rows, lengths, head major, gate
    ("f32", "i8", 4, 2, 256, 64, True, 64, [1], [1], False, False),
    ("f32", "i8", 4, 2, 256, 64, True, 16, [5, 0, 3, 1], [5, 0, 40, 200], False, True),
    ("bf16", "i8", 8, 1, 128, 128, True, 7, [2, 9], [9, 9], True, False),
    ("f16", "i8", 3, 3, 64, 32, False, 1, [4], [6], False, False),
    ("bf16", "bf16", 6, 2, 128, 128, False, 100, [33, 1], [33, 101], False, False),
    ("f16", "f16", 5, 5, 64, 20, True, 16, [17], [100], True, True),
    ("f32", "f16", 2, 1, 256, 0, True, 32, [1, 1, 1], [1, 2, 33], False, False),
    ("f32", "bf16", 0, 2, 64, 64, False, 32, [3], [35], False, False),
    ("f16", "bf16", 2, 2, 128, 2, True, 8, [3], [8], False, False),
    ("bf16", "f16", 2, 2, 256, 256, True, 8, [2, 2], [9, 17], True, False),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:7])))
def test_append(L, case):
    act, cache, heads, nkv, hd, rope, norm, page, rows, lengths, head_major, gate = case
    plan = Plan(rows, lengths, page, nkv, hd, cache, seed=3, head_major=head_major, spare=2)
    before, scales = plan.randomize(5)   # (NaN where no sequence holds anything: left so)
    x = append_inputs(plan, act, heads, rope, norm, 7, gate)
    if len(rows) > 1 and cache == "i8":
        x["v"][0].zero_()   # an all-zero row: zeros and scale 0
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    check_append(plan, x, act, heads, norm, before, scales)


def test_append_far_positions(L):
    """Positions whose angles a 32-bit product gets wrong by hundredths, one page each; a cache whose last pages lie
    beyond 2^32 values."""
    page, hd, nkv = 4096, 256, 2
    plan = Plan([1], [1], page, nkv, hd, "i8", extra_pages=0)
    n_pages = 1030   # 1030 * 2 * 4096 * 2 * 256 values > 2^32
    buf = torch.zeros(n_pages, 2, page, nkv, hd, dtype=torch.int8, device="cuda")
    sc = torch.zeros(n_pages, 2, page, nkv, device="cuda")
    pos = 1_000_003
    table = torch.full((1, pos // page + 1), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = n_pages - 1
    length = torch.tensor([pos + 1], dtype=torch.int32, device="cuda")
    plan.kv.k, plan.kv.v, plan.kv.n_pages = buf[:, 0].data_ptr(), buf[:, 1].data_ptr(), n_pages
    plan.kv.k_scale, plan.kv.v_scale = sc[:, 0].data_ptr(), sc[:, 1].data_ptr()
    plan.batch.length, plan.batch.pages, plan.batch.max_pages = length.data_ptr(), table.data_ptr(), table.shape[1]
    x = append_inputs(plan, "f32", 2, 64, True, 1, theta=1e4)
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    freq, kn, qn = x["freq"].cpu().numpy(), x["kn"].cpu().numpy(), x["qn"].cpu().numpy()
    for h in range(nkv):
        y = bh.norm_rotate(x["k"][0, h * hd:(h + 1) * hd].cpu().double().numpy(), pos, kn, 1e-6, freq)
        codes, s = bh.codes_of(y)
        assert np.array_equal(buf[-1, 0, pos % page, h].cpu().numpy(), codes) and float(sc[-1, 0, pos % page, h]) == float(s)
    y = bh.norm_rotate(x["q"][0, 0].cpu().double().numpy(), pos, qn, 1e-6, freq)
    assert np.abs(x["q_out"][0, 0].cpu().double().numpy() - y).max() <= ((hd + 5) / 2 + 12) * 2.0**-24 * 2 * np.abs(y).max() * 2


def test_append_in_place_and_other_stream(L):
    plan = Plan([2, 1], [70, 3], 16, 2, 128, "f16")
    x = append_inputs(plan, "f16", 4, 64, True, 2)
    y = append_inputs(plan, "f16", 4, 64, True, 2)
    y["desc"].q_out = y["q"].data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(y["desc"]), side.cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(x["q_out"][:3], y["q"][:3])


def test_append_bad_plans(L):
    """A page id out of range, a sequence longer than its table, more rows than positions, rows out of order: flagged,
    the bad rows left out, the good ones stored."""
    def run(plan):
        x = append_inputs(plan, "f32", 2, 32, False, 4)
        before, sc = plan.view.cpu().clone(), plan.scale_view.cpu().clone()
        assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
        torch.cuda.synchronize()
        assert L.gcuda_op_status(1) == 2
        return x, before, sc

    for bad in (-1, 10**6):
        plan = Plan([1, 1], [5, 17], 16, 2, 64, "i8")
        plan.table[0, 0] = bad
        x, before, sc = run(plan)
        plan.rows[0] = 0   # (the first sequence's row is not stored; its queries are rotated all the same)
        plan.start_host[0] = 1
        x["q_out"][0] = 77.0
        check_append(plan, x, "f32", 2, False, before, sc)
    for lengths, starts in (([49, 17], None), ([5, -3], None), ([5, 17], [0, 5, 2]), ([5, 17], [0, 1, 9]), ([5, 17], [-1, 1, 2])):
        plan = Plan([1, 1], [5, 17], 16, 2, 64, "i8")
        plan.length.copy_(torch.tensor(lengths, dtype=torch.int32))
        if starts:
            plan.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        before = plan.view.cpu().clone()
        x, before, sc = run(plan)
        good = [s for s in (0, 1) if 0 <= lengths[s] <= 32 and not starts]
        changed = (plan.view.cpu() != before).flatten(1).any(1)
        want = torch.zeros_like(changed)
        for s in good:
            p = lengths[s] - 1
            want[plan.table_host[s, p // 16]] = True
        assert not (changed & ~want).any() or starts
    plan = Plan([3], [2], 16, 2, 64, "i8")   # three rows, two positions: the first row has none
    x, before, sc = run(plan)
    check_append(plan, x, "f32", 2, False, before, sc)


# ------------------------------------------------------------------------------------------------- attention ----
def attn_inputs(L, plan, act, heads, seed, window=0, q_scale=1.0, gate=False, scale=None):
    g = torch.Generator().manual_seed(seed)
    hd = plan.dim
    wide = 2 * hd if gate else hd
    q = (q_scale * torch.randn(plan.n_rows, heads, wide, generator=g)).to(TORCH[act]).cuda()
    out = torch.full((plan.n_rows, heads, hd), 55.0, dtype=TORCH[act], device="cuda")
    lse = torch.full((plan.n_rows, heads), 55.0, device="cuda")
    need = L.gcuda_op_paged_attn_work_bytes(ref(plan.kv), ref(plan.batch), heads)
    assert need > 0
    work = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")   # (its contents do not matter)
    d = gb.AttnRows(type=CODE[act], n_heads=heads, window=window, scale=scale if scale is not None else 1 / math.sqrt(hd),
                    q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_stride=q.stride(0), q_head_stride=wide,
                    out_stride=out.stride(0))
    return dict(q=q, out=out, lse=lse, work=work, desc=d, need=need, window=window)


def run_attn(L, plan, x, st=None):
    return L.gcuda_op_paged_attn(ref(plan.kv), ref(plan.batch), ref(x["desc"]), x["work"].data_ptr(), x["need"],
                                 stream() if st is None else st)


def check_attn(plan, x, act, heads, skip=()):
    """out and lse of every row within what the kernel's arithmetic rounds: a score is a float sum of dim products (its
    error at most (dim + 10) 2^-24 of the sum of their sizes; queries are held to 22 bits of their row's largest: 2^-21
    more of max |q| sum |k|, which that sum over sqrt(dim) bounds loosely), a weight's relative error twice the scores'
    and a few roundings; weights are rounded to the cache's 16-bit type (f16 for int8) unless the activations are
    float (then to twice its bits); sums are float."""
    hd = plan.dim
    scale = float(x["desc"].scale)
    out, lse = x["out"].cpu().double(), x["lse"].cpu().double()
    weight_step = HALF_STEP["bf16" if plan.cache == "bf16" else "f16"]
    if act == "f32":
        weight_step = 2 * weight_step**2
    seen_rows = set()
    for s, n in enumerate(plan.rows):
        if s in skip:
            seen_rows.update(range(int(plan.start_host[s]), int(plan.start_host[s]) + n))
            continue
        keys, values = plan.values(s, 0, plan.lengths[s]), plan.values(s, 1, plan.lengths[s])
        for i in range(n):
            row = int(plan.start_host[s]) + i
            seen_rows.add(row)
            end = max(0, plan.lengths[s] - n + i + 1)
            begin = max(0, end - x["window"]) if x["window"] else 0
            q = x["q"][row, :, :hd].cpu().double()
            o, l, size, mag = bh.attend(q, keys[begin:end], values[begin:end], scale)
            if end == 0:
                assert (out[row] == 0).all() and (lse[row] == -math.inf).all()
                continue
            visible = end - begin
            kmax = keys[begin:end].abs().sum(-1).amax()
            ds = mag * (hd + 10) * 2.0**-24 + 2.0**-21 * q.abs().amax(-1) * kmax * abs(scale)
            tol = size * (2 * ds[:, None] + weight_step + (visible + 40) * 2.0**-24) + HALF_STEP[act] * 1.01 * o.abs() + 1e-30
            if act == "f16":
                tol = tol + 2.0**-25   # (f16's smallest step, halved)
            assert ((out[row] - o).abs() <= tol).all(), (s, i, float(((out[row] - o).abs() / tol).max()))
            assert ((lse[row] - l).abs() <= ds + (visible + 40) * 2.0**-24 + 2.0**-22 * l.abs()).all(), (s, i)
    for row in range(plan.n_rows):
        if row not in seen_rows:
            assert (out[row] == 55).all() and (lse[row] == 55).all(), row


ATTN = [
    # act, cache, heads, kv heads, dim, page, rows, lengths, window, head major, gate
    ("f32", "i8", 16, 2, 256, 64, [1], [1], 0, False, False),
    ("f32", "i8", 16, 2, 256, 64, [1], [1000], 0, False, True),
    ("f32", "i8", 16, 2, 256, 64, [5, 0, 5, 2], [300, 0, 5, 65], 0, False, False),
    ("bf16", "i8", 16, 2, 256, 16, [1] * 9, [1, 2, 15, 16, 17, 31, 33, 64, 257], 0, True, False),
    ("f16", "i8", 8, 8, 128, 7, [1, 3], [100, 3], 0, False, False),
    ("bf16", "bf16", 16, 2, 256, 64, [1, 1], [129, 640], 0, False, False),
    ("f16", "f16", 12, 4, 64, 16, [8, 1, 4], [50, 63, 4], 0, True, False),
    ("f32", "bf16", 5, 1, 128, 100, [2, 1], [199, 301], 0, False, False),
    ("f32", "f16", 4, 2, 64, 1, [1, 2], [40, 41], 0, False, False),
    ("bf16", "f16", 32, 1, 128, 32, [1, 3], [90, 33], 0, False, False),
    ("f16", "bf16", 4, 4, 256, 32, [8], [8], 0, False, False),
    ("f32", "i8", 10, 2, 64, 64, [4, 1, 1], [500, 70, 9], 33, False, False),
    ("bf16", "bf16", 8, 2, 128, 16, [8, 2, 1], [300, 5, 1], 1, False, False),
    ("f16", "f16", 40, 2, 128, 16, [7, 1], [260, 31], 100, False, False),
    ("f32", "i8", 8, 1, 256, 64, [3, 2, 4], [1, 2, 0], 0, False, False),   # rows before the first position
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(len(c[6])) + "-w" + str(c[8]))
def test_attend(L, case):
    act, cache, heads, nkv, hd, page, rows, lengths, window, head_major, gate = case
    plan = Plan(rows, lengths, page, nkv, hd, cache, seed=11, head_major=head_major, spare=3)
    plan.randomize(13)
    x = attn_inputs(L, plan, act, heads, 17, window, gate=gate)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, heads)
    again = x["out"].clone()
    x["work"].random_(0, 256)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    assert torch.equal(again, x["out"])   # the same bits, whatever the scratch held


@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "i8"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("q_scale", [1e-3, 30.0])
def test_attend_flat_and_peaked(L, act, cache, q_scale):
    """Scores nearly equal over a long cache, and one position far above the rest."""
    plan = Plan([1, 2], [3000, 1029], 64, 2, 128, cache, seed=1)
    plan.randomize(2)
    x = attn_inputs(L, plan, act, 8, 3, q_scale=q_scale)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 8)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attend_scales_far_apart(L, act):
    """int8 rows whose scales span many powers of two: a tiny value row with nearly all the weight, zero rows, and large
    rows with none."""
    plan = Plan([1, 1], [130, 40], 16, 2, 64, "i8", seed=4)
    codes, sc = plan.randomize(5)
    sc[:, 1] *= torch.pow(2.0, torch.randint(-60, 20, sc[:, 1].shape, generator=torch.Generator().manual_seed(6)).float())
    sc[:, 0, ::5] = 0.0
    plan.scale_view.copy_(sc)
    x = attn_inputs(L, plan, act, 4, 7, q_scale=3.0)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 4)


@pytest.mark.parametrize("cache", ["i8", "bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attend_unseen_values_do_not_matter(L, cache, bad):
    """Rows that do not see the batch's later positions, whatever those hold; rows that do see them give no number."""
    plan = Plan([4, 3], [37, 3], 16, 2, 64, cache, seed=8)
    plan.randomize(9)
    x = attn_inputs(L, plan, "bf16", 8, 10)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    clean = x["out"].clone()
    for s in (0, 1):
        p = plan.lengths[s] - 1   # only the last row of each sequence sees it
        at = (int(plan.table_host[s, p // 16]), slice(None), p % 16)
        (plan.scale_view if cache == "i8" else plan.view)[at] = bad
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    for s in (0, 1):
        r0, n = int(plan.start_host[s]), plan.rows[s]
        assert torch.equal(x["out"][r0:r0 + n - 1], clean[r0:r0 + n - 1])
        assert not torch.isfinite(x["out"][r0 + n - 1].float()).any()


def test_attend_bad_plans(L):
    """A page out of range inside a sequence: its positions not attended to; a bad sequence left out; both flagged."""
    for bad in (-1, 10**6):
        plan = Plan([1, 2, 1], [50, 20, 70], 16, 2, 64, "i8", seed=2)
        plan.randomize(3)
        plan.table[0, 1] = bad           # positions 16 .. 31
        plan.length[1] = 10**6
        x = attn_inputs(L, plan, "f32", 4, 5)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        assert L.gcuda_op_status(1) == 2
        assert (x["out"][1:3] == 55).all() and (x["lse"][1:3] == 55).all()
        check_attn(plan, x, "f32", 4, skip=(0, 1))
        keys, values = (torch.cat([plan.values(0, w, 16), plan.values(0, w, 50)[32:]]) for w in (0, 1))
        o, l, _, _ = bh.attend(x["q"][0].cpu().double(), keys, values, 1 / 8)
        assert (x["out"][0].cpu().double() - o).abs().max() <= 1e-5 * values.abs().max()
        assert (x["lse"][0].cpu().double() - l).abs().max() <= 1e-4
    for starts in ([0, 9, 2, 3], [-2, 1, 2, 3], [0, 1, 2, 99]):
        plan = Plan([1, 1, 1], [5, 6, 7], 16, 2, 64, "bf16", seed=2)
        plan.randomize(3)
        plan.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        x = attn_inputs(L, plan, "bf16", 4, 5)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        assert L.gcuda_op_status(1) == 2
        assert torch.isfinite(x["out"].float()).all()


def test_attend_beyond_32_bits(L):
    """A cache of more than 2^32 values, the sequence on its first and last pages."""
    page, hd, nkv = 4096, 256, 2
    n_pages = 1030
    plan = Plan([1], [2 * page], page, nkv, hd, "i8", extra_pages=0)
    buf = torch.zeros(n_pages, 2, page, nkv, hd, dtype=torch.int8, device="cuda")
    sc = torch.full((n_pages, 2, page, nkv), math.nan, device="cuda")
    table = torch.tensor([[n_pages - 1, 0]], dtype=torch.int32, device="cuda")
    for p in (0, n_pages - 1):
        buf[p] = torch.randint(-127, 128, buf[p].shape, device="cuda", dtype=torch.int8)
        sc[p] = 0.01
    plan.view, plan.scale_view, plan.table_host = buf[[0, n_pages - 1]], sc[[0, n_pages - 1]], np.array([[1, 0]])
    plan.kv.k, plan.kv.v, plan.kv.n_pages = buf[:, 0].data_ptr(), buf[:, 1].data_ptr(), n_pages
    plan.kv.k_scale, plan.kv.v_scale = sc[:, 0].data_ptr(), sc[:, 1].data_ptr()
    plan.batch.pages = table.data_ptr()
    x = attn_inputs(L, plan, "bf16", 4, 1)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, "bf16", 4)


def test_attend_many_sequences(L):
    """More sequences than CTAs, lengths of every residue; their rows do not depend on their neighbours."""
    rng = np.random.default_rng(0)
    lengths = [int(v) for v in rng.integers(0, 90, 700)]
    plan = Plan([1] * 700, lengths, 16, 1, 64, "f16", seed=3)
    plan.randomize(4)
    x = attn_inputs(L, plan, "f16", 2, 5)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    out = x["out"].cpu().double()
    q = x["q"].cpu().double()
    view = plan.view.cpu().double()
    for s, n in enumerate(lengths):
        if n == 0:
            assert (out[s] == 0).all()
            continue
        flat = view[plan.table_host[s, : -(-n // 16)]].transpose(1, 2).flatten(0, 1)[:n]   # [position][2][head][dim]
        o, _, size, _ = bh.attend(q[s], flat[:, 0], flat[:, 1], 1 / 8)
        assert ((out[s] - o).abs() <= size * (2.0**-11 + 1e-5) + 2.0**-11 * 1.01 * o.abs() + 2.0**-25).all(), s


# ---------------------------------------------------------------------------------------------------- adjust ----
def rules_for(S, k, V, seed, history=20, biases=6, masks=True, mask_row=True, penalties=(True, True, True), pad=True):
    rng = np.random.default_rng(seed)
    h = {}
    h["history"] = rng.integers(0, min(V, 40), (S, history)).astype(np.int32)   # (many duplicates)
    if pad and history > 2:
        h["history"][:, 1] = -1
    h["history_len"] = rng.integers(0, history + 1, S).astype(np.int32)
    h["drafts"] = rng.integers(0, min(V, 40), (S, max(k, 1))).astype(np.int32)
    if k > 1:
        h["drafts"][0, 1] = -1
        h["drafts"][-1, 1] = h["drafts"][-1, 0]   # the same token twice
    h["repetition"], h["frequency"], h["presence"] = ((1 + rng.random(S)).astype(np.float32), rng.random(S).astype(np.float32),
                                                     rng.standard_normal(S).astype(np.float32))
    h["bias_id"] = rng.integers(0, min(V, 8), (S, max(biases, 1))).astype(np.int32)   # (duplicates)
    h["bias"] = (3 * rng.standard_normal((S, max(biases, 1)))).astype(np.float32)
    if biases > 3:
        h["bias"][0, 3] = -np.inf
        h["bias_id"][-1, 2] = -5
    h["bias_len"] = rng.integers(0, biases + 1, S).astype(np.int32)
    rows = S * (k + 1)
    M = rows if not mask_row else max(1, rows // 2)
    h["mask"] = rng.integers(0, 2**32, (M, (V + 31) // 32 + 2), dtype=np.uint64).astype(np.uint32)   # (a wide stride)
    h["mask"][0] = 0   # a row that allows nothing
    h["mask_row"] = rng.integers(-1, M, rows).astype(np.int32)
    t = {n: torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda() for n, a in h.items()}
    r = gb.LogitRules(history=t["history"].data_ptr() if history else None,
                      history_len=t["history_len"].data_ptr() if history else None, history_stride=history,
                      drafts=t["drafts"].data_ptr() if k else None, bias_stride=max(biases, 1), mask_stride=h["mask"].shape[1])
    for n, on in zip(("repetition", "frequency", "presence"), penalties):
        if on:
            setattr(r, n, t[n].data_ptr())
    if biases:
        r.bias_id, r.bias, r.bias_len = t["bias_id"].data_ptr(), t["bias"].data_ptr(), t["bias_len"].data_ptr()
    if masks:
        r.mask, r.n_masks = t["mask"].data_ptr(), M
        if mask_row:
            r.mask_row = t["mask_row"].data_ptr()
    return h, t, r


def check_adjust(x, got, act, S, k, V, h, history, biases, masks, mask_row, penalties):
    """Within five float roundings of the steps' sizes, and the type's; everywhere else the same bits."""
    for s in range(S):
        rule = tuple(float(h[n][s]) if on else d for n, on, d in zip(("repetition", "frequency", "presence"), penalties, (1.0, 0.0, 0.0)))
        for i in range(k + 1):
            row = s * (k + 1) + i
            m = None
            if masks:
                j = int(h["mask_row"][row]) if mask_row else row
                m = h["mask"][j] if j >= 0 else None
            n = int(h["history_len"][s]) if history else 0
            nb = int(h["bias_len"][s]) if biases else 0
            bias = list(zip(h["bias_id"][s, :nb].tolist(), h["bias"][s, :nb].tolist()))
            before = x[row].double().numpy()
            want = bh.adjust_row(before, V, h["history"][s, :n].tolist() if history else [], h["drafts"][s, :i].tolist(), rule, bias, m)
            g = got[row].double().numpy()
            assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want)), row
            fin = np.isfinite(want)
            with np.errstate(invalid="ignore"):
                big = np.abs(before) * 2 + 12 + (n + k) * abs(rule[1])
            assert (np.abs(g - want)[fin] <= (5 * 2.0**-24 * big + HALF_STEP[act] * 1.01 * np.abs(want) + 1e-7 * (act == "f16"))[fin]).all(), row
            touched = set(h["history"][s, :n].tolist() if history else []) | set(h["drafts"][s, :i].tolist()) | {t for t, _ in bias}
            same = fin & ~np.isin(np.arange(V), list(touched))
            assert np.array_equal(g[same], before[same])


ADJUST = [
    # act, S, k, V, history, biases, masks, mask_row, penalties
    ("f32", 1, 0, 1, 3, 2, True, True, (True, True, True)),
    ("f32", 3, 4, 1000, 20, 6, True, True, (True, True, True)),
    ("f32", 2, 0, 9001, 300, 0, False, False, (True, False, False)),
    ("bf16", 2, 8, 257, 40, 6, True, False, (False, True, False)),
    ("f16", 4, 1, 4099, 0, 5, True, True, (False, False, True)),
    ("bf16", 5, 0, 20011, 1, 1, False, False, (False, False, False)),
    ("f32", 2, 3, 8192, 50, 6, True, True, (True, True, True)),
    ("f16", 1, 2, 33, 5, 0, True, True, (True, True, False)),
]


@pytest.mark.parametrize("case", ADJUST, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("layout", ["apart", "in place", "strided"])
def test_adjust(L, case, layout):
    act, S, k, V, history, biases, masks, mask_row, penalties = case
    h, t, r = rules_for(S, k, V, 5, history, biases, masks, mask_row, penalties)
    rows = S * (k + 1)
    g = torch.Generator().manual_seed(3)
    x = (4 * torch.randn(rows, V, generator=g)).to(TORCH[act])
    if V > 30:
        x[0, 20], x[0, 21], x[-1, 22] = math.inf, -math.inf, math.nan
        x[0, 23] = 0.0
    pad_in, pad_out = (5, 3) if layout == "strided" else (0, 0)
    src = torch.full((rows, V + pad_in), 9.0, dtype=TORCH[act], device="cuda")
    src[:, :V] = x.cuda()
    dst = src if layout == "in place" else torch.full((rows, V + pad_out), 7.0, dtype=TORCH[act], device="cuda")
    assert L.gcuda_op_logits_adjust(ref(r), src.data_ptr(), dst.data_ptr(), CODE[act], S, k, V, src.stride(0), dst.stride(0),
                                    stream()) == 0
    torch.cuda.synchronize()
    got = dst.cpu()
    assert (got[:, V:] == 7.0).all()
    check_adjust(x, got[:, :V], act, S, k, V, h, history, biases, masks, mask_row, penalties)


def test_adjust_bad_ids(L):
    """Ids beyond the vocabulary and mask rows beyond the masks: left out, flagged; lengths beyond the lists: clamped."""
    S, k, V = 2, 2, 500
    x = torch.randn(S * (k + 1), V)
    for what, flag in (("history", 4), ("drafts", 4), ("bias_id", 4), ("history_len", 2), ("bias_len", 2), ("mask_row", 2)):
        h, t, r = rules_for(S, k, V, 9, pad=False)
        h["history_len"][:], h["bias_len"][:] = 20, 6
        t["history_len"].fill_(20), t["bias_len"].fill_(6)
        if what in ("history", "drafts", "bias_id"):
            t[what][1, 0] = V
            h[what][1, 0] = -1
        elif what == "mask_row":
            t[what][3] = r.n_masks
            h[what][3] = -1
        else:
            t[what][1] = 10**6
        out = torch.empty(S * (k + 1), V, device="cuda")
        src = x.cuda()
        assert L.gcuda_op_logits_adjust(ref(r), src.data_ptr(), out.data_ptr(), gb.F32, S, k, V, V, V, stream()) == 0
        torch.cuda.synchronize()
        assert L.gcuda_op_status(1) == flag, what
        check_adjust(x, out.cpu(), "f32", S, k, V, h, 20, 6, True, True, (True, True, True))


# ----------------------------------------------------------------------------------------------- used together ----
def test_a_step_of_many_conversations(L):
    """Verify steps as a serving loop runs them, captured once: the rows appended, their attention, a projection to
    logits, the rules, the greedy acceptance; replayed as the conversations grow, each step against the definitions."""
    S, k, heads, nkv, hd, page, V = 3, 2, 8, 2, 64, 16, 200
    T = k + 1
    final = [60, 21, 33]
    plan = Plan([T] * S, final, page, nkv, hd, "i8", seed=21)
    lengths = [30, T, 17]
    x = append_inputs(plan, "f32", heads, 32, True, 22)
    y = attn_inputs(L, plan, "f32", heads, 23)
    y["desc"].q, y["desc"].q_stride, y["desc"].q_head_stride = x["q_out"].data_ptr(), x["q_out"].stride(0), hd
    h, t, r = rules_for(S, k, V, 24, history=8, biases=3)
    proj = torch.randn(heads * hd, V, generator=torch.Generator().manual_seed(25)).cuda()
    logits = torch.empty(S * T, V, device="cuda")
    adjusted = torch.empty_like(logits)
    scratch = torch.zeros(S * T, dtype=torch.int64, device="cuda")
    accepted, nxt = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")

    def step():
        st = stream()
        assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), st) == 0
        assert run_attn(L, plan, y, st) == 0
        torch.mm(y["out"].view(S * T, heads * hd), proj, out=logits)
        assert L.gcuda_op_logits_adjust(ref(r), logits.data_ptr(), adjusted.data_ptr(), gb.F32, S, k, V, V, V, st) == 0
        assert L.gcuda_op_greedy_verify(adjusted.data_ptr(), t["drafts"].data_ptr(), S, k, V, scratch.data_ptr(),
                                        accepted.data_ptr(), nxt.data_ptr(), st) == 0

    # (the cache's earlier positions: rows of an earlier step)
    plan.randomize(26)
    plan.scale_view.nan_to_num_(0.01)
    plan.length.copy_(torch.tensor(lengths, dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for grow in ([0, 0, 0], [2, 3, 1], [3, 1, 2]):
        lengths = [a + b for a, b in zip(lengths, grow)]
        plan.lengths = lengths
        plan.length.copy_(torch.tensor(lengths, dtype=torch.int32))
        x["k"].normal_()
        x["q"].normal_()
        before, sc = plan.view.cpu().clone(), plan.scale_view.cpu().clone()
        x["q_out"].fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        check_append(plan, x, "f32", heads, True, before, sc)
        y["q"] = x["q_out"]
        check_attn(plan, y, "f32", heads)
        check_adjust(logits.cpu(), adjusted.cpu(), "f32", S, k, V, h, 8, 3, True, True, (True, True, True))
        rows = adjusted.cpu().view(S, T, V)
        for s in range(S):
            best = [int(v) for v in rows[s].argmax(-1)]
            n = 0
            while n < k and best[n] == int(h["drafts"][s, n]):
                n += 1
            assert int(accepted[s]) == n and int(nxt[s]) == best[n]


def test_two_calls_at_once(L):
    """Two streams with a scratch of their own give what they give one after the other."""
    plans, xs, want = [], [], []
    for i in range(2):
        p = Plan([2] * 40, [400 + 13 * j for j in range(40)], 32, 2, 128, "bf16", seed=i)
        p.randomize(i + 5)
        x = attn_inputs(L, p, "bf16", 8, i + 9)
        assert run_attn(L, p, x) == 0
        torch.cuda.synchronize()
        plans.append(p), xs.append(x), want.append(x["out"].clone())
        x["out"].zero_()
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for p, x, s in zip(plans, xs, sides):
            assert run_attn(L, p, x, s.cuda_stream) == 0
    torch.cuda.synchronize()
    for x, w in zip(xs, want):
        assert torch.equal(x["out"], w)


FIRST_CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import batch_helpers as bh
from geode_b200 import batch as gb, cuda_lib
from test_batch_gpu import attn_inputs, run_attn, check_attn
L = cuda_lib()
plan = bh.Plan([1, 2], [40, 70], 16, 2, 64, "i8")
plan.randomize(1)
x = attn_inputs(L, plan, "f32", 4, 2)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    assert run_attn(L, plan, x) == 0
graph.replay()
torch.cuda.synchronize()
check_attn(plan, x, "f32", 4)
print("captured")
"""


def test_first_call_of_a_process_captured(L):
    """The library's first call on a device may be one that is captured."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALL.format(root=os.path.dirname(here), tests=here)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
