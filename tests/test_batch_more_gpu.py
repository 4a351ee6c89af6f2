"""The paged operators over every kernel shape - head dims, cache and activation types, blocks of 8, 16 and 40 query rows, one
and two blocks - and their bounds: nothing outside the scratch, the rows and the cache's own positions is written; memory
that is not the current device's is refused."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from geode_b200 import batch as gb  # noqa: E402
from geode_b200 import cuda_lib  # noqa: E402
from batch_helpers import Plan, ref  # noqa: E402
from test_batch_gpu import append_inputs, attn_inputs, check_append, check_attn, run_attn, stream  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return cuda_lib()


@pytest.mark.parametrize("tokens", [1, 2, 5, 8])   # of 8 query heads a key head: 8, 16, 40 and 64 rows
@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache", ["i8", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_shape(L, dim, cache, act, tokens):
    plan = Plan([tokens, 1, tokens], [130 + tokens, 17, tokens], 24, 2, dim, cache, seed=dim + tokens, spare=1)
    plan.randomize(dim + 1)
    x = attn_inputs(L, plan, act, 16, dim + 2)
    guard = torch.full((x["need"] + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    x["work"] = guard
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, act, 16)
    assert (guard[x["need"]:] == 0xAB).all()
    assert L.gcuda_op_status(1) == 0


@pytest.mark.parametrize("cache,tokens", [("i8", 1), ("i8", 5), ("bf16", 2), ("f16", 8)])
def test_cut_items(L, cache, tokens):
    """One long sequence: its items are cut among all CTAs, and their parts joined; the same bits run after run."""
    plan = Plan([tokens], [6001], 16, 1, 128, cache, seed=3)
    plan.randomize(4)
    x = attn_inputs(L, plan, "f32", 8, 5, window=0)
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    check_attn(plan, x, "f32", 8)
    first = x["out"].clone()
    for _ in range(5):
        x["out"].zero_()
        x["work"].random_(0, 256)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        assert torch.equal(first, x["out"])


@pytest.mark.parametrize("cache", ["i8", "f16"])
def test_no_lse_and_strided_out(L, cache):
    plan = Plan([3, 1], [50, 9], 16, 2, 64, cache, seed=6)
    plan.randomize(7)
    x = attn_inputs(L, plan, "f16", 4, 8)
    assert run_attn(L, plan, x) == 0
    wide = torch.full((plan.n_rows, 4 * 64 + 5), 55.0, dtype=torch.float16, device="cuda")
    x["desc"].out, x["desc"].out_stride, x["desc"].lse = wide.data_ptr(), wide.stride(0), None
    lse = x["lse"].clone()
    assert run_attn(L, plan, x) == 0
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :256].reshape(plan.n_rows, 4, 64), x["out"]) and (wide[:, 256:] == 55).all()
    assert torch.equal(lse, x["lse"])


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache", ["i8", "bf16", "f16"])
@pytest.mark.parametrize("dim,rope", [(64, 64), (64, 8), (128, 36), (256, 256), (256, 250)])
def test_append_every_shape(L, dim, rope, cache, act):
    plan = Plan([1, 6, 0, 2], [1, 30, 0, 49], 12, 3, dim, cache, seed=dim + rope, head_major=rope % 16 == 0, spare=2)
    before, scales = plan.randomize(rope)
    x = append_inputs(plan, act, 6, rope, rope != 64, 3, gate=dim == 128)
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    check_append(plan, x, act, 6, rope != 64, before, scales)
    assert L.gcuda_op_status(1) == 0


@pytest.mark.parametrize("window", [2**31 - 1, 2**30, 2**30 - 1, 300, 7])
def test_windows(L, window):
    """Windows beyond any sequence see everything; the difference of a position and a window stays in 32 bits."""
    plan = Plan([8, 2, 3], [200, 2, 0], 16, 2, 64, "i8", seed=9)
    plan.randomize(10)
    for tokens in (2, 16):   # (1 and 8 query heads a key head: both kernels)
        x = attn_inputs(L, plan, "f32", tokens, 11, window=window)
        assert run_attn(L, plan, x) == 0
        torch.cuda.synchronize()
        check_attn(plan, x, "f32", tokens)


def test_append_many_sequences(L):
    """More sequences than one round of the search looks at, some without rows."""
    rows = [(i * 7) % 3 for i in range(1500)]
    plan = Plan(rows, [r + i % 5 for i, r in enumerate(rows)], 4, 1, 64, "i8", seed=1)
    before, scales = plan.randomize(2)
    x = append_inputs(plan, "bf16", 1, 16, True, 3)
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
    torch.cuda.synchronize()
    check_append(plan, x, "bf16", 1, True, before, scales)


def test_ties_of_the_codes(L):
    """Values at exactly half a step round to the even code: 63.5 of amax / 2 and every odd multiple of amax / 254."""
    plan = Plan([1], [1], 4, 1, 64, "i8")
    x = append_inputs(plan, "f32", 0, 0, False, 1)
    v = torch.arange(64, dtype=torch.float32) * 4 + 1
    v[63] = 254.0          # codes 127 v / 254 = v / 2: every one of them a half
    for sign in (1.0, -1.0):
        x["v"][0] = sign * v.cuda()
        x["k"][0, :64] = sign * v.cuda()
        assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(x["desc"]), stream()) == 0
        torch.cuda.synchronize()
        want = torch.round(sign * v.double() / 2).to(torch.int8)   # (to even)
        page = plan.table_host[0, 0]
        assert torch.equal(plan.view[page, 0, 0, 0].cpu(), want) and torch.equal(plan.view[page, 1, 0, 0].cpu(), want)


def test_memory_elsewhere_is_refused(L):
    plan = Plan([1], [5], 16, 2, 64, "bf16")
    x = attn_inputs(L, plan, "bf16", 4, 1)
    host = torch.zeros(1 << 16).numpy()   # (kept alive: ordinary host memory)
    x["desc"].out = host.ctypes.data // 256 * 256 + 256
    assert run_attn(L, plan, x) == -1
    y = append_inputs(plan, "bf16", 4, 64, False, 1)
    y["desc"].k = host.ctypes.data // 256 * 256 + 256
    assert L.gcuda_op_paged_append(ref(plan.kv), ref(plan.batch), ref(y["desc"]), stream()) == -1
    r = gb.LogitRules()
    d = torch.zeros(100, device="cuda")
    assert L.gcuda_op_logits_adjust(ref(r), d.data_ptr(), host.ctypes.data // 256 * 256 + 256, gb.F32, 1, 0, 100, 100, 100, stream()) == -1
    # no rules at all: a copy
    out = torch.ones(100, device="cuda")
    assert L.gcuda_op_logits_adjust(ref(r), d.data_ptr(), out.data_ptr(), gb.F32, 1, 0, 100, 100, 100, stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, d)


def test_adjust_replayed_and_beside_another(L):
    """A captured adjustment follows its lists from replay to replay, beside another on a second stream."""
    S, k, V = 3, 1, 5000
    src = torch.randn(S * 2, V, device="cuda")
    dst, dst2 = torch.empty_like(src), torch.empty_like(src)
    hist = torch.randint(0, V, (S, 50), dtype=torch.int32, device="cuda")
    n = torch.zeros(S, dtype=torch.int32, device="cuda")
    pen = torch.full((S,), 0.5, device="cuda")
    r = gb.LogitRules(history=hist.data_ptr(), history_len=n.data_ptr(), history_stride=50, presence=pen.data_ptr())
    call = lambda out, st: L.gcuda_op_logits_adjust(C.byref(r), src.data_ptr(), out.data_ptr(), gb.F32, S, k, V, V, V, st)  # noqa: E731
    assert call(dst, stream()) == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(dst, stream()) == 0
    side = torch.cuda.Stream()
    for length in (0, 1, 50, 7):
        n.fill_(length)
        torch.cuda.synchronize()
        graph.replay()
        assert call(dst2, side.cuda_stream) == 0
        torch.cuda.synchronize()
        want = src.clone()
        for s in range(S):
            for t in set(hist[s, :length].tolist()):
                want[2 * s:2 * s + 2, t] -= 0.5
        assert torch.equal(dst, want) and torch.equal(dst2, want)
