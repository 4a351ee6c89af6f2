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
