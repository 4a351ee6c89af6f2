"""A handle's set-up copies and its kernels keep one order: everything goes through the handle's own streams, which neither wait
for the default stream nor are waited for by it."""
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from geode_b200 import synth  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_copies_on_the_default_stream():
    """A copy or a zeroing on the default stream has no order with the handle's streams: the zeroing of a new buffer could land
    behind the copy into it, and the step read a table of zeros."""
    with open(os.path.join(ROOT, "geode_b200", "csrc", "backend.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert re.findall(r"\bcudaMem(?:cpy|set|cpy2D|set2D)\(", code) == []
    assert len(re.findall(r"cudaStreamCreateWithFlags\(&g->\w+, cudaStreamNonBlocking\)", code)) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("arch", ["qwen35", "qwen35moe"])
def test_setup_while_the_device_is_busy(tmp_path, arch):
    """Handles opened and used at once while another stream keeps every SM busy: the first step's logits are the oracle's."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import oracle_py as op
    from geode_b200.backend import Backend

    shape = synth.tiny_shape(arch, n_layers=4, ctx=64)
    synth.write_pack(str(tmp_path), shape, seed=11)
    ora = op.Oracle(str(tmp_path))
    toks = np.random.default_rng(5).integers(0, shape.vocab, 5)
    ref = ora.forward(ora.new_state(shape.ctx), toks, logits=True, hidden=False)["logits"]
    span = ref.max(axis=-1) - ref.min(axis=-1)
    a = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            for _ in range(20):
                b = a @ a
        be = Backend(str(tmp_path), context=shape.ctx, max_tokens=5)
        got, _ = be.verify(toks, logits=True, hidden=False)
        be.close()
        assert (np.abs(got - ref).max(axis=-1) <= 1e-2 * span).all()
    torch.cuda.synchronize()
    del b
