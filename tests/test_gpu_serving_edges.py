"""The serving operators where their kernels' paths change: tiles, warps and
chunks by size, rows of every alignment, buffers wider than their rows."""

import numpy as np
import pytest
from test_gpu_serving import make_rules, rules_reference, to_rules

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def ctx(torch):
    from llm_mojo_b200 import build
    from llm_mojo_b200.tensor import Context

    build.build()
    c = Context(0)
    c.use_torch_stream()
    yield c
    c.close()


# 1024 logits a tile for few rows, 2048 and 4096 for more
@pytest.mark.parametrize("V,n", [(1021, 2), (1022, 2), (1023, 2), (5119, 1), (2046, 150), (2047, 150), (4094, 150),
                                 (4095, 150)])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_rules_last_tile(torch, ctx, V, n, shift):
    """Vocabularies that end one or two logits before a tile does: depending
    on a row's alignment there is a last tile without a token, to which no
    token of the history belongs."""
    from llm_mojo_b200.serving import process_logits

    r = make_rules(V, n, 60, V + shift)
    x = (np.random.default_rng(V).standard_normal((n, V + 5)) * 3).astype(np.float32)
    out, top = process_logits(ctx, torch.from_numpy(x).cuda()[:, shift: shift + V], to_rules(torch, r))
    want, best = rules_reference(np.ascontiguousarray(x[:, shift: shift + V]), **r)
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(top.cpu().numpy(), best)
