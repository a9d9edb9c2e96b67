"""The decode step and the generator over a paged cache: what they refuse, and
what a sequence's neighbours may not change."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def model(torch):
    from llm_mojo_b200 import build, synth
    from llm_mojo_b200.model import Model
    from llm_mojo_b200.tensor import Context

    build.build()
    ctx = Context(0)
    m = Model(ctx, synth.gpt2_random_init(0, n_layer=2), n_layer=2, max_t=128)
    yield m
    m.free()
    ctx.close()


def i32(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bad", [dict(max_len=0), dict(max_len=2**31 - 1), dict(cols=0)])
def test_refused_step_changes_nothing(torch, model, bad):
    """A step whose attention would be refused stores nothing either."""
    from llm_mojo_b200 import _lib
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.serving import PagedKVCache

    bt = Batch(model, 1, 1)
    c = PagedKVCache(model.ctx, "f32", 2, 1, 16, 12, 64)
    c.k.fill_(5.0), c.v.fill_(5.0)
    zero, one, logits = i32(torch, [0]), i32(torch, [1]), torch.zeros(1, 50257, device="cuda")
    torch.cuda.synchronize()
    at = dict(dict(max_len=1, cols=1), **bad)
    assert _lib.lib().llmq_batch_paged_step(
        model.ctx.h, bt.h, c.h, 1, zero.data_ptr(), zero.data_ptr(), zero.data_ptr(), zero.data_ptr(), 1, at["cols"],
        one.data_ptr(), at["max_len"], None, 0, logits.data_ptr()) == _lib.ERR_INVALID
    model.ctx.sync()
    assert torch.all(c.k == 5.0) and torch.all(c.v == 5.0) and torch.count_nonzero(logits) == 0
    c.free()
    bt.free()
