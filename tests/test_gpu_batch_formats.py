"""Batched decode of models whose layers are per-channel int8, or whose head
has the layers' format: the formats that the lane-mode GEMM does not take
there run on the CUDA cores at every batch size."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,head", [("int8-ch-a16", "int8"), ("int4-g32-a16", "same"), ("int8-ch-a16", "same")])
def test_batch_and_paged_step(dtype, head):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from llm_mojo_b200 import build, synth
    from llm_mojo_b200.model import Batch, Model
    from llm_mojo_b200.serving import PagedKVCache
    from llm_mojo_b200.tensor import Context

    build.build()
    B, P, steps = 17, 4, 5
    ctx = Context(0)
    m = Model(ctx, synth.gpt2_random_init(0, n_layer=1), dtype, head, n_layer=1, max_t=32)
    prompts = synth.uniform_ids(B * P, 3).reshape(B, P)
    bt = Batch(m, B, P)
    got = bt.generate(prompts, steps)
    single = np.array([m.generate(list(prompts[b]), steps) for b in range(B)])
    assert np.array_equal(got, single)
    want = torch.zeros(50257, device="cuda")
    with ctx.torch_stream():
        cache = PagedKVCache(ctx, "int8", 1, B, 16, 12, 64)
        table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
        toks = torch.from_numpy(prompts.astype(np.int32)).cuda()
        logits = torch.zeros(B, 50257, device="cuda")
        for t in range(P):
            pos = torch.full((B,), t, dtype=torch.int32, device="cuda")
            bt.paged_step(cache, toks[:, t].contiguous(), pos, pos, table, pos + 1, t + 1, logits)
    for b in (0, 9, 16):
        for t in range(P):
            m.forward([int(prompts[b, t])], t, want)
        ctx.sync()
        torch.cuda.synchronize()
        # roundings of the attention and what the 16-bit activations make of them
        assert float((logits[b] - want).abs().max()) <= 1e-2 * float(want.abs().max()), b
    cache.free()
    bt.free()
    m.free()
    ctx.close()
