"""The decode loop over a paged cache: the model's logits, eviction, rules."""

import numpy as np
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


@pytest.mark.parametrize("kind,B", [("int8", 3), ("int8", 20), ("f32", 2), ("bf16", 2)])
def test_paged_step_logits(torch, model, kind, B):
    """Each sequence's logits after every token of a 40-token text are the
    model's own. The int8 cache holds the same codes, so only roundings of
    the attention differ, and what the 16-bit activations make of them: 1e-2
    of the largest logit, the bound of the act16 model against the
    reference. The model's cache is int8: the float caches differ by its
    quantization as well, 2 codes in 254 of a value's range at most, and get
    the same bound."""
    from llm_mojo_b200 import synth
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.serving import PagedKVCache

    T = 40
    ids = synth.uniform_ids(B * T, 5).reshape(B, T)
    want = torch.zeros(50257, device="cuda")
    ref = np.zeros((B, 3, 50257), dtype=np.float32)
    for b in range(B):
        for t in range(T):
            model.forward([int(ids[b, t])], t, want)
            if t in (0, 17, T - 1):
                torch.cuda.synchronize()
                ref[b, (0, 17, T - 1).index(t)] = want.cpu().numpy()
    before = model.ctx.stream
    model.ctx.use_torch_stream()
    bt = Batch(model, B, 1)
    cache = PagedKVCache(model.ctx, kind, 2, B * 5, 8, 12, 64)
    table = torch.from_numpy(np.random.default_rng(1).permutation(B * 5).astype(np.int32).reshape(B, 5)).cuda()
    toks = torch.from_numpy(ids.astype(np.int32)).cuda()
    logits = torch.zeros(B, 50257, device="cuda")
    weights = torch.zeros(2, B, 12, T, device="cuda")
    try:
        for t in range(T):
            pos = torch.full((B,), t, dtype=torch.int32, device="cuda")
            bt.paged_step(cache, toks[:, t].contiguous(), pos, pos, table, pos + 1, t + 1, logits, weights=None)
            if t in (0, 17, T - 1):
                got = logits.cpu().numpy()
                r = ref[:, (0, 17, T - 1).index(t)]
                assert np.abs(got - r).max() <= 1e-2 * np.abs(r).max(), t
        # with weights: the same logits, and each row's weights add up to one per head and step
        for t in range(T):
            pos = torch.full((B,), t, dtype=torch.int32, device="cuda")
            bt.paged_step(cache, toks[:, t].contiguous(), pos, pos, table, pos + 1, T, logits, weights=weights)
        assert np.array_equal(logits.cpu().numpy(), got)
        assert float((weights.double().sum(-1) - T).abs().max()) < T * 40 * 2.0 ** -22
    finally:
        bt.free()
        cache.free()
        model.ctx.sync()
        model.ctx.set_stream(before)


def test_generator_equals_batch(torch, model):
    """Greedy ids over the paged cache against the batched decode's."""
    from llm_mojo_b200 import synth
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.paged_generate import PagedGenerator

    prompts = synth.uniform_ids(4 * 6, 9).reshape(4, 6)
    gen = PagedGenerator(model, 4, max_len=64)
    got = gen.generate([list(map(int, p)) for p in prompts], 12)
    gen.free()
    bt = Batch(model, 4, 8)
    want = bt.generate(prompts, 12)
    bt.free()
    assert np.array_equal(np.array(got), want)


def test_generator_ragged_and_bounded(torch, model):
    """Prompts of different lengths generate what each does alone; a bounded
    cache runs past its limit, keeps its budget and returns its pages."""
    from llm_mojo_b200.paged_generate import PagedGenerator

    prompts = [[50256], [11, 22, 33, 44, 55], list(range(1000, 1021))]
    gen = PagedGenerator(model, 3, max_len=64)
    together = gen.generate(prompts, 8)
    assert together == [gen.generate([p], 8)[0] for p in prompts]
    gen.free()
    small = PagedGenerator(model, 3, limit=24, budget=12, sinks=2, recent=4, page_size=8)
    a = small.generate(prompts, 50)
    assert a == small.generate(prompts, 50) and all(len(x) == 50 for x in a)
    # before the first cut nothing differs
    assert [x[:2] for x in a] == [x[:2] for x in together]
    small.free()


def test_generator_rules(torch, model):
    """A mask allows only its tokens; a bias forces one; a penalty ends a
    repetition; where nothing is allowed, EOT."""
    from llm_mojo_b200.paged_generate import PagedGenerator

    gen = PagedGenerator(model, 2, max_len=64)
    prompts = [[5, 6], [7]]
    even = torch.zeros(2, 50257, dtype=torch.bool)
    even[:, ::2] = True
    for temperature in (0.0, 0.9):
        out = gen.generate(prompts, 10, allowed=lambda at, texts: even, temperature=temperature)
        assert all(t % 2 == 0 for x in out for t in x)
    assert gen.generate(prompts, 5, bias={777: 1e6, 12: -1.0}) == [[777] * 5] * 2
    out = gen.generate(prompts, 20, frequency=1e4)
    assert all(len(set(x)) == 20 for x in out)
    none = torch.zeros(2, 50257, dtype=torch.bool)
    assert gen.generate(prompts, 3, allowed=lambda at, texts: none, temperature=0.5) == [[50256] * 3] * 2
    with pytest.raises(ValueError):
        gen.generate([[]], 3)
    with pytest.raises(ValueError):
        gen.generate([[1]] * 3, 3)
    gen.free()


def test_paged_step_refusals(torch, model):
    from llm_mojo_b200._lib import ERR_INVALID, LlmqError
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.serving import PagedKVCache

    bt = Batch(model, 2, 1)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    logits = torch.zeros(1, 50257, device="cuda")
    for shape in ((1, 1, 16, 12, 64), (2, 1, 16, 6, 64), (2, 1, 16, 12, 128)):
        c = PagedKVCache(model.ctx, "int8", *shape)
        with pytest.raises(LlmqError) as e:
            bt.paged_step(c, one, one, one, table, one + 1, 1, logits)
        assert e.value.status == ERR_INVALID
        c.free()
    c = PagedKVCache(model.ctx, "int8", 2, 1, 16, 12, 64)
    three = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(LlmqError):
        bt.paged_step(c, three, three, three, table.expand(3, -1), three + 1, 1, torch.zeros(3, 50257, device="cuda"))
    c.free()
    bt.free()
