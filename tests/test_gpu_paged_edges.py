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


def test_step_checks_its_tensors(torch, model):
    """Types, shapes, strides and devices that the step would misread, and
    weights that it would write past the end of, are refused."""
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.serving import PagedKVCache

    bt = Batch(model, 2, 1)
    c = PagedKVCache(model.ctx, "int8", 2, 2, 16, 12, 64)
    zero, table, logits = i32(torch, [0, 0]), i32(torch, [[0], [1]]), torch.zeros(2, 50257, device="cuda")
    wide = torch.zeros(2, 50260, device="cuda")
    w = torch.zeros(2, 2, 12, 4, device="cuda")
    ok = dict(tokens=zero, positions=zero, slots=zero, table=table, lens=zero + 1, max_len=4, logits=logits, weights=w)
    for bad in (dict(tokens=zero.long()), dict(positions=zero.float()), dict(slots=zero[:1]), dict(lens=zero.long()),
                dict(lens=zero.cpu()), dict(table=table.long()), dict(table=table[:1]), dict(table=table[0]),
                dict(logits=logits.double()), dict(logits=logits[:, 1:]), dict(logits=wide[:, :50257]),
                dict(weights=w[:1]), dict(weights=w[:, :1]), dict(weights=w[:, :, :11]), dict(weights=w[..., :3]),
                dict(weights=w.double()), dict(weights=w.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            bt.paged_step(c, **dict(ok, **bad))
    bt.paged_step(c, **ok)
    c.free()
    bt.free()


def test_step_is_ordered_with_the_current_stream(torch, model):
    """On a context with a stream of its own the step takes what torch's
    current stream has written, and the caller reads what it wrote."""
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.serving import PagedKVCache

    bt = Batch(model, 1, 1)
    c = PagedKVCache(model.ctx, "f32", 2, 1, 16, 12, 64)
    assert not model.ctx.on_torch_stream()
    zero, table = i32(torch, [0]), i32(torch, [[0]])
    want = torch.zeros(1, 50257, device="cuda")
    bt.paged_step(c, i32(torch, [777]), zero, zero, table, zero + 1, 1, want)
    big = torch.randn(8192, 8192, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        tok, logits = zero.clone(), torch.zeros(1, 50257, device="cuda")
        for _ in range(30):
            big @ big
        tok.fill_(777)
        bt.paged_step(c, tok, zero, zero, table, zero + 1, 1, logits)
        got = logits.clone()
    side.synchronize()
    assert torch.equal(got, want)
    c.free()
    bt.free()


def test_generator_refuses_what_it_cannot_run(torch, model):
    """When it is made, not at the first cut."""
    from llm_mojo_b200.paged_generate import PagedGenerator

    for bad in (dict(max_len=64, limit=100, budget=70), dict(max_len=64, limit=100, budget=64),
                dict(limit=32, budget=16), dict(limit=32, budget=16, recent=10, sinks=7), dict(limit=32, budget=32),
                dict(limit=32), dict(limit=32, budget=16, recent=8, sinks=-1), dict(page_size=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            PagedGenerator(model, 2, **bad)
    gen = PagedGenerator(model, 1, max_len=40, limit=100, budget=39, recent=30, sinks=9)
    for prompt in ([-1], [5, 50257]):
        with pytest.raises(ValueError):
            gen.generate([prompt], 2)
    with pytest.raises(ValueError):
        gen.generate([[1]], -1)
    assert gen.generate([[1]], 0) == [[]]
    assert len(gen.generate([[1]], 60)[0]) == 60  # cut at 40, 20 times
    gen.free()


def test_neighbours_do_not_change_a_sampled_text(torch, model):
    from llm_mojo_b200.paged_generate import PagedGenerator

    gen = PagedGenerator(model, 3, max_len=64)
    prompts = [[5, 6], list(range(100, 120)), [7]]
    all_three = gen.generate(prompts, 8, temperature=0.9)
    assert gen.generate(prompts[:1], 8, temperature=0.9) == all_three[:1]
    assert gen.generate(prompts[:2], 8, temperature=0.9) == all_three[:2]
    assert gen.generate([[1] * 30, *prompts[1:]], 8, temperature=0.9)[1:] == all_three[1:]
    assert gen.generate([[1], [2], prompts[0]], 8, temperature=0.9, seed=1335)[2] == all_three[0]
    assert gen.generate(prompts, 8, temperature=0.9, seed=1) != all_three
    gen.free()


@pytest.mark.parametrize("bounded", [False, True])
def test_a_text_that_is_done_holds_nothing(torch, model, monkeypatch, bounded):
    """It takes no pages beyond its own, gives them back, grows no further for
    `allowed`, and its end changes nothing for the others."""
    from llm_mojo_b200 import paged_generate

    taken, pools = [], []

    class Pool(paged_generate.PagePool):
        def __init__(self, n):
            super().__init__(n)
            pools.append(self)

        def take(self, n):
            taken.append(n)
            return super().take(n)

    monkeypatch.setattr(paged_generate, "PagePool", Pool)
    kw = dict(limit=24, budget=12, sinks=2, recent=4) if bounded else dict(max_len=64)
    gen = paged_generate.PagedGenerator(model, 2, page_size=8, **kw)
    prompts = [[1], list(range(40))]
    seen = []
    out = gen.generate(prompts, 5, allowed=lambda at, texts: seen.append([len(t) for t in texts]))
    assert [max(x) for x in zip(*seen)] == [6, 44]  # the whole of the shorter, the longer before its last token
    if not bounded:
        assert sum(taken) == -(-5 // 8) + -(-44 // 8)
    assert len(pools[0].free) == gen.cache.n_pages - (3 if bounded else 6)  # the longer's last 20 positions, or all 44
    for b in range(2):
        assert gen.generate([prompts[b]], 5) == [out[b]]
    gen.free()


def test_the_pool_is_the_only_cache(torch, model):
    """A generator's memory for cache positions is its pool; its batch has no
    contiguous caches beside it, and generates nothing by itself."""
    from llm_mojo_b200._lib import ERR_INVALID, LlmqError
    from llm_mojo_b200.model import Batch
    from llm_mojo_b200.paged_generate import PagedGenerator

    def used(make):
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        x = make()
        torch.cuda.synchronize()
        return x, before - torch.cuda.mem_get_info()[0]

    Batch(model, 1, 1).free()  # the kernels' own memory
    n, position = 256, 2 * 12 * 2 * (64 + 4)  # layers, heads, keys and values with their scales
    whole, with_caches = used(lambda: Batch(model, n, 1))
    whole.free()
    torch.cuda.empty_cache()
    gen, got = used(lambda: PagedGenerator(model, n, max_len=16))
    # the pool holds 16 positions a sequence, the caches the model's 128; 2 MB a buffer at most
    assert got <= with_caches + n * (16 - 128) * position + (8 << 20)
    with pytest.raises(LlmqError) as e:
        gen.batch.generate([[1]], 1)
    assert e.value.status == ERR_INVALID
    assert len(gen.generate([[1]], 3)[0]) == 3
    gen.free()
    for bad in (-1, 129):
        with pytest.raises(LlmqError):
            Batch(model, 1, bad)


@pytest.mark.parametrize("dtype,head", [("int8-ch-a16", "int8"), ("int4-g32-a16", "same"), ("int4-g32-a16", "int8")])
def test_tiles_are_built_where_they_are_read(torch, dtype, head):
    """A model's first batch builds the lane-mode GEMM's copies of the weights
    that it takes: BLOCKED int4 layers and the per-channel int8 head, rows to
    a multiple of 128."""
    from llm_mojo_b200 import synth
    from llm_mojo_b200.model import Batch, Model
    from llm_mojo_b200.tensor import Context

    def used(make):
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        x = make()
        torch.cuda.synchronize()
        return x, before - torch.cuda.mem_get_info()[0]

    ctx = Context(0)
    layers = 4
    tensors = synth.gpt2_random_init(0, n_layer=layers)
    first = Model(ctx, tensors, n_layer=layers, max_t=32)
    Batch(first, 16, 1).free()  # the kernels' own memory
    first.free()
    m = Model(ctx, tensors, dtype, head, n_layer=layers, max_t=32)
    a, first = used(lambda: Batch(m, 16, 1))
    b, second = used(lambda: Batch(m, 16, 1))
    copies = [n * 768 * 768 for n in (3, 1, 4, 4)] * layers * (dtype[:4] == "int4") + [50304 * 768] * (head == "int8")
    page = 2 << 20
    assert sum(copies) <= first - second <= sum(-(-x // page) * page for x in copies), (first, second)
    a.free()
    b.free()
    m.free()
    ctx.close()
