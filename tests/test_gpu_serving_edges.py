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


# ---- attention ---------------------------------------------------------------


def pool(torch, ctx, kind, n_pages, ps, hk, D, seed):
    """A cache of one layer with random rows, and its values in 64 bits
    [n_pages, n_kv_head, page_size, head_dim]."""
    from llm_mojo_b200.serving import PagedKVCache

    c = PagedKVCache(ctx, kind, 1, n_pages, ps, hk, D)
    g = torch.Generator(device="cuda").manual_seed(seed)
    val = []
    for t, s in ((c.k, c.ks), (c.v, c.vs)):
        if s is None:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            val.append(t[0].double())
        else:
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda", dtype=torch.int8))
            s.copy_(torch.rand(s.shape, generator=g, device="cuda") * 0.03 + 0.002)
            val.append(t[0].double() * s[0].double()[..., None])
    return c, *val


def check_attend(torch, c, k, v, q, table, lens, weighted):
    """attend of every sequence against 64 bits, a table row after another.
    Tolerance, of the values' largest: a score's rounding errors, one per
    product and sum, add up like a random walk, four deviations of which
    shift the weights by as much, relatively; the sums over positions
    likewise; 16 roundings for exponentials, scales and the join."""
    n, H, D = q.shape
    hk, ps, top = c.n_kv_head, c.page_size, int(lens.max())
    w = torch.rand(n, hk, top, device="cuda") if weighted else None
    wo = torch.full_like(w, -7.0) if weighted else None
    out = c.attend(0, q, table, lens, top, weights=w, weights_out=wo)
    pos = torch.arange(top, device="cuda")
    for b, length in enumerate(lens.tolist()):
        page = table[b][pos[:length] // ps].long()
        ok = (page >= 0) & (page < c.n_pages)
        at = pos[:length][ok]
        if not at.numel():
            assert torch.count_nonzero(out[b]) == 0
            assert not weighted or torch.equal(wo[b], w[b])
            continue
        kb, vb = k[page[ok], :, at % ps], v[page[ok], :, at % ps]  # [positions, kv head, D]
        qb = q[b].double().view(hk, H // hk, D)
        p = torch.softmax(torch.einsum("hgd,lhd->hgl", qb, kb) / D ** 0.5, -1)
        smax = float(torch.einsum("hgd,lhd->hgl", qb.abs(), kb.abs()).max()) / D ** 0.5
        rel = 2.0 ** -23 * (4 * D ** 0.5 * smax + 4 * at.numel() ** 0.5 + 16)
        want = torch.einsum("hgl,lhd->hgd", p, vb).reshape(H, D)
        assert float((out[b].double() - want).abs().max()) <= rel * float(vb.abs().max()), b
        if weighted:
            add = w[b].double()
            add[:, at] += p.sum(1)
            assert float((wo[b].double() - add).abs().max()) <= rel * (H // hk) + 2.0 ** -23 * (H // hk + 1), b


@pytest.mark.parametrize("kind", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("n,hk,G,D,ps,top", [
    # one warp a CTA: more than 16 units (sequence, kv head, up to 8 query heads) an SM, up to 256 positions
    (256, 12, 1, 64, 16, 100),
    (256, 12, 8, 64, 5, 100),
    (208, 12, 1, 64, 5, 256),
    (304, 8, 1, 128, 16, 77),
    (304, 8, 3, 128, 7, 70),
    (304, 8, 11, 32, 16, 60),
    (304, 8, 6, 96, 48, 90),
    # two: more than 8
    (256, 12, 1, 64, 16, 300),
    (256, 12, 2, 64, 5, 300),
    (128, 12, 8, 64, 16, 300),
    (160, 8, 1, 32, 1, 500),
    (160, 8, 8, 96, 3, 280),
    (160, 8, 5, 128, 64, 290),
])
@pytest.mark.parametrize("weighted", [False, True])
def test_attend_full_batches(torch, ctx, kind, n, hk, G, D, ps, top, weighted):
    """Batches that fill the GPU with CTAs of one and of two warps, lengths
    from nothing on, a missing page here and there."""
    rng = np.random.default_rng(n + D + G)
    lens = rng.integers(0, top + 1, n)
    lens[:4] = top, 1, 0, min(top, 17)
    need = -(-lens // ps)
    n_pages = int(need.sum()) + 1
    table = np.full((n, need.max()), -1, dtype=np.int32)
    ids, at = rng.permutation(n_pages), 0
    for b, x in enumerate(need):
        table[b, :x] = ids[at: at + x]
        at += x
    table[5::9, 0] = -1
    table[7::9, -1] = n_pages
    c, k, v = pool(torch, ctx, kind, n_pages, ps, hk, D, 5)
    q = torch.randn(n, hk * G, D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda") * 1.5
    check_attend(torch, c, k, v, q, torch.from_numpy(table).cuda(), torch.from_numpy(lens.astype(np.int32)).cuda(),
                 weighted)
    c.free()


@pytest.mark.parametrize("kind", ["int8", "bf16", "f32"])
def test_attend_long_sums_are_not_biased(torch, ctx, kind):
    """Positive values with equal weights, 20000 positions in one chunk, of
    which a warp has 313 tiles of 16. A tile's product may truncate 16
    addends, 2^-24 of the largest, up to twice the mean, each: 2^-23 of the
    sum, twice for the terms; what else is rounded is rounded to nearest: on
    the average over all outputs 3 of 2^-23. An output alone: these, 16 for
    the join, and 313 roundings like a random walk."""
    n, hk, D, top, ps = 80, 12, 64, 20000, 16
    n_pages = top // ps
    c, _, _ = pool(torch, ctx, kind, n_pages, ps, hk, D, 3)
    g = torch.Generator(device="cuda").manual_seed(3)
    c.k.zero_()
    if kind == "int8":
        c.v.copy_(torch.randint(1, 128, c.v.shape, generator=g, device="cuda", dtype=torch.int8))
        c.vs.copy_(0.5 + 0.5 * torch.rand(c.vs.shape, generator=g, device="cuda"))
    else:
        c.v.copy_(0.1 + torch.rand(c.v.shape, generator=g, device="cuda"))
    order = torch.randperm(n_pages, generator=g, device="cuda")
    lens = [top - 7 * b for b in range(n)]
    out = c.attend(0, torch.ones(n, hk, D, device="cuda"), order.to(torch.int32)[None].expand(n, -1),
                   torch.tensor(lens, dtype=torch.int32, device="cuda"), top)
    v = c.v[0].double() if c.vs is None else c.v[0].double() * c.vs[0].double()[..., None]
    v = v[order].transpose(1, 2).reshape(top, hk, D)
    want = torch.stack([v[:x].mean(0) for x in lens])
    ulps = (out.double() - want) / want * 2.0 ** 23
    assert abs(float(ulps.mean())) <= 3
    assert float(ulps.abs().max()) <= 19 + (top / 64) ** 0.5
    c.free()


@pytest.mark.parametrize("kind", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("n,hk,G,D,ps,top", [(256, 12, 1, 64, 16, 9000), (80, 12, 1, 64, 24, 8500),
                                             (60, 12, 2, 32, 5, 4200), (80, 8, 5, 96, 32, 4500)])
def test_attend_chunks_of_several_runs(torch, ctx, kind, n, hk, G, D, ps, top):
    """So many sequences that a chunk is a whole sequence, longer than the
    4096 positions whose rows are looked up at a time; missing pages in the
    second run."""
    rng = np.random.default_rng(top)
    need = -(-top // ps)
    table = rng.permutation(need).astype(np.int32)
    table[4100 // ps], table[-1] = -1, need
    lens = rng.integers(4097, top + 1, n).astype(np.int32)
    lens[:5] = top, 4096, 4097, 0, 8192 if top > 8192 else 4098
    c, k, v = pool(torch, ctx, kind, need, ps, hk, D, 6)
    q = torch.randn(n, hk * G, D, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") * 1.5
    check_attend(torch, c, k, v, q, torch.from_numpy(table)[None].cuda().expand(n, -1), torch.from_numpy(lens).cuda(),
                 True)
    c.free()


# ---- eviction ----------------------------------------------------------------


@pytest.mark.parametrize("length", [48, 11])
def test_evict_writes_only_its_rows(torch, ctx, length):
    """Rows of weights inside a wider buffer: what lies between them, and
    after the last, stays."""
    from llm_mojo_b200 import _lib
    from llm_mojo_b200.serving import PagedKVCache

    c = PagedKVCache(ctx, "bf16", 1, 8, 16, 2, 64)
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    dst = torch.tensor([[4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    w = torch.rand(2, 48, device="cuda")
    wide = torch.full((4, 33), 7.0, device="cuda")  # two rows of 20
    kept, n = torch.zeros(2, 20, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _lib.lib().llmq_paged_evict(ctx.h, c.h, 0, 1, 1, table.data_ptr(), 3, 3, lens.data_ptr(), 48, w.data_ptr(),
                                       48, 20, 0, 0, dst.data_ptr(), 2, 2, kept.data_ptr(), wide.data_ptr(), 33,
                                       n.data_ptr()) == _lib.OK
    for h in range(2):
        keep = kept[h][kept[h] >= 0].long()
        assert keep.numel() == min(length, 20) == int(n[0])
        assert torch.equal(wide[h, : keep.numel()], w[h, keep]) and torch.count_nonzero(wide[h, keep.numel(): 20]) == 0
    assert torch.all(wide[:, 20:] == 7.0) and torch.all(wide[2:] == 7.0)
    c.free()


@pytest.mark.parametrize("kind", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("budget", [20, 60])  # below and above the lengths
def test_evict_refuses_positions_without_a_page(torch, ctx, kind, budget):
    """A sequence that would keep a position whose page is missing gets
    length -1, and attention gives zeros for it, not what the destination
    held; missing positions that are not kept do not matter."""
    c, k, v = pool(torch, ctx, kind, 20, 16, 2, 64, 4)
    for t in (c.k, c.v) if kind != "int8" else (c.ks, c.vs):
        t[0, 8:] = float("nan")  # the destinations
    table = torch.tensor([[0, -1, 2], [3, 4, 5], [0, 20, 2]], dtype=torch.int32, device="cuda")
    dst = torch.arange(8, 20, dtype=torch.int32, device="cuda").view(3, 4)
    lens = torch.tensor([48, 48, 48], dtype=torch.int32, device="cuda")
    w = torch.rand(1, 3, 2, 48, device="cuda") + 1.0
    w[:, 2, :, 16:32] = float("nan")
    kept, _, got = c.evict(table, lens, 48, w, budget, dst, sinks=2, recent=3)
    n = min(48, budget)
    assert got.tolist() == [-1, n, n if budget == 20 else -1]
    q = torch.randn(3, 4, 64, device="cuda")
    out = c.attend(0, q, dst, got, n)
    for b in range(3):
        if got[b] < 0:
            assert torch.count_nonzero(out[b]) == 0
            continue
        for h in range(4):
            at = kept[0, b, h // 2, :n].long()
            kb, vb = (x[table[b][at // 16].long(), h // 2, at % 16] for x in (k, v))
            p = torch.softmax(kb @ q[b, h].double() / 8, 0)
            smax = float((kb.abs() @ q[b, h].double().abs()).max()) / 8
            tol = 2.0 ** -23 * (32 * smax + 4 * n ** 0.5 + 16) * float(vb.abs().max())
            assert float((out[b, h].double() - p @ vb).abs().max()) <= tol
    c.free()


# ---- views -------------------------------------------------------------------


def test_weights_of_one_head_or_sequence(torch, ctx):
    """The stride of a dimension of one says nothing: rows of a wider buffer
    with such a dimension put in are taken; rows that are not evenly spaced,
    or overlap, are not."""
    from llm_mojo_b200._lib import LlmqError

    c, k, v = pool(torch, ctx, "bf16", 8, 16, 1, 64, 3)
    q = torch.randn(2, 3, 64, device="cuda")
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 33], dtype=torch.int32, device="cuda")
    want = torch.zeros(2, 1, 48, device="cuda")
    c.attend(0, q, table, lens, 48, weights_out=want)
    wide = torch.zeros(2, 60, device="cuda")
    rows = wide[:, :48].unsqueeze(1)
    assert rows.stride() == (60, 48, 1)
    c.attend(0, q, table, lens, 48, weights=rows, weights_out=rows)
    assert torch.equal(rows, want) and torch.count_nonzero(wide[:, 48:]) == 0
    one = torch.zeros(48, device="cuda").as_strided((1, 1, 48), (5, 7, 1))
    c.attend(0, q[:1], table[:1], lens[:1], 48, weights_out=one)
    assert torch.equal(one, want[:1])
    dst = torch.tensor([[6], [7]], dtype=torch.int32, device="cuda")
    kept, w, n = c.evict(table, lens, 48, want[None], 16, dst)
    kept2, w2, n2 = c.evict(table, lens, 48, rows[None], 16, dst)
    assert torch.equal(kept, kept2) and torch.equal(w, w2) and torch.equal(n, n2)
    with pytest.raises(LlmqError):
        c.attend(0, q, table, lens, 48, weights_out=torch.zeros(1, 1, 48, device="cuda").expand(2, 1, 48))
    two, _, _ = pool(torch, ctx, "bf16", 8, 16, 2, 64, 3)
    uneven = torch.zeros(2, 3, 48, device="cuda")[:, :2]
    with pytest.raises(ValueError):
        two.attend(0, torch.randn(2, 2, 64, device="cuda"), table, lens, 48, weights_out=uneven)
    with pytest.raises(ValueError):
        two.evict(table, lens, 48, uneven[None], 16, dst)
    c.free()
    two.free()


# ---- logits ------------------------------------------------------------------


@pytest.mark.parametrize("n,H", [(5, 700), (6, 700), (12, 5000), (30, 1), (256, 300)])
def test_rules_of_full_batches(torch, ctx, n, H):
    """1024, 2048 and 4096 logits a tile, the argmax by tickets (5 rows) and
    by a second launch (from 6 on), each rule at work, infinities among
    the logits, in place too."""
    from llm_mojo_b200.serving import process_logits

    V = 50257
    r = make_rules(V, n, H, n)
    x = (np.random.default_rng(n).standard_normal((n, V)) * 3).astype(np.float32)
    x[0, 40000], x[1, :: 7], x[-1, 5] = np.inf, np.float32(2.5), -np.inf
    r["mask"][-1] = 0  # nothing is left
    r["mask"][-2] = 0
    r["mask"][-2, 50256 // 32] = 1 << (50256 % 32)  # the last token alone
    want, best = rules_reference(x, **r)
    assert best[-1] == -1 and best[-2] == 50256
    logits = torch.from_numpy(x).cuda()
    out, top = process_logits(ctx, logits, to_rules(torch, r))
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(top.cpu().numpy(), best)
    process_logits(ctx, logits, to_rules(torch, r), out=logits, argmax=top.fill_(-9))
    assert torch.equal(out, logits) and np.array_equal(top.cpu().numpy(), best)
