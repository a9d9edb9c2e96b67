"""The serving operators (paged store, paged attention of one new token,
eviction by accumulated weight, rules on logits) against plain definitions:
attention in 64 bits, everything else exactly."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PAGED = ("int8", "bf16", "f32")


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


def make_cache(torch, ctx, kind, layers, n_pages, ps, hk, d, seed, garbage=False):
    """A cache of random rows; with garbage, NaN and infinities everywhere
    (the caller writes the rows that count)."""
    from llm_mojo_b200.serving import PagedKVCache

    c = PagedKVCache(ctx, kind, layers, n_pages, ps, hk, d)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):
        if kind == "int8":
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda", dtype=torch.int8))
        else:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    if kind == "int8":
        for t in (c.ks, c.vs):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda") * 0.03 + 0.002)
    return c


def values(c, name, layer):
    """float64 values of the pool's layer [n_pages, n_kv_head, ps, d]."""
    x = getattr(c, name)[layer].double()
    s = getattr(c, name + "s")
    return x if s is None else x * s[layer].double()[..., None]


def make_table(torch, lens, ps, seed, first=0, extra=0):
    need = [-(-n // ps) for n in lens]
    ids = np.random.default_rng(seed).permutation(sum(need) + extra) + first
    t = np.full((len(lens), max(1, max(need))), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(t).cuda(), sum(need) + extra


def reference(torch, c, layer, q, table, lens, scale, drop=None):
    """out, the softmax weights per kv head, and the tolerance of each
    sequence. `drop` leaves one position out (a planted mistake)."""
    k, v = values(c, "k", layer), values(c, "v", layer)
    n, H, D = q.shape
    G, ps = H // c.n_kv_head, c.page_size
    out = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    ws, tol = [], []
    tab = table.cpu().numpy()
    for b in range(n):
        pos = [j for j in range(lens[b]) if 0 <= tab[b, j // ps] < c.n_pages and j != drop]
        w = torch.zeros(c.n_kv_head, max(1, lens[b]), dtype=torch.float64, device="cuda")
        t = 0.0
        if pos:
            pg, sl = torch.tensor([tab[b, j // ps] for j in pos]).long().cuda(), torch.tensor([j % ps for j in pos]).cuda()
            kb, vb = k[pg, :, sl], v[pg, :, sl]  # [len, hk, d]
            for h in range(H):
                qq = q[b, h].double()
                s = kb[:, h // G] @ qq * scale
                p = torch.softmax(s, 0)
                out[b, h] = p @ vb[:, h // G]
                w[h // G, torch.tensor(pos).cuda()] += p
                # a score's rounding errors, one per product and sum, add up
                # like a random walk: four deviations of it shift the weights
                # by as much, relatively; the sums over positions likewise;
                # 16 roundings for exponentials, scales and the join
                smax = float((kb[:, h // G].abs() @ qq.abs()).max() * scale)
                r = 2.0 ** -23 * (4 * math.sqrt(D) * smax + 4 * math.sqrt(len(pos)) + 16)
                t = max(t, r)
        ws.append(w)
        tol.append((t, float(v.nan_to_num(0, 0, 0).abs().max()) if pos else 0.0))
    return out, ws, tol


SHAPES = [
    # head_dim, kv heads, queries per kv head, page size, lengths
    (64, 12, 1, 16, [1, 15, 16, 17, 0, 130, 255]),
    (64, 2, 3, 20, [1023, 7, 512, 64]),
    (128, 2, 4, 64, [700, 1, 129]),
    (128, 1, 8, 5, [33, 2, 61]),
    (32, 3, 11, 16, [100, 48]),
    (96, 2, 2, 1, [37, 1, 5]),
    (96, 1, 6, 48, [311, 48, 49]),
    (64, 1, 1, 128, [9001]),
    (32, 1, 1, 7, [1]),
]


@pytest.mark.parametrize("kind", PAGED)
@pytest.mark.parametrize("D,hk,G,ps,lens", SHAPES)
@pytest.mark.parametrize("weighted", [False, True])
def test_attend_matches_64_bits(torch, ctx, kind, D, hk, G, ps, lens, weighted):
    table, n_pages = make_table(torch, lens, ps, 1, extra=2)
    c = make_cache(torch, ctx, kind, 2, n_pages, ps, hk, D, 5)
    n, top = len(lens), max(lens)
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randn(n, hk * G, D, generator=g, device="cuda") * 1.5
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    win = torch.rand(n, hk, top + 3, generator=g, device="cuda") if weighted else None
    wout = torch.full_like(win, -7.0) if weighted else None
    out = c.attend(1, q, table, ln, top, weights=win, weights_out=wout)
    again = c.attend(1, q, table, ln, top)
    assert torch.equal(out, again)  # with weights or without, the same bits
    ref, ws, tol = reference(torch, c, 1, q, table, lens, 1 / math.sqrt(D))
    for b in range(n):
        rel, vmax = tol[b]
        assert float((out[b].double() - ref[b]).abs().max()) <= rel * vmax, (b, lens[b])
        if weighted:
            want = win[b].double().clone()
            want[:, : lens[b]] += ws[b][:, : lens[b]]
            err = (wout[b, :, :top].double() - want[:, :top]).abs().max()
            assert float(err) <= rel * G + 2.0 ** -23 * (G + 1), b
            assert float(wout[b, :, top:].max()) == -7.0  # past max_len nothing is written


@pytest.mark.parametrize("kind", PAGED)
def test_attend_tolerance_finds_a_lost_position(torch, ctx, kind):
    """The tolerance of test_attend_matches_64_bits is below what the loss of
    any position of more than average weight, of 255, changes."""
    lens = [255]
    table, n_pages = make_table(torch, lens, 16, 2)
    c = make_cache(torch, ctx, kind, 1, n_pages, 16, 1, 64, 6)
    q = torch.randn(1, 1, 64, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    ref, ws, tol = reference(torch, c, 0, q, table, lens, 0.125)
    heavy = (ws[0][0] > 1 / 255).nonzero()[:, 0].tolist()
    assert len(heavy) > 10
    for drop in heavy:
        bad, _, _ = reference(torch, c, 0, q, table, lens, 0.125, drop=drop)
        assert float((bad - ref).abs().max()) > tol[0][0] * tol[0][1]


@pytest.mark.parametrize("kind", PAGED)
@pytest.mark.parametrize("ps", [16, 12])
def test_attend_ignores_what_is_masked(torch, ctx, kind, ps):
    """Missing pages, and NaN and infinities past the length and in pages
    that no sequence has, leave the result as it is without them."""
    lens, D, hk, G = [90, 31, 200], 64, 2, 2
    table, n_pages = make_table(torch, lens, ps, 3, extra=3)
    table[0, 2] = -1
    table[2, 5] = n_pages  # outside the pool
    table[2, 0] = -5
    c = make_cache(torch, ctx, kind, 1, n_pages, ps, hk, D, 9)
    q = torch.randn(3, hk * G, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    w1, w2 = torch.zeros(3, hk, 200, device="cuda"), torch.zeros(3, hk, 200, device="cuda")
    clean = c.attend(0, q, table, ln, 200, weights_out=w1)
    ref, ws, tol = reference(torch, c, 0, q, table, lens, 0.125)
    used = torch.zeros(n_pages, ps, dtype=torch.bool)
    tab = table.cpu().numpy()
    for b, n in enumerate(lens):
        for j in range(n):
            if 0 <= tab[b, j // ps] < n_pages:
                used[tab[b, j // ps], j % ps] = True
    junk = ~used.cuda()[:, None, :].expand(n_pages, hk, ps)
    for name in ("k", "v"):
        if kind == "int8":
            getattr(c, name + "s")[0][junk] = float("nan")
            getattr(c, name)[0][junk] = -128
        else:
            getattr(c, name)[0][junk] = float("nan")
            getattr(c, name)[0][junk.logical_and(torch.rand(junk.shape, device="cuda") < 0.5)] = float("inf")
    dirty = c.attend(0, q, table, ln, 200, weights_out=w2)
    assert torch.equal(clean, dirty) and torch.equal(w1, w2)
    for b in range(3):
        assert float((clean[b].double() - ref[b]).abs().max()) <= tol[b][0] * tol[b][1]
    assert torch.count_nonzero(w1[0, :, 2 * ps:3 * ps]) == 0


@pytest.mark.parametrize("kind", PAGED)
def test_attend_of_nothing_is_zero(torch, ctx, kind):
    c = make_cache(torch, ctx, kind, 1, 4, 16, 2, 64, 1)
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 64, device="cuda")
    out = torch.full((3, 4, 64), 5.0, device="cuda")
    w = torch.full((3, 2, 40), 2.0, device="cuda")
    lens = torch.tensor([0, 20, -3], dtype=torch.int32, device="cuda")
    c.attend(0, q, table, lens, 40, out=out, weights=w, weights_out=w)
    assert torch.count_nonzero(out) == 0 and torch.all(w == 2.0)


@pytest.mark.parametrize("kind", PAGED)
def test_attend_lengths_are_cut(torch, ctx, kind):
    """To max_len and to what the table holds."""
    table, n_pages = make_table(torch, [64, 64], 16, 4)
    c = make_cache(torch, ctx, kind, 1, n_pages, 16, 1, 64, 2)
    q = torch.randn(2, 1, 64, device="cuda")
    big = torch.tensor([1000, 2**31 - 1], dtype=torch.int32, device="cuda")
    for top, want in ((37, 37), (5000, 64)):
        a = c.attend(0, q, table, big, top)
        ref, _, tol = reference(torch, c, 0, q, table, [want, want], 0.125)
        for b in range(2):
            assert float((a[b].double() - ref[b]).abs().max()) <= tol[b][0] * tol[b][1]


@pytest.mark.parametrize("kind", PAGED)
@pytest.mark.parametrize("gain", [60.0, 1e-30, 0.0])
def test_attend_extreme_scores(torch, ctx, kind, gain):
    """Scores far apart (one position takes all), denormal and all equal."""
    lens = [300, 17]
    table, n_pages = make_table(torch, lens, 32, 5)
    c = make_cache(torch, ctx, kind, 1, n_pages, 32, 2, 64, 3)
    q = torch.randn(2, 4, 64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") * gain
    out = c.attend(0, q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 300)
    ref, _, tol = reference(torch, c, 0, q, table, lens, 0.125)
    for b in range(2):
        assert float((out[b].double() - ref[b]).abs().max()) <= tol[b][0] * tol[b][1]


def test_attend_int8_scales_of_any_size(torch, ctx):
    """Value scales over thirty orders of magnitude, zero among them."""
    lens = [150]
    table, n_pages = make_table(torch, lens, 16, 6)
    c = make_cache(torch, ctx, "int8", 1, n_pages, 16, 1, 64, 4)
    g = torch.Generator(device="cuda").manual_seed(3)
    c.vs.copy_(10.0 ** (torch.rand(c.vs.shape, generator=g, device="cuda") * 30 - 25))
    c.vs[0, :, :, 3] = 0.0
    q = torch.randn(1, 1, 64, generator=g, device="cuda")
    out = c.attend(0, q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 150)
    ref, _, tol = reference(torch, c, 0, q, table, lens, 0.125)
    assert float((out.double() - ref).abs().max()) <= tol[0][0] * tol[0][1]
    c.vs.mul_(1e-20)
    out = c.attend(0, q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 150)
    ref, _, tol = reference(torch, c, 0, q, table, lens, 0.125)
    assert float((out.double() - ref).abs().max()) <= tol[0][0] * tol[0][1]


@pytest.mark.parametrize("kind", PAGED)
def test_attend_views_and_streams(torch, ctx, kind):
    """Strided queries, outputs and tables; the context's own stream; a side
    stream of torch: the same bits as the plain call."""
    from llm_mojo_b200.tensor import Context

    lens = [77, 200, 5]
    table, n_pages = make_table(torch, lens, 16, 7)
    c = make_cache(torch, ctx, kind, 1, n_pages, 16, 2, 64, 5)
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(3, 3 * 4 * 64 + 1, generator=g, device="cuda")
    q = qkv[:, 1: 257].unflatten(1, (4, 64))  # rows and starts that are not 16-byte aligned
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = c.attend(0, q.contiguous(), table, ln, 200)
    wide = torch.full((3, table.shape[1] + 5), 10**6, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    buf = torch.zeros(3, 6, 64, device="cuda")
    got = c.attend(0, q, wide[:, : table.shape[1]], ln, 200, out=buf[:, 1:5])
    assert torch.equal(got, want) and torch.count_nonzero(buf[:, 0]) == 0 and torch.count_nonzero(buf[:, 5]) == 0
    own = Context(0)
    try:
        c.ctx = own
        assert not own.on_torch_stream()
        assert torch.equal(c.attend(0, q, table, ln, 200), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q2 = q * 1.0
            own.use_torch_stream()
            w = torch.zeros(3, 2, 200, device="cuda")
            got = c.attend(0, q2, table, ln, 200, weights_out=w)
        side.synchronize()
        assert torch.equal(got, want)
    finally:
        c.ctx = ctx
        own.close()


def test_attend_shared_table_row(torch, ctx):
    """One table row broadcast to several sequences (a shared prefix)."""
    table, n_pages = make_table(torch, [120], 16, 8)
    c = make_cache(torch, ctx, "bf16", 1, n_pages, 16, 1, 64, 6)
    q = torch.randn(4, 2, 64, device="cuda")
    ln = torch.tensor([120, 3, 64, 100], dtype=torch.int32, device="cuda")
    got = c.attend(0, q, table.expand(4, -1), ln, 120)
    assert torch.equal(got, c.attend(0, q, table.repeat(4, 1), ln, 120))


def test_pool_offsets_past_32_bits(torch, ctx):
    """A pool of more than 2^32 bytes and 2^31 elements: rows at its end."""
    from llm_mojo_b200.serving import PagedKVCache

    ps, hk, D = 64, 8, 128
    n_pages = (1 << 31) // (ps * hk * D) + 40
    c = PagedKVCache(ctx, "bf16", 1, n_pages, ps, hk, D)
    g = torch.Generator(device="cuda").manual_seed(5)
    n = 100
    table = torch.tensor([[n_pages - 1, n_pages - 3, 0]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(n, hk, D, generator=g, device="cuda") for _ in range(2))
    c.store(0, k, v, torch.arange(n, dtype=torch.int32, device="cuda"), table,
            seq=torch.zeros(n, dtype=torch.int32, device="cuda"))
    for pos, page in ((0, n_pages - 1), (99, n_pages - 3)):
        assert torch.equal(c.k[0, page, :, pos % ps], k[pos].bfloat16())
    q = torch.randn(1, 2 * hk, D, generator=g, device="cuda")
    w = torch.zeros(1, hk, n, device="cuda")
    out = c.attend(0, q, table, torch.tensor([n], dtype=torch.int32, device="cuda"), n, weights_out=w)
    kd, vd = k.bfloat16().double(), v.bfloat16().double()
    for h in range(2 * hk):
        p = torch.softmax(kd[:, h // 2] @ q[0, h].double() / math.sqrt(D), 0)
        smax = float((kd[:, h // 2].abs() @ q[0, h].abs().double()).max() / math.sqrt(D))
        tol = 2.0 ** -23 * (4 * math.sqrt(D) * smax + 4 * math.sqrt(n) + 16) * float(vd.abs().max())
        assert float((out[0, h].double() - p @ vd[:, h // 2]).abs().max()) <= tol
    dst = torch.tensor([[n_pages - 2]], dtype=torch.int32, device="cuda")
    kept, _, lens = c.evict(table, torch.tensor([n], dtype=torch.int32, device="cuda"), n, w[None], 50, dst, recent=10)
    assert int(lens[0]) == 50
    for h in range(hk):
        assert torch.equal(c.k[0, n_pages - 2, h, :50], k[kept[0, 0, h].long(), h].bfloat16())
    c.free()


# ---- store -------------------------------------------------------------------


def quantize8(x):
    """QuantKV[8]: float32, codes half away from zero."""
    s = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    s[s == 0] = 1
    r = x * (np.float32(1) / s)[..., None]
    return np.trunc(r + np.copysign(np.float32(0.5), r)).astype(np.int8), s


@pytest.mark.parametrize("kind", PAGED)
@pytest.mark.parametrize("D,hk,ps", [(64, 12, 16), (32, 1, 5), (128, 3, 1), (96, 2, 64)])
def test_store(torch, ctx, kind, D, hk, ps):
    rng = np.random.default_rng(1)
    n = 45
    c = make_cache(torch, ctx, kind, 2, 40, ps, hk, D, 8)
    before = [t.clone() if t is not None else None for t in (c.k, c.v, c.ks, c.vs)]
    wide = rng.standard_normal((n, 3 * hk * D + 1)).astype(np.float32) * 3
    wide[4] = 0.0
    x = torch.from_numpy(wide).cuda()
    k, v = x[:, 1: 1 + hk * D].unflatten(1, (hk, D)), x[:, 1 + hk * D: 1 + 2 * hk * D].unflatten(1, (hk, D))
    table = rng.permutation(40).astype(np.int32).reshape(4, 10)
    table[3, 0], table[2, 0] = -1, 40
    slots = rng.permutation(4 * 10 * ps)[:n] if ps > 1 else np.arange(40).repeat(2)[:n]
    seq, pos = (slots // (10 * ps)).astype(np.int32), (slots % (10 * ps)).astype(np.int32)
    if ps == 1:
        pos[1::2] = -1  # the second of each pair is skipped
    pos[0] = -1
    pos[1] = 10 * ps  # past the table
    seq[2], seq[3] = 4, -1
    c.store(1, k, v, torch.from_numpy(pos).cuda(), torch.from_numpy(table).cuda(), seq=torch.from_numpy(seq).cuda())
    want = [t.cpu() if t is not None else None for t in before]
    for r in range(n):
        if not (0 <= seq[r] < 4 and 0 <= pos[r] < 10 * ps) or not 0 <= table[seq[r], pos[r] // ps] < 40:
            continue
        page, slot = table[seq[r], pos[r] // ps], pos[r] % ps
        for i, a in enumerate((k, v)):
            row = a[r].cpu().numpy()
            if kind == "int8":
                codes, s = quantize8(row)
                want[i][1, page, :, slot] = torch.from_numpy(codes)
                want[2 + i][1, page, :, slot] = torch.from_numpy(s)
            else:
                want[i][1, page, :, slot] = torch.from_numpy(row).to(want[i].dtype)
    for got, w in zip((c.k, c.v, c.ks, c.vs), want):
        assert w is None or torch.equal(got.cpu(), w)


def test_store_one_row_per_sequence(torch, ctx):
    c = make_cache(torch, ctx, "int8", 1, 3, 8, 2, 64, 9)
    k, v = torch.randn(2, 2, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    table = torch.tensor([[2], [0], [1]], dtype=torch.int32, device="cuda")
    c.store(0, k, v, torch.tensor([3, 7], dtype=torch.int32, device="cuda"), table)
    for b, (page, slot) in enumerate([(2, 3), (0, 7)]):
        codes, s = quantize8(k[b].cpu().numpy())
        assert np.array_equal(c.k[0, page, :, slot].cpu().numpy(), codes)
        assert np.array_equal(c.ks[0, page, :, slot].cpu().numpy(), s)


# ---- eviction ----------------------------------------------------------------


def evict_reference(w, length, budget, sinks, recent):
    if length <= budget:
        return np.arange(length)
    mid = np.arange(sinks, length - recent)
    key = np.where(np.isnan(w[mid]), -np.inf, w[mid])
    order = np.lexsort((mid, np.isnan(w[mid]), -key))
    return np.sort(np.concatenate([np.arange(sinks), mid[order[: budget - sinks - recent]],
                                   np.arange(length - recent, length)]))


@pytest.mark.parametrize("kind", PAGED)
@pytest.mark.parametrize("D,hk,ps,lens,budget,sinks,recent", [
    (64, 12, 16, [1024], 512, 4, 64),
    (64, 2, 20, [300, 40, 41, 0, 1], 40, 4, 11),
    (128, 1, 64, [2500, 2499], 1000, 0, 0),
    (32, 3, 7, [50, 9], 9, 4, 5),      # nothing to choose
    (96, 2, 1, [33, 70], 1, 0, 0),
    (64, 1, 16, [5000], 4999, 1, 1),
    (64, 1, 128, [70001], 333, 2, 100),
])
@pytest.mark.parametrize("dist", ["spread", "ties", "odd"])
def test_evict(torch, ctx, kind, D, hk, ps, lens, budget, sinks, recent, dist):
    rng = np.random.default_rng(2)
    layers, n, top = 2, len(lens), max(lens)
    table, used = make_table(torch, lens, ps, 11)
    dst, more = make_table(torch, [min(x, budget) for x in lens], ps, 12, first=used)
    c = make_cache(torch, ctx, kind, layers + 1, used + more, ps, hk, D, 13)
    before = [t.clone() if t is not None else None for t in (c.k, c.v, c.ks, c.vs)]
    w = rng.random((layers, n, hk, top + 2)).astype(np.float32) ** 6
    if dist == "ties":
        w = np.floor(w * 4).astype(np.float32)
    if dist == "odd":
        w = (w - 0.1).astype(np.float32)
        pick = rng.random(w.shape)
        w[pick < 0.1], w[(pick >= 0.1) & (pick < 0.15)], w[pick > 0.95] = np.nan, -0.0, 0.0
        w[(pick > 0.5) & (pick < 0.52)] = np.inf
    wt = torch.from_numpy(w).cuda()
    kept, wout, lout = c.evict(table, torch.tensor(lens, dtype=torch.int32, device="cuda"), top, wt, budget, dst,
                               sinks=sinks, recent=recent, layer0=1, n_layers=layers)
    kept, wout = kept.cpu().numpy(), wout.cpu().numpy()
    tab, dtab = table.cpu().numpy(), dst.cpu().numpy()
    want = [t.cpu() if t is not None else None for t in before]
    for layer in range(layers):
        for b in range(n):
            for h in range(hk):
                keep = evict_reference(w[layer, b, h, : lens[b]], lens[b], budget, sinks, recent)
                m = len(keep)
                assert np.array_equal(kept[layer, b, h, :m], keep), (layer, b, h)
                assert np.all(kept[layer, b, h, m:] == -1)
                assert np.array_equal(wout[layer, b, h, :m], w[layer, b, h, keep], equal_nan=True)
                assert np.all(wout[layer, b, h, m:] == 0)
                j = np.arange(m)
                for t, o in zip(want, before):
                    if t is not None and m:
                        t[1 + layer, dtab[b, j // ps], h, j % ps] = o.cpu()[1 + layer, tab[b, keep // ps], h, keep % ps]
    assert lout.cpu().tolist() == [min(x, budget) for x in lens]
    for got, wnt in zip((c.k, c.v, c.ks, c.vs), want):
        # only the rows of the destination pages change
        assert wnt is None or torch.equal(got.cpu(), wnt)


def test_evict_without_source_or_destination_pages(torch, ctx):
    """Positions whose source or destination page is missing are not moved;
    the selection is the same."""
    c = make_cache(torch, ctx, "bf16", 1, 6, 16, 1, 64, 14)
    table = torch.tensor([[0, -1, 2]], dtype=torch.int32, device="cuda")
    dst = torch.tensor([[3, 99]], dtype=torch.int32, device="cuda")
    before = c.k.clone()
    w = torch.rand(1, 1, 1, 48, device="cuda")
    kept, _, _ = c.evict(table, torch.tensor([48], dtype=torch.int32, device="cuda"), 48, w, 20, dst)
    keep = evict_reference(w[0, 0, 0].cpu().numpy(), 48, 20, 0, 0)
    assert np.array_equal(kept[0, 0, 0].cpu().numpy(), keep)
    for j in range(16):
        src = before[0, 3, 0, j] if 16 <= keep[j] < 32 else before[0, int(keep[j]) // 16, 0, int(keep[j]) % 16]
        assert torch.equal(c.k[0, 3, 0, j], src)
    for page in (0, 1, 2, 4, 5):
        assert torch.equal(c.k[0, page], before[0, page])


def test_attention_after_eviction(torch, ctx):
    """What is left attends as the definition does over the kept positions,
    and the weights go on accumulating."""
    lens, budget, D = [200, 90], 64, 64
    table, used = make_table(torch, lens, 16, 15)
    dst, more = make_table(torch, [64, 64], 16, 16, first=used)
    c = make_cache(torch, ctx, "int8", 1, used + more, 16, 2, D, 17)
    q = torch.randn(2, 4, D, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    w = torch.zeros(1, 2, 2, 200, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.attend(0, q, table, ln, 200, weights=w[0], weights_out=w[0])
    kept, wk, ln2 = c.evict(table, ln, 200, w, budget, dst, sinks=2, recent=8)
    before = wk.clone()
    out = c.attend(0, q, dst, ln2, budget, weights=wk[0], weights_out=wk[0])
    ref, ws, tol = reference(torch, c, 0, q, dst, [64, 64], 0.125)
    for b in range(2):
        assert float((out[b].double() - ref[b]).abs().max()) <= tol[b][0] * tol[b][1]
        assert float((wk[0, b].double() - before[0, b].double() - ws[b]).abs().max()) <= 2 * tol[b][0] + 2.0 ** -21
    k, v = values(c, "k", 0), values(c, "v", 0)
    for b in range(2):  # the kept rows are the source's
        for h in range(2):
            keep = kept[0, b, h].long()
            src = table[b][keep // 16].long()
            at = dst[b][torch.arange(64, device="cuda") // 16].long()
            assert torch.equal(k[at, h, torch.arange(64, device="cuda") % 16], k[src, h, keep % 16])
            assert torch.equal(v[at, h, torch.arange(64, device="cuda") % 16], v[src, h, keep % 16])


# ---- logits ------------------------------------------------------------------


def rules_reference(x, rep, pres, freq, ids, n_ids, n_prompt, bias, mask):
    f = np.float32
    x = x.copy()
    n, V = x.shape
    for r in range(n):
        if ids is not None:
            hist = ids[r, : max(0, min(n_ids[r], ids.shape[1]))]
            ok = (hist >= 0) & (hist < V)
            count = np.bincount(hist[ok], minlength=V)
            said = np.bincount(hist[max(0, n_prompt[r]):][ok[max(0, n_prompt[r]):]], minlength=V)
            if rep is not None:
                x[r] = np.where(count > 0, np.where(x[r] > 0, x[r] / f(rep[r]), x[r] * f(rep[r])), x[r])
            if freq is not None:
                x[r] = np.where(said > 0, x[r] - f(freq[r]) * said.astype(f), x[r])
            if pres is not None:
                x[r] = np.where(said > 0, x[r] - f(pres[r]), x[r])
        if bias is not None:
            add = {}
            for i in range(bias[0][r], bias[0][r + 1]):
                t = int(bias[1][i])
                add[t] = bias[2][i] if t not in add else f(add[t] + bias[2][i])
            for t, b in add.items():
                if 0 <= t < V:
                    x[r, t] = f(x[r, t] + b)
        if mask is not None:
            allowed = np.unpackbits(mask[r].view(np.uint8), bitorder="little")[:V].astype(bool)
            x[r] = np.where(allowed, x[r], f(-np.inf))
    best = []
    for r in range(n):
        ok = np.where(x[r] > -np.inf)[0]
        best.append(int(ok[np.argmax(x[r][ok])]) if ok.size else -1)
    return x, np.array(best, dtype=np.int32)


def make_rules(V, n, H, seed, bias=True, mask=True):
    rng = np.random.default_rng(seed)
    ids = rng.integers(-2, V + 2, (n, H)).astype(np.int32)
    ids[:, ::3] = rng.integers(0, min(V, 7), ids[:, ::3].shape)  # tokens that repeat
    n_ids = rng.integers(-1, H + 3, n).astype(np.int32)
    n_prompt = rng.integers(-1, H + 1, n).astype(np.int32)
    b = None
    if bias:
        rows = [np.sort(rng.integers(-1, V + 1, rng.integers(0, 40))).astype(np.int32) for _ in range(n)]
        off = np.concatenate([[0], np.cumsum([len(x) for x in rows])]).astype(np.int32)
        val = rng.standard_normal(off[-1]).astype(np.float32) * 4
        b = (off, np.concatenate(rows) if off[-1] else np.zeros(0, np.int32), val)
    m = None
    if mask:
        m = rng.integers(-2**31, 2**31, (n, (V + 31) // 32 + 1)).astype(np.int32)
        m[n // 2] = 0
    f = lambda lo, hi: (rng.random(n) * (hi - lo) + lo).astype(np.float32)  # noqa: E731
    return dict(rep=f(0.8, 1.5), pres=f(-1, 1), freq=f(-0.5, 0.5), ids=ids, n_ids=n_ids, n_prompt=n_prompt, bias=b,
                mask=m)


def to_rules(torch, r):
    from llm_mojo_b200.serving import LogitRules

    c = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    return LogitRules(repetition=c(r["rep"]), presence=c(r["pres"]), frequency=c(r["freq"]), ids=c(r["ids"]),
                      n_ids=c(r["n_ids"]), n_prompt=c(r["n_prompt"]),
                      bias=None if r["bias"] is None else tuple(c(a) for a in r["bias"]), mask=c(r["mask"]))


@pytest.mark.parametrize("V,n,H", [(1, 3, 4), (31, 2, 9), (33, 5, 50), (4096, 2, 300), (4097, 3, 2), (50257, 4, 1024),
                                   (50257, 1, 1), (130001, 2, 5000)])
@pytest.mark.parametrize("bias,mask", [(True, True), (False, False), (True, False), (False, True)])
def test_logit_rules_exact(torch, ctx, V, n, H, bias, mask):
    from llm_mojo_b200.serving import process_logits

    r = make_rules(V, n, H, V + H, bias, mask)
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    x[0, V // 2] = np.inf
    x[0, V // 3] = -np.inf
    x[:, :: 5] = np.float32(1.25)  # equal logits
    want, best = rules_reference(x, **r)
    logits = torch.from_numpy(x).cuda()
    out, top = process_logits(ctx, logits, to_rules(torch, r))
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(top.cpu().numpy(), best)
    assert np.array_equal(logits.cpu().numpy(), x)
    out2, top2 = process_logits(ctx, logits, to_rules(torch, r), out=logits, argmax=top)  # in place
    assert out2.data_ptr() == logits.data_ptr() and torch.equal(out2, out) and torch.equal(top2.cpu(), torch.from_numpy(best))


def test_logit_rules_nan(torch, ctx):
    """NaN stays where it is allowed and is never the argmax; a masked NaN
    becomes -infinity."""
    from llm_mojo_b200.serving import LogitRules, process_logits

    x = torch.full((3, 70), float("nan"), device="cuda")
    x[0, 40] = -5.0
    x[2, 3] = -1.0
    mask = torch.full((3, 3), -1, dtype=torch.int32, device="cuda")
    mask[2] = 1 << 4
    out, top = process_logits(ctx, x, LogitRules(mask=mask))
    assert top.tolist() == [40, -1, -1]
    allowed = torch.zeros(70, dtype=torch.bool, device="cuda")
    allowed[[4, 36, 68]] = True  # bit 4 of each word
    assert torch.equal(torch.isnan(out[2]), allowed) and torch.equal(torch.isneginf(out[2]), ~allowed)


@pytest.mark.parametrize("rows", [1, 3])
def test_logit_rules_views_and_parts(torch, ctx, rows):
    """Strided logits, outputs, histories and masks; each rule on its own; an
    empty history."""
    from llm_mojo_b200.serving import LogitRules, process_logits

    V = 5003
    r = make_rules(V, rows, 60, 21)
    x = np.random.default_rng(4).standard_normal((rows, V + 7)).astype(np.float32)
    full = to_rules(torch, r)
    wide = torch.full((rows, 90), 3, dtype=torch.int32, device="cuda")
    wide[:, 1:61] = full.ids
    full.ids = wide[:, 1:61]
    buf = torch.zeros(rows, V + 5, device="cuda")
    out, top = process_logits(ctx, torch.from_numpy(x).cuda()[:, 3: 3 + V], full, out=buf[:, 1: 1 + V])
    want, best = rules_reference(np.ascontiguousarray(x[:, 3: 3 + V]), **r)
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(top.cpu().numpy(), best)
    assert torch.count_nonzero(buf[:, 0]) == 0 and torch.count_nonzero(buf[:, V + 1:]) == 0
    logits = torch.from_numpy(np.ascontiguousarray(x[:, :V])).cuda()
    t = to_rules(torch, r)
    none = dict(rep=None, pres=None, freq=None, ids=None, n_ids=None, n_prompt=None, bias=None, mask=None)
    hist = dict(ids=t.ids, n_ids=t.n_ids, n_prompt=t.n_prompt)
    nh = {k: r[k] for k in ("ids", "n_ids", "n_prompt")}
    for rules, ref in ((LogitRules(repetition=t.repetition, **hist), dict(none, rep=r["rep"], **nh)),
                       (LogitRules(presence=t.presence, **hist), dict(none, pres=r["pres"], **nh)),
                       (LogitRules(frequency=t.frequency, **hist), dict(none, freq=r["freq"], **nh)),
                       (LogitRules(bias=t.bias), dict(none, bias=r["bias"])),
                       (LogitRules(mask=t.mask), dict(none, mask=r["mask"])), (LogitRules(), none)):
        out, top = process_logits(ctx, logits, rules)
        want, best = rules_reference(logits.cpu().numpy(), **ref)
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(top.cpu().numpy(), best)
    # without n_prompt the whole history is the answer
    out, _ = process_logits(ctx, logits, LogitRules(frequency=t.frequency, ids=t.ids, n_ids=t.n_ids))
    want, _ = rules_reference(logits.cpu().numpy(), **dict(none, freq=r["freq"], ids=r["ids"], n_ids=r["n_ids"],
                                                         n_prompt=np.zeros(rows, np.int32)))
    assert np.array_equal(out.cpu().numpy(), want)
    empty = torch.zeros(rows, 0, dtype=torch.int32, device="cuda")
    out, _ = process_logits(ctx, logits, LogitRules(repetition=t.repetition, ids=empty, n_ids=t.n_ids))
    assert torch.equal(out, logits)


def test_rules_then_sample(torch, ctx):
    """A processed row feeds the sampler: a single allowed token is drawn."""
    from llm_mojo_b200 import kernels
    from llm_mojo_b200.serving import LogitRules, process_logits

    x = torch.randn(1, 50257, device="cuda")
    mask = torch.zeros(1, 1571, dtype=torch.int32, device="cuda")
    mask[0, 1234 // 32] = 1 << (1234 % 32)
    out, top = process_logits(ctx, x, LogitRules(mask=mask))
    rng = kernels.Rng(1)
    assert int(top[0]) == 1234 and int(kernels.sample(ctx, out[0], 0.8, 40, rng)[0]) == 1234


# ---- refusals ----------------------------------------------------------------


def test_refusals(torch, ctx):
    from llm_mojo_b200._lib import ERR_INVALID, ERR_NOMEM, ERR_UNSUPPORTED, LlmqError
    from llm_mojo_b200.serving import LogitRules, PagedKVCache, process_logits

    def refused(status, fn, *a, **k):
        with pytest.raises(LlmqError) as e:
            fn(*a, **k)
        assert e.value.status == status, e.value

    for bad in ((0, 4, 16, 1, 64), (1, 0, 16, 1, 64), (1, 4, 0, 1, 64), (1, 4, 16, 0, 64), (1, 4, 16, 1, 48),
                (1, 4, 16, 1, 160), (1, 4, 16, 1, -64)):
        refused(ERR_INVALID, PagedKVCache, ctx, "bf16", *bad)
    refused(ERR_NOMEM, PagedKVCache, ctx, "f32", 1000, 2**31 - 1, 1024, 64, 128)
    with pytest.raises(ValueError):
        PagedKVCache(ctx, "intattn", 1, 4, 16, 1, 64)
    import ctypes as C

    from llm_mojo_b200._lib import KV_INTATTN, lib

    h = C.c_void_p()
    assert lib().llmq_paged_create(ctx.h, KV_INTATTN, 1, 4, 16, 1, 64, C.byref(h)) == ERR_UNSUPPORTED and not h
    c = make_cache(torch, ctx, "bf16", 2, 4, 16, 2, 64, 1)
    q, table = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    for layer in (-1, 2):
        refused(ERR_INVALID, c.attend, layer, q, table, lens, 5)
        refused(ERR_INVALID, c.store, layer, q[:, :2], q[:, :2], lens, table)
    refused(ERR_INVALID, c.attend, 0, q[:, :3], table, lens, 5)  # heads that do not divide
    refused(ERR_INVALID, c.attend, 0, q, table, lens, 0)
    refused(ERR_INVALID, c.attend, 0, q, table, lens, 5, out=torch.zeros(1, 4, 64, device="cuda").expand(2, -1, -1))
    refused(ERR_INVALID, c.store, 0, torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"),
            torch.zeros(3, dtype=torch.int32, device="cuda"), table)  # more rows than sequences
    w = torch.zeros(2, 2, 2, 32, device="cuda")
    dst = table + 2
    for kw in (dict(budget=4, sinks=3, recent=2), dict(budget=4, sinks=-1), dict(budget=4, recent=-1),
               dict(budget=33), dict(budget=4, layer0=1, n_layers=2)):
        kw = dict(dict(sinks=0, recent=0), **kw)
        budget = kw.pop("budget")
        ww = w if budget != 33 else torch.zeros(2, 2, 2, 64, device="cuda")
        refused(ERR_INVALID, c.evict, table, lens, ww.shape[3], ww, budget, dst, **kw)
    x = torch.zeros(2, 40, device="cuda")
    pen = torch.ones(2, device="cuda")
    refused(ERR_INVALID, process_logits, ctx, x, LogitRules(repetition=pen))
    refused(ERR_INVALID, process_logits, ctx, x, LogitRules(n_ids=lens))
    refused(ERR_INVALID, process_logits, ctx, x, LogitRules(), out=torch.zeros(1, 40, device="cuda").expand(2, -1))
    for fn in (lambda: c.attend(0, q.half(), table, lens, 5), lambda: c.attend(0, q.cpu(), table, lens, 5),
               lambda: c.attend(0, q, table.long(), lens, 5), lambda: c.attend(0, q, table[:1], lens, 5),
               lambda: c.attend(0, q, table, lens[:1], 5), lambda: c.attend(0, q[:, :, ::2], table, lens, 5),
               lambda: c.attend(0, q, table, lens, 40, weights_out=torch.zeros(2, 2, 39, device="cuda")),
               lambda: c.attend(0, q, table, lens, 5, weights=torch.zeros(2, 2, 39, device="cuda")),
               lambda: c.attend(0, q.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :32], table, lens, 5),
               lambda: c.store(0, q, q, lens, table), lambda: c.evict(table, lens, 32, w[:1], 4, dst),
               lambda: c.evict(table, lens, 33, w, 4, dst), lambda: c.evict(table, lens, 32, w, 0, dst),
               lambda: process_logits(ctx, x[0], LogitRules()), lambda: process_logits(ctx, x.double(), LogitRules()),
               lambda: process_logits(ctx, x, LogitRules(mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))),
               lambda: process_logits(ctx, x, LogitRules(ids=table[:1], n_ids=lens))):
        with pytest.raises(ValueError):
            fn()
    # the context works on
    c.attend(0, q, table, lens, 5)
    torch.cuda.synchronize()


def test_views_keep_the_pool(torch, ctx):
    """The pool lives as long as a view of it."""
    c = make_cache(torch, ctx, "f32", 1, 2, 4, 1, 32, 3)
    want = c.k.clone()
    k = c.k
    del c
    import gc

    gc.collect()
    assert torch.equal(k, want)


@pytest.mark.parametrize("kind", PAGED)
def test_c_owned_pool(torch, ctx, kind):
    """llmq_paged_create's own buffers start as zeros and hold what is
    stored; borrowed ones must be there and aligned."""
    import ctypes as C

    from llm_mojo_b200 import _lib
    from llm_mojo_b200.serving import KINDS

    L = _lib.lib()
    h = C.c_void_p()
    assert L.llmq_paged_create(ctx.h, KINDS[kind], 2, 3, 4, 2, 32, C.byref(h)) == _lib.OK
    size = [C.c_int() for _ in range(6)]
    assert L.llmq_paged_shape(h, *[C.byref(s) for s in size]) == _lib.OK
    assert [s.value for s in size] == [KINDS[kind], 2, 3, 4, 2, 32]
    table = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")
    q = torch.ones(1, 2, 32, device="cuda")
    out = torch.full((1, 2, 32), 9.0, device="cuda")
    lens = torch.tensor([8], dtype=torch.int32, device="cuda")
    args = (q.data_ptr(), 64, out.data_ptr(), 64, 1, 2, table.data_ptr(), 2, 2, lens.data_ptr(), 8, 1.0, None, None, 0)
    assert L.llmq_paged_attend(ctx.h, h, 1, *args) == _lib.OK
    assert torch.count_nonzero(out) == 0
    x = torch.full((8, 2, 32), 2.0, device="cuda")
    pos, seq = torch.arange(8, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    assert L.llmq_paged_store(ctx.h, h, 1, x.data_ptr(), 64, x.data_ptr(), 64, seq.data_ptr(), pos.data_ptr(), 8,
                              table.data_ptr(), 2, 2, 1) == _lib.OK
    assert L.llmq_paged_attend(ctx.h, h, 1, *args) == _lib.OK
    torch.cuda.synchronize()
    assert float((out - 2.0).abs().max()) < 2.0 ** -20
    assert L.llmq_paged_free(h) == _lib.OK
    b = torch.zeros(4096, device="cuda")
    for ptr in ((None, b.data_ptr()), (b.data_ptr(), b.data_ptr() + 4)):
        assert L.llmq_paged_create_in(ctx.h, KINDS[kind], 1, 1, 4, 1, 32, *ptr, b.data_ptr(), b.data_ptr(),
                                      C.byref(h)) == _lib.ERR_INVALID and not h


def test_capture(torch):
    """Calls captured in a graph replay with new inputs; a workspace that
    would have to grow during a capture is refused, and the capture goes on."""
    from llm_mojo_b200._lib import ERR_INVALID, LlmqError
    from llm_mojo_b200.serving import LogitRules, process_logits
    from llm_mojo_b200.tensor import Context

    own = Context(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own.use_torch_stream()
        lens = [700, 90]
        table, n_pages = make_table(torch, lens, 16, 3)
        c = make_cache(torch, own, "bf16", 1, n_pages, 16, 2, 64, 4)
        q = torch.randn(2, 4, 64, device="cuda")
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        w, wo = torch.zeros(2, 2, 700, device="cuda"), torch.zeros(2, 2, 700, device="cuda")
        x = torch.randn(2, 50257, device="cuda")
        pen = torch.full((2,), 1.2, device="cuda")
        ids = torch.randint(0, 50257, (2, 50), dtype=torch.int32, device="cuda")
        rules = LogitRules(repetition=pen, ids=ids, n_ids=torch.full((2,), 50, dtype=torch.int32, device="cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(LlmqError) as e:
                c.attend(0, q, table, ln, 700, weights=w, weights_out=wo)
            assert e.value.status == ERR_INVALID
            q.add_(0.0)
        c.attend(0, q, table, ln, 700, weights=w, weights_out=wo)
        process_logits(own, x, rules)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = c.attend(0, q, table, ln, 700, weights=w, weights_out=wo)
            y, top = process_logits(own, x, rules)
        for _ in range(3):
            q.normal_()
            x.normal_()
            graph.replay()
            got = [t.clone() for t in (out, wo, y, top)]
            w2 = torch.zeros_like(wo)
            want = [c.attend(0, q, table, ln, 700, weights=w, weights_out=w2), w2, *process_logits(own, x, rules)]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        side.synchronize()
        del graph
    c.free()
    own.close()


def test_capture_outlives_the_workspace_it_used(torch):
    """A captured call replays after larger ones have made the workspace grow."""
    from llm_mojo_b200.serving import LogitRules, process_logits
    from llm_mojo_b200.tensor import Context

    own = Context(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own.use_torch_stream()
        lens = [700, 90]
        table, n_pages = make_table(torch, lens, 16, 3)
        c = make_cache(torch, own, "bf16", 1, n_pages, 16, 2, 64, 4)
        q = torch.randn(2, 4, 64, device="cuda")
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        wo = torch.zeros(2, 2, 700, device="cuda")
        x = torch.randn(2, 5000, device="cuda")
        rules = LogitRules()
        c.attend(0, q, table, ln, 700, weights_out=wo)
        process_logits(own, x, rules)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = c.attend(0, q, table, ln, 700, weights_out=wo)
            y, top = process_logits(own, x, rules)
        graph.replay()
        want = [t.clone() for t in (out, wo, y, top)]
        rows = 512
        tables, lns = table[:1].repeat(rows, 1), ln[:1].repeat(rows)
        many = torch.randn(rows, 4, 64, device="cuda")
        for n in (64, 128, rows):
            c.attend(0, many[:n], tables[:n], lns[:n], 700, weights_out=torch.empty(n, 2, 700, device="cuda"))
        process_logits(own, torch.randn(rows, 5000, device="cuda"), rules)
        for t in (out, wo, y, top):
            t.zero_()
        for _ in range(3):
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip((out, wo, y, top), want))
        side.synchronize()
        del graph
    c.free()
    own.close()


@pytest.mark.parametrize("kind", PAGED)
def test_attend_nan_stays_in_its_head(torch, ctx, kind):
    """A query with a NaN gives NaN for its own head; the others, of the same
    key head, too, are as without it."""
    table, n_pages = make_table(torch, [150], 16, 3)
    c = make_cache(torch, ctx, kind, 1, n_pages, 16, 2, 64, 4)
    q = torch.randn(1, 8, 64, device="cuda")
    ln = torch.tensor([150], dtype=torch.int32, device="cuda")
    want = c.attend(0, q, table, ln, 150)
    q[0, 5, 11] = float("nan")
    got = c.attend(0, q, table, ln, 150)
    assert torch.isnan(got[0, 5]).all()
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert torch.equal(got[0, keep], want[0, keep])
