"""Cases of the serving operators: the paged KV cache's store, attention of
one new token per sequence over it, eviction by accumulated attention weight,
and the rules on logits. Each case runs through the framework (own = True) or
in plain torch operations (own = False)."""

import math
import random

import numpy as np
import torch

own = False

ELEM = {"int8": 1, "bf16": 2, "f32": 4}
DTYPE = {"int8": torch.int8, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # one GPT-2 sequence early in its answer: latency
        dict(name="attend_single", op="attend", kind="int8", seqs=1, heads=12, kv_heads=12, dim=64, page=16,
             max_len=200, ragged=False, weights=False),
        # a full batch of short GPT-2 sequences of different ages
        dict(name="attend_batch", op="attend", kind="int8", seqs=256, heads=12, kv_heads=12, dim=64, page=16,
             max_len=256, ragged=True, weights=False),
        # one long document, twelve heads: the length is all there is to split
        dict(name="attend_long", op="attend", kind="int8", seqs=1, heads=12, kv_heads=12, dim=64, page=64,
             max_len=131071, ragged=False, weights=False),
        # grouped heads over long ragged contexts, with the weights that eviction needs
        dict(name="attend_grouped", op="attend", kind="bf16", seqs=8, heads=32, kv_heads=8, dim=128, page=64,
             max_len=32768, ragged=True, weights=True),
        # a few float32 sequences, three heads to a key head, pages that end inside a tile
        dict(name="attend_odd", op="attend", kind="f32", seqs=5, heads=6, kv_heads=2, dim=64, page=20,
             max_len=1023, ragged=True, weights=True),
        # one new token of each sequence of a batch
        dict(name="store_step", op="store", kind="bf16", seqs=256, rows=1, kv_heads=12, dim=64, page=16),
        # the prompts of a few sequences
        dict(name="store_prompts", op="store", kind="bf16", seqs=7, rows=2341, kv_heads=8, dim=128, page=64),
        # a GPT-2 sequence at its position limit, halved in every layer
        dict(name="evict_gpt2", op="evict", kind="f32", layers=12, seqs=1, kv_heads=12, dim=64, page=16,
             max_len=1024, ragged=False, budget=512, sinks=4, recent=64),
        # long ragged sequences cut to a budget, some already below it
        dict(name="evict_long", op="evict", kind="bf16", layers=4, seqs=8, kv_heads=8, dim=128, page=64,
             max_len=16384, ragged=True, budget=4096, sinks=4, recent=511),
        # GPT-2's logits of one sequence: penalties only
        dict(name="logits_single", op="logits", rows=1, vocab=50257, history=100, bias=0, mask=False),
        # a batch of GPT-2 rows, every rule
        dict(name="logits_batch", op="logits", rows=256, vocab=50257, history=1024, bias=300, mask=True),
        # a wide odd vocabulary with long histories
        dict(name="logits_wide", op="logits", rows=61, vocab=200003, history=8192, bias=37, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "evict", "evict", "logits", "logits"])
    if op == "logits":
        rows = _log(rng, 1, 256)
        vocab = min(_log(rng, 1000, 260000), 12_000_000 // rows) | 1
        return dict(op=op, rows=rows, vocab=vocab, history=_log(rng, 1, 8192), bias=rng.choice([0, 1, 37, 300]),
                    mask=rng.random() < 0.7)
    # the store and the eviction return the cache itself: kinds whose values it holds as they are
    kind = rng.choice(["int8", "bf16", "f32"] if op == "attend" else ["bf16", "f32"])
    dim = rng.choice([32, 64, 64, 96, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128, _log(rng, 1, 100)])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 16])
    row = kv_heads * 2 * dim * ELEM[kind]  # bytes of one position
    if op == "store":
        seqs = _log(rng, 1, 256)
        rows = rng.choice([1, _log(rng, 1, max(2, min(4096, 60_000_000 // (kv_heads * dim * 4 * seqs))))])
        return dict(op=op, kind=kind, seqs=seqs, rows=rows, kv_heads=kv_heads, dim=dim, page=page)
    if op == "attend":
        group = rng.choice([1, 1, 2, 3, 4, 6, 8, 11])
        seqs = _log(rng, 1, 256)
        top = max(1, min(131072, 500_000_000 // (row * seqs)))
        # the work per position grows with the group, and so does the plain form's score array
        top = max(1, min(top, 30_000_000 // (seqs * kv_heads * group)))
        max_len = _log(rng, 1, top)
        return dict(op=op, kind=kind, seqs=seqs, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                    max_len=max_len, ragged=rng.random() < 0.7, weights=rng.random() < 0.5)
    layers = _log(rng, 1, 12)
    seqs = _log(rng, 1, 16)
    max_len = _log(rng, 2, max(3, min(65536, 400_000_000 // (row * layers * seqs))))
    budget = max(1, int(max_len * rng.uniform(0.1, 0.9)))
    recent = rng.randint(0, budget // 2)
    return dict(op=op, kind=kind, layers=layers, seqs=seqs, kv_heads=kv_heads, dim=dim, page=page, max_len=max_len,
                ragged=rng.random() < 0.7, budget=budget, sinks=rng.randint(0, min(8, budget - recent)),
                recent=recent)


# ---- inputs ------------------------------------------------------------------


def _lens(case):
    """The sequences' lengths: the first is the longest; of eight or more
    ragged ones the last is empty."""
    n, top = case["seqs"], case["max_len"]
    if not case["ragged"]:
        return [top] * n
    rng = random.Random(n * 1000003 + top)
    lens = [top] + [rng.randint(1, top) for _ in range(n - 1)]
    if n >= 8:
        lens[-1] = 0
    return lens


def _pages(lens, page, gen, first=0):
    """Shuffled page ids for sequences of these lengths: the table [n, widest]
    (-1 where a sequence has no page) and the number of pages."""
    need = [-(-n // page) for n in lens]
    total = sum(need)
    order = (torch.randperm(total, generator=gen, device="cuda").to(torch.int32) + first).split(need)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    for b, ids in enumerate(order):
        table[b, : need[b]] = ids
    return table, total


def _fill(kind, shape, gen):
    """Random cache rows [..., dim] with a few loud channels, as the kind
    stores them: (values, scales or None)."""
    dim = shape[-1]
    loud = 1.0 + 2.0 * (torch.rand(dim, generator=gen, device="cuda") < 0.05)
    x = torch.randn(shape, generator=gen, device="cuda") * loud
    if kind != "int8":
        return x.to(DTYPE[kind]), None
    s = x.abs().amax(-1) / 127.0
    return torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8), s


def _cache(case, layers, n_pages, gen):
    """The cache with random contents: tensors k, v (and ks, vs), and the
    framework's handle that owns them."""
    shape = (layers, n_pages, case["kv_heads"], case["page"], case["dim"])
    st = {}
    if own:
        from llm_mojo_b200.serving import PagedKVCache
        from llm_mojo_b200.tensor import Context

        ctx = Context(torch.cuda.current_device())
        ctx.use_torch_stream()
        st["ctx"] = ctx
        cache = PagedKVCache(ctx, case["kind"], layers, n_pages, case["page"], case["kv_heads"], case["dim"])
        st["cache"] = cache
        st["k"], st["v"], st["ks"], st["vs"] = cache.k, cache.v, cache.ks, cache.vs
    else:
        st["k"] = torch.empty(shape, dtype=DTYPE[case["kind"]], device="cuda")
        st["v"] = torch.empty_like(st["k"])
        st["ks"] = st["vs"] = None
        if case["kind"] == "int8":
            st["ks"] = torch.empty(shape[:-1], device="cuda")
            st["vs"] = torch.empty(shape[:-1], device="cuda")
    for name in ("k", "v"):
        for layer in range(layers):
            val, s = _fill(case["kind"], shape[1:], gen)
            st[name][layer].copy_(val)
            if s is not None:
                st[name + "s"][layer].copy_(s)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"attend": _prepare_attend, "store": _prepare_store, "evict": _prepare_evict,
            "logits": _prepare_logits}[case["op"]](case, gen)


def _prepare_attend(case, gen):
    lens = _lens(case)
    table, total = _pages(lens, case["page"], gen)
    st = _cache(case, 1, max(1, total), gen)
    n, h = case["seqs"], case["heads"]
    st.update(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              q=torch.randn(n, h, case["dim"], generator=gen, device="cuda") * 1.5, w=None, wo=None)
    if case["weights"]:
        st["w"] = torch.rand(n, case["kv_heads"], case["max_len"], generator=gen, device="cuda")
        st["wo"] = torch.zeros_like(st["w"])
    return st


def _prepare_store(case, gen):
    n, rows = case["seqs"], case["rows"]
    rng = random.Random(n * 1009 + rows)
    start = [rng.randint(0, 40) for _ in range(n)]  # tokens that each sequence holds already
    table, total = _pages([s + rows for s in start], case["page"], gen)
    st = _cache(case, 1, total, gen)
    kv = case["kv_heads"] * case["dim"]
    pos = torch.tensor(start, dtype=torch.int32, device="cuda")[:, None] + torch.arange(
        rows, dtype=torch.int32, device="cuda")
    seq = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].expand(n, rows)
    # keys and values as columns of one projection's rows
    qkv = torch.randn(n * rows, 3 * kv, generator=gen, device="cuda")
    shape = (n * rows, case["kv_heads"], case["dim"])
    st.update(case=case, table=table, pos=pos.reshape(-1).contiguous(), seq=seq.reshape(-1).contiguous(),
              nk=qkv[:, kv: 2 * kv].unflatten(1, shape[1:]), nv=qkv[:, 2 * kv:].unflatten(1, shape[1:]))
    return st


def _prepare_evict(case, gen):
    lens = _lens(case)
    table, total = _pages(lens, case["page"], gen)
    dst, more = _pages([min(n, case["budget"]) for n in lens], case["page"], gen, first=total)
    st = _cache(case, case["layers"], max(1, total + more), gen)
    shape = (case["layers"], case["seqs"], case["kv_heads"], case["max_len"])
    # accumulated weights: most of it on a few positions, and many exact zeros
    w = torch.rand(shape, generator=gen, device="cuda") ** 6 * 4.0
    w = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.2, torch.zeros_like(w), w)
    st.update(case=case, table=table, dst=dst, w=w, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return st


def _prepare_logits(case, gen):
    n, V, H = case["rows"], case["vocab"], case["history"]
    dev = dict(generator=gen, device="cuda")
    rng = random.Random(n * 7919 + V + H)
    n_ids = [H] + [rng.randint(0, H) for _ in range(n - 1)]
    n_prompt = [rng.randint(0, k) for k in n_ids]
    ids = (torch.rand(n, H, **dev) ** 4 * V).to(torch.int32).clamp_(0, V - 1)  # frequent tokens have low ids
    st = dict(case=case, logits=torch.randn(n, V, **dev) * 3.0, ids=ids,
              n_ids=torch.tensor(n_ids, dtype=torch.int32, device="cuda"),
              n_prompt=torch.tensor(n_prompt, dtype=torch.int32, device="cuda"),
              repetition=1.0 + 0.3 * torch.rand(n, **dev), presence=0.6 * torch.rand(n, **dev),
              frequency=0.4 * torch.rand(n, **dev), bias=None, mask=None)
    if case["bias"]:
        counts = [rng.randint(0, min(case["bias"], V)) for _ in range(n)]
        off = torch.tensor([0, *np.cumsum(counts).tolist()], dtype=torch.int32, device="cuda")
        bid = torch.cat([torch.rand(V, **dev).argsort()[:c].sort().values for c in counts]).to(torch.int32)
        st["bias"] = (off, bid, torch.randn(bid.numel(), **dev) * 5.0)
    if case["mask"]:
        words = (V + 31) // 32
        mask = torch.randint(-(2**31), 2**31, (n, words), dtype=torch.int64, **dev)
        for r in range(n):  # every third row: a grammar state that allows a few words of the vocabulary
            if r % 3 == 1:
                mask[r] = torch.where(torch.rand(words, **dev) < 0.02, mask[r], 0)
        if n >= 8:
            mask[-1] = 0  # a row that nothing is left of
        st["mask"] = mask.to(torch.int32)
    if own:
        from llm_mojo_b200.serving import LogitRules
        from llm_mojo_b200.tensor import Context

        st["ctx"] = Context(torch.cuda.current_device())
        st["ctx"].use_torch_stream()
        st["rules"] = LogitRules(repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                                 ids=ids, n_ids=st["n_ids"], n_prompt=st["n_prompt"], bias=st["bias"],
                                 mask=st["mask"])
    return st


# ---- one pass ----------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if own:
        return {"attend": _own_attend, "store": _own_store, "evict": _own_evict, "logits": _own_logits}[op](st)
    return {"attend": _plain_attend, "store": _plain_store, "evict": _plain_evict, "logits": _plain_logits}[op](st)


def _own_attend(st):
    out = st["cache"].attend(0, st["q"], st["table"], st["lens"], st["case"]["max_len"], weights=st["w"],
                             weights_out=st["wo"])
    return out if st["w"] is None else (out, st["wo"])


def _own_store(st):
    c = st["cache"]
    c.store(0, st["nk"], st["nv"], st["pos"], st["table"], seq=None if st["case"]["rows"] == 1 else st["seq"])
    return c.k, c.v


def _own_evict(st):
    c, case = st["cache"], st["case"]
    kept, w, lens = c.evict(st["table"], st["lens"], case["max_len"], st["w"], case["budget"], st["dst"],
                            sinks=case["sinks"], recent=case["recent"])
    return kept, w, lens, c.k, c.v


def _own_logits(st):
    from llm_mojo_b200.serving import process_logits

    return process_logits(st["ctx"], st["logits"], st["rules"])


def _plain_attend(st):
    case, q, lens, table = st["case"], st["q"], st["lens"], st["table"]
    n, h, hk, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    pos = torch.arange(case["max_len"], device="cuda")
    page = table[:, pos // case["page"]].long()
    ok = (pos < lens[:, None]) & (page >= 0)
    page, slot = page.clamp(min=0), (pos % case["page"]).expand(n, -1)
    k = st["k"][0][page, :, slot].float()  # [n, len, kv_heads, dim]
    v = st["v"][0][page, :, slot].float()
    if st["ks"] is not None:
        k = k * st["ks"][0][page, :, slot][..., None]
        v = v * st["vs"][0][page, :, slot][..., None]
    ok = ok[:, None, None, :]
    s = torch.matmul(q.view(n, hk, h // hk, d), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p, v.transpose(1, 2)).reshape(n, h, d)
    if st["w"] is None:
        return out
    st["wo"].copy_(st["w"] + p.sum(2))
    return out, st["wo"]


def _plain_store(st):
    case, dt = st["case"], DTYPE[st["case"]["kind"]]
    seq, pos = st["seq"].long(), st["pos"].long()
    page = st["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    st["k"][0][page, :, slot] = st["nk"].to(dt)
    st["v"][0][page, :, slot] = st["nv"].to(dt)
    return st["k"], st["v"]


def _plain_evict(st):
    case, lens, w = st["case"], st["lens"].long(), st["w"]
    L, n, hk, top = w.shape
    budget = case["budget"]
    pos = torch.arange(top, device="cuda")
    ln = lens[:, None]
    # sinks and recent positions first, then by weight, then what is not there; equal weights by index
    always = (pos < case["sinks"]) | (pos >= ln - case["recent"])
    rank = torch.where(always[None, :, None], torch.full_like(w, math.inf), w)
    rank = torch.where((pos < ln)[None, :, None], rank, torch.full_like(w, -math.inf))
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    new_len = lens.clamp(max=budget)
    j = torch.arange(budget, device="cuda")
    live = j < new_len[:, None]
    kept = torch.where(live[None, :, None], best[..., : budget], top).sort(dim=-1).values  # order of the positions
    j = j[: kept.shape[-1]]
    live = live[None, :, None, : kept.shape[-1]].expand_as(kept)
    src = kept.clamp(max=top - 1)
    wo = torch.where(live, w.gather(-1, src), torch.zeros((), device="cuda"))
    li, bi, hi, ji = live.nonzero(as_tuple=True)
    sp = kept[li, bi, hi, ji]
    spage, sslot = st["table"][bi, sp // case["page"]].long(), sp % case["page"]
    dpage, dslot = st["dst"][bi, ji // case["page"]].long(), ji % case["page"]
    for c in (st["k"], st["v"]):
        c[li, dpage, hi, dslot] = c[li, spage, hi, sslot]
    return torch.where(live, kept, -1).to(torch.int32), wo, new_len.to(torch.int32), st["k"], st["v"]


def _plain_logits(st):
    case, x = st["case"], st["logits"]
    n, V, H = case["rows"], case["vocab"], case["history"]
    j = torch.arange(H, device="cuda")
    there = j < st["n_ids"][:, None]
    answer = there & (j >= st["n_prompt"][:, None])
    ids = st["ids"].long()
    c_all = torch.zeros(n, V, device="cuda").scatter_add_(1, ids, there.float())
    c_out = torch.zeros(n, V, device="cuda").scatter_add_(1, ids, answer.float())
    r = st["repetition"][:, None]
    x = torch.where(c_all > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * c_out
    x = torch.where(c_out > 0, x - st["presence"][:, None], x)
    if st["bias"] is not None:
        off, bid, val = st["bias"]
        row = torch.searchsorted(off[1:].contiguous(), torch.arange(bid.numel(), device="cuda", dtype=torch.int32),
                                 right=True)
        x = x.index_put((row, bid.long()), val, accumulate=True)
    if st["mask"] is not None:
        t = torch.arange(V, device="cuda")
        bit = (st["mask"][:, t // 32] >> (t % 32).to(torch.int32)) & 1
        x = torch.where(bit == 1, x, torch.full_like(x, -math.inf))
    top = x.amax(1)
    first = torch.where(x == top[:, None], torch.arange(V, device="cuda"), V).amin(1)
    return x, torch.where(top == -math.inf, -1, first).to(torch.int32)


# ---- work --------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "logits":
        n, V, H = case["rows"], case["vocab"], case["history"]
        rng = random.Random(n * 7919 + V + H)
        ids = H + sum(rng.randint(0, H) for _ in range(n - 1))
        return {"bytes": n * V * 8 + ids * 4 + (n * ((V + 31) // 32) * 4 if case["mask"] else 0) + n * 24
                + n * case["bias"] * 4, "flops": n * V * 3}
    kv = case["kv_heads"] * case["dim"]
    es = ELEM[case["kind"]]
    if op == "store":
        rows = case["seqs"] * case["rows"]
        return {"bytes": rows * (2 * kv * (4 + es) + 12), "flops": rows * 2 * kv}
    lens = _lens(case)
    if op == "attend":
        total = sum(lens)
        per = 2 * kv * es + (8 * case["kv_heads"] if case["kind"] == "int8" else 0)
        per += 8 * case["kv_heads"] if case["weights"] else 0
        return {"bytes": total * per + 8 * case["seqs"] * case["heads"] * case["dim"]
                + sum(-(-n // case["page"]) for n in lens) * 4 + 4 * case["seqs"],
                "flops": 4 * total * case["heads"] * case["dim"]}
    heads = case["layers"] * case["kv_heads"]
    keep = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": sum(lens) * heads * 4 + keep * heads * (4 * case["dim"] * es)
            + case["seqs"] * case["budget"] * heads * 8, "flops": sum(lens) * heads}


# ---- the definitions in 64 bits ----------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"attend": _exact_attend, "store": _exact_store, "evict": _exact_evict,
            "logits": _exact_logits}[case["op"]](st)


def _exact_attend(st):
    case = st["case"]
    n, hk, d = case["seqs"], case["kv_heads"], case["dim"]
    g = case["heads"] // hk
    out = torch.zeros(n, case["heads"], d, dtype=torch.float64, device="cuda")
    wo = None if st["w"] is None else st["w"].double()
    table = st["table"].tolist()
    for b, length in enumerate(st["lens"].tolist()):
        if length == 0:
            continue
        pages = torch.tensor(table[b][: -(-length // case["page"])], device="cuda")
        for h in range(hk):
            def rows(name):
                x = st[name][0, pages, h].double()
                if st[name + "s"] is not None:
                    x = x * st[name + "s"][0, pages, h].double()[..., None]
                return x.reshape(-1, d)[:length]

            k, v = rows("k"), rows("v")
            for i in range(h * g, (h + 1) * g):
                z = torch.mv(k, st["q"][b, i].double()) / math.sqrt(d)
                e = (z - z.max()).exp()
                e = e / e.sum()
                out[b, i] = torch.mv(v.T, e)
                if wo is not None:
                    wo[b, h, :length] += e
    return out if wo is None else (out, wo)


def _exact_store(st):
    """Row by row from the table; the stored types round to nearest."""
    case = st["case"]
    pages, seq, pos = (st[x].cpu().numpy() for x in ("table", "seq", "pos"))
    res = []
    for name, new in (("k", "nk"), ("v", "nv")):
        pool = st[name].double()
        rows = st[new].to(DTYPE[case["kind"]]).double()
        flat = pool[0].permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["dim"])
        at = [int(pages[s][p // case["page"]]) * case["page"] + int(p) % case["page"] for s, p in zip(seq, pos)]
        flat[torch.tensor(at, device="cuda")] = rows
        pool[0] = flat.reshape(pool.shape[1], case["page"], case["kv_heads"], case["dim"]).permute(0, 2, 1, 3)
        res.append(pool)
    return tuple(res)


def _exact_evict(st):
    case = st["case"]
    L, n, hk, top = st["w"].shape
    page, budget = case["page"], case["budget"]
    w = st["w"].double().cpu().numpy()
    table, dst, lens = (st[x].cpu().numpy() for x in ("table", "dst", "lens"))
    kept = np.full((L, n, hk, budget), -1, dtype=np.int32)
    wo = np.zeros((L, n, hk, budget))
    k, v = st["k"].clone(), st["v"].clone()
    for b in range(n):
        length = int(lens[b])
        for layer in range(L):
            for h in range(hk):
                row = w[layer, b, h, :length]
                if length <= budget:
                    keep = np.arange(length)
                else:
                    first, last = case["sinks"], length - case["recent"]
                    mid = np.arange(first, last)
                    best = mid[np.argsort(-row[first:last], kind="stable")[: budget - first - case["recent"]]]
                    keep = np.sort(np.concatenate([np.arange(first), best, np.arange(last, length)]))
                m = len(keep)
                kept[layer, b, h, :m] = keep
                wo[layer, b, h, :m] = row[keep]
                if m == 0:
                    continue
                sp, dp = table[b][keep // page], dst[b][np.arange(m) // page]
                ss, ds = keep % page, np.arange(m) % page
                sp, dp, ss, ds = (torch.as_tensor(a, device="cuda").long() for a in (sp, dp, ss, ds))
                k[layer, dp, h, ds] = k[layer, sp, h, ss]
                v[layer, dp, h, ds] = v[layer, sp, h, ss]
    dev = dict(device="cuda")
    return (torch.as_tensor(kept, **dev), torch.as_tensor(wo, **dev),
            torch.as_tensor(np.minimum(lens, budget).astype(np.int32), **dev), k, v)


def _exact_logits(st):
    case = st["case"]
    n, V = case["rows"], case["vocab"]
    x = st["logits"].double().cpu().numpy()
    host = {key: st[key].cpu().numpy() for key in ("ids", "n_ids", "n_prompt", "repetition", "presence", "frequency")}
    bias = None if st["bias"] is None else [a.cpu().numpy() for a in st["bias"]]
    mask = None if st["mask"] is None else st["mask"].cpu().numpy().view(np.uint32)
    for r in range(n):
        ids = host["ids"][r, : host["n_ids"][r]]
        seen = np.unique(ids)
        rep = float(host["repetition"][r])
        x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        said, times = np.unique(ids[host["n_prompt"][r]:], return_counts=True)
        x[r, said] -= float(host["frequency"][r]) * times + float(host["presence"][r])
        if bias is not None:
            a, b = bias[0][r], bias[0][r + 1]
            x[r, bias[1][a:b]] += bias[2][a:b]
        if mask is not None:
            allowed = np.unpackbits(mask[r].view(np.uint8), bitorder="little")[:V].astype(bool)
            x[r, ~allowed] = -np.inf
    return torch.as_tensor(x, device="cuda"), None
