"""Generation for sequences of any lengths over one paged cache: the serving
operators as a decode loop runs them. Each step stores the tokens' keys and
values, attends over the sequences' pages (accumulating softmax weights where
the cache is bounded), applies the rules to the logits and takes the next
tokens; a sequence that outgrows its limit is cut to its budget by weight and
its old pages go back to the pool.

    python -m llm_mojo_b200.paged_generate

runs a small random-init model.
"""

from __future__ import annotations

import torch

from . import kernels
from .model import Batch, Model
from .serving import LogitRules, PagedKVCache, process_logits


class PagePool:
    """The free pages of a cache."""

    def __init__(self, n_pages: int):
        self.free = list(range(n_pages - 1, -1, -1))

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise RuntimeError(f"the page pool has {len(self.free)} pages left, {n} are needed")
        return [self.free.pop() for _ in range(n)]

    def give(self, pages: list[int]):
        self.free.extend(reversed(pages))


class PagedGenerator:
    """Generates for up to max_seqs sequences at once with a GPT-2 `model`.

    kind: the cache ('int8', 'bf16' or 'f32'). limit: a sequence's cache is
    cut when it holds this many positions (None: never; max_len at most), to
    `budget` positions, of which the first `sinks` and the last `recent`
    always stay.
    Memory for cache positions is then max_seqs * limit, and budget more
    while a sequence is cut, whatever the texts' lengths."""

    def __init__(self, model: Model, max_seqs: int, kind: str = "int8", page_size: int = 16, max_len: int = 1024,
                 limit: int | None = None, budget: int | None = None, sinks: int = 4, recent: int = 32):
        if limit is not None and not 0 < (budget or 0) < min(limit, max_len):
            raise ValueError("a limit needs a positive budget below it and below max_len")
        if limit is not None and (min(sinks, recent) < 0 or sinks + recent > budget):
            raise ValueError("sinks and recent must fit in the budget")
        if min(max_seqs, page_size, max_len) <= 0:
            raise ValueError("max_seqs, page_size and max_len must be positive")
        self.model, self.max_seqs, self.page_size = model, max_seqs, page_size
        self.limit, self.budget, self.sinks, self.recent = limit, budget, sinks, recent
        self.cap = min(max_len, limit or max_len)  # positions that a sequence's cache may hold
        self.cols = -(-self.cap // page_size)
        self.batch = Batch(model, max_seqs, 0)
        n_pages = max_seqs * self.cols + (-(-budget // page_size) * max_seqs if limit else 0)
        n_head = 12
        self.cache = PagedKVCache(model.ctx, kind, model.n_layer, n_pages, page_size, n_head, 64)
        self.n_head = n_head

    def generate(self, prompts, steps: int, repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0,
                 bias: dict[int, float] | None = None, allowed=None, temperature: float = 0.0, top_k: int = 40,
                 seed: int = 1337) -> list[list[int]]:
        """`steps` tokens for each of the prompts (lists of ids, any lengths).
        allowed(step, texts) -> bool CPU tensor [n, V], or None, is a
        grammar's say on each step; where it leaves nothing, and at
        temperature 0, the token is process_logits's argmax (EOT 50256 if
        there is none), else a draw of sample. Prompt b's draws, one per token
        of its answer, come from a generator of its own, of seed + b: what the
        other prompts are does not change them."""
        if not 0 < len(prompts) <= self.max_seqs or any(len(p) == 0 for p in prompts):
            raise ValueError(f"between 1 and {self.max_seqs} prompts, none empty")
        if any(not 0 <= t < self.model.V for p in prompts for t in p):
            raise ValueError(f"token ids must be in [0, {self.model.V})")
        if steps < 0:
            raise ValueError("steps must not be negative")
        with self.model.ctx.torch_stream():
            return self._generate(prompts, steps, repetition, presence, frequency, bias, allowed, temperature, top_k, seed)

    def _generate(self, prompts, steps, repetition, presence, frequency, bias, allowed, temperature, top_k, seed):
        B, V, ps, dev = len(prompts), self.model.V, self.page_size, "cuda"
        total = max(len(p) for p in prompts) + steps
        if total - 1 > 1024:
            raise ValueError("GPT-2 has 1024 positions")
        if not self.limit and total - 1 > self.cap:
            raise ValueError(f"texts of up to {self.cap} positions")
        pool = PagePool(self.cache.n_pages)
        pages: list[list[int]] = [[] for _ in range(B)]
        table = torch.full((B, self.cols), -1, dtype=torch.int32, device=dev)
        weights = None
        if self.limit:
            weights = torch.zeros(self.model.n_layer, B, self.n_head, self.cap, device=dev)
        history = torch.zeros(B, total, dtype=torch.int32)
        for b, p in enumerate(prompts):
            history[b, : len(p)] = torch.tensor(p)
        history = history.to(dev)
        n_prompt = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)

        def row(x):
            return torch.full((B,), x, device=dev)

        rules = LogitRules(repetition=row(repetition), presence=row(presence), frequency=row(frequency), ids=history,
                           n_ids=torch.zeros(B, dtype=torch.int32, device=dev), n_prompt=n_prompt)
        if bias:
            ids = sorted(bias)
            rules.bias = (torch.arange(B + 1, dtype=torch.int32, device=dev) * len(ids),
                          torch.tensor(ids * B, dtype=torch.int32, device=dev),
                          torch.tensor([bias[i] for i in ids] * B, device=dev))
        rngs = [kernels.Rng(seed + b) for b in range(B)] if temperature > 0 else []
        logits = torch.empty(B, V, device=dev)
        held = [0] * B  # positions in each cache
        texts = [list(p) for p in prompts]
        ends = [len(p) + steps - 1 for p in prompts]  # the step after a text's last
        for at in range(total - 1):
            # a text that is done stores nothing, attends to nothing and gives its pages back
            live = [b for b in range(B) if at < ends[b]]
            for b in range(B):
                if at >= ends[b] and pages[b]:
                    pool.give(pages[b])
                    pages[b] = []
                    table[b] = -1
            if self.limit:
                full = [b for b in live if held[b] >= self.cap]
                if full:
                    self._cut(full, held, pages, table, weights, pool)
            slots = [-1] * B
            for b in live:
                if held[b] % ps == 0:
                    pages[b] += pool.take(1)
                    table[b, held[b] // ps] = pages[b][-1]
                slots[b] = held[b]
                held[b] += 1
            slots = torch.tensor(slots, dtype=torch.int32, device=dev)
            lens = slots + 1
            pos = torch.full((B,), at, dtype=torch.int32, device=dev)
            self.batch.paged_step(self.cache, history[:, at].contiguous(), pos, slots, table, lens,
                                  max(held[b] for b in live), logits, weights)
            rules.n_ids.fill_(at + 1)
            rules.mask = None
            if allowed is not None:
                ok = allowed(at, texts)
                rules.mask = None if ok is None else pack_mask(ok).to(dev)
            out, top = process_logits(self.model.ctx, logits, rules)
            nxt = torch.where(top < 0, 50256, top)
            if temperature > 0:
                for b in live:
                    if len(prompts[b]) <= at + 1 and int(top[b]) >= 0:
                        kernels.sample(self.model.ctx, out[b], temperature, top_k, rngs[b], nxt[b:b + 1])
            # inside a prompt its own next token stands
            history[:, at + 1] = torch.where(at + 1 < n_prompt, history[:, at + 1], nxt)
            if allowed is not None:
                for b in live:
                    if len(prompts[b]) <= at + 1:
                        texts[b].append(int(history[b, at + 1]))
        done = history.cpu()
        return [done[b, len(p): len(p) + steps].tolist() for b, p in enumerate(prompts)]

    def _cut(self, rows, held, pages, table, weights, pool):
        """Evicts in the sequences `rows` together."""
        idx = torch.tensor(rows, device="cuda")
        new = [pool.take(-(-self.budget // self.page_size)) for _ in rows]
        src = table[idx]
        dst = torch.full_like(src, -1)
        dst[:, : len(new[0])] = torch.tensor(new, dtype=torch.int32, device="cuda")
        lens = torch.tensor([held[b] for b in rows], dtype=torch.int32, device="cuda")
        _, kept, _ = self.cache.evict(src, lens, self.cap, weights[:, idx].contiguous(), self.budget, dst,
                                      sinks=self.sinks, recent=self.recent, n_layers=self.model.n_layer)
        fresh = torch.zeros_like(weights[:, idx])
        fresh[..., : self.budget] = kept
        weights[:, idx] = fresh
        table[idx] = dst
        for b, p in zip(rows, new):
            pool.give(pages[b])
            pages[b] = p
            held[b] = self.budget

    def free(self):
        self.batch.free()
        self.cache.free()


def pack_mask(ok):
    """bool [n, V] -> int32 [n, ceil(V / 32)], bit t % 32 of word t // 32."""
    n, V = ok.shape
    bits = torch.zeros(n, (V + 31) // 32 * 32, dtype=torch.int64)
    bits[:, :V] = ok
    words = (bits.view(n, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def main():
    from . import synth
    from .tensor import Context

    ctx = Context(0)
    model = Model(ctx, synth.gpt2_random_init(0, n_layer=2), n_layer=2, max_t=64)
    gen = PagedGenerator(model, 4, limit=32, budget=16, recent=8)
    prompts = [[50256], [11, 22, 33], list(range(100, 140))]
    print("greedy:   ", gen.generate(prompts, 8))
    print("penalties:", gen.generate(prompts, 8, repetition=1.3, frequency=0.2))
    even = torch.zeros(3, model.V, dtype=torch.bool)
    even[:, ::2] = True
    print("even ids: ", gen.generate(prompts, 8, allowed=lambda at, texts: even, temperature=0.8))
    gen.free()


if __name__ == "__main__":
    main()
