"""Serving operators on device tensors: a KV cache in pages for sequences of
any lengths (store, attention of one new token per sequence, eviction by
accumulated attention weight) and the rules between the head and the sampler.

Arguments are torch CUDA tensors of the context's device (float32 values,
int32 ids, lengths and tables). Calls are issued on the context's stream. On
torch's current stream (Context.use_torch_stream) they are asynchronous, like
torch's own; on another stream they are synchronised with torch's before and
after, as the kernels layer's are.
"""

from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

from ._lib import KV_BF16, KV_F32, KV_QUANT8, check, lib
from .tensor import Context

KINDS = {"int8": KV_QUANT8, "bf16": KV_BF16, "f32": KV_F32}


class _Array:
    """A device buffer of the library as torch.as_tensor takes it; holds its
    owner, so that views outlive no storage."""

    def __init__(self, owner, ptr: int, shape, typestr: str):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 3}


def _check(ctx: Context, name: str, t, dtype, ndim: int, inner: int = 1):
    """t as the call takes it: on the context's device, `dtype`, `ndim`
    dimensions of which the last `inner` are contiguous."""
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} must be on cuda:{ctx.device}, not {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")
    want = 1
    for i in range(ndim - 1, ndim - 1 - inner, -1):
        if t.shape[i] != 1 and t.stride(i) != want:
            raise ValueError(f"{name}: the last {inner} dimensions must be contiguous")
        want *= t.shape[i]
    return t.data_ptr()


def _shape(name: str, t, want):
    if tuple(t.shape) != tuple(want):
        raise ValueError(f"{name} must be {tuple(want)}, not {tuple(t.shape)}")


class _Ordered:
    """Orders a call with torch's current stream."""

    def __init__(self, ctx: Context):
        self.ctx = ctx

    def __enter__(self):
        import torch

        self.same = self.ctx.on_torch_stream()
        if not self.same:
            torch.cuda.current_stream(self.ctx.device).synchronize()

    def __exit__(self, *exc):
        if not self.same:
            self.ctx.sync()


class PagedKVCache:
    """The pages of one cache, for all its sequences: kind 'int8' (codes with
    a float32 scale per position and head, QuantKV[8]'s rule), 'bf16' or
    'f32'. k and v are torch views of the pool, [n_layer, n_pages, n_kv_head,
    page_size, head_dim]; ks and vs of its scales (None without).

    A page table (int32 [n_seqs, n]) gives the page of each run of page_size
    positions; an entry outside the pool (-1) is no page."""

    def __init__(self, ctx: Context, kind: str, n_layer: int, n_pages: int, page_size: int, n_kv_head: int,
                 head_dim: int):
        import torch

        if kind not in KINDS:
            raise ValueError(f"unknown paged cache kind {kind}")
        self.ctx, self.kind = ctx, kind
        self.n_layer, self.n_pages, self.page_size = n_layer, n_pages, page_size
        self.n_kv_head, self.head_dim = n_kv_head, head_dim
        h = C.c_void_p()
        check(lib().llmq_paged_create(ctx.h, KINDS[kind], n_layer, n_pages, page_size, n_kv_head, head_dim,
                                      C.byref(h)), ctx.h)
        self._storage = _Storage(ctx, h)
        self.h = h
        ptr = [C.c_void_p() for _ in range(4)]
        check(lib().llmq_paged_buffers(h, *[C.byref(p) for p in ptr]))
        shape = (n_layer, n_pages, n_kv_head, page_size, head_dim)
        typestr = {"int8": "|i1", "bf16": "<i2", "f32": "<f4"}[kind]

        def view(p, shape, typestr):
            return torch.as_tensor(_Array(self._storage, p.value, shape, typestr), device=f"cuda:{ctx.device}")

        self.k, self.v = view(ptr[0], shape, typestr), view(ptr[1], shape, typestr)
        if kind == "bf16":
            self.k, self.v = self.k.view(torch.bfloat16), self.v.view(torch.bfloat16)
        self.ks = self.vs = None
        if kind == "int8":
            self.ks, self.vs = view(ptr[2], shape[:-1], "<f4"), view(ptr[3], shape[:-1], "<f4")

    def store(self, layer: int, k, v, pos, table, seq=None):
        """Stores rows k, v [n, n_kv_head, head_dim] (any row stride: the
        columns of a projection will do) at positions pos [n] of sequences seq
        [n] (None: row r is sequence r). A negative position is skipped."""
        import torch

        ctx, n = self.ctx, k.shape[0]
        kp, vp = _check(ctx, "k", k, torch.float32, 3, 2), _check(ctx, "v", v, torch.float32, 3, 2)
        _shape("k", k, (n, self.n_kv_head, self.head_dim))
        _shape("v", v, (n, self.n_kv_head, self.head_dim))
        pp = _check(ctx, "pos", pos, torch.int32, 1)
        _shape("pos", pos, (n,))
        sp = None
        if seq is not None:
            sp = _check(ctx, "seq", seq, torch.int32, 1)
            _shape("seq", seq, (n,))
        tp = _check(ctx, "table", table, torch.int32, 2)
        with _Ordered(ctx):
            check(lib().llmq_paged_store(ctx.h, self.h, layer, kp, k.stride(0), vp, v.stride(0), sp, pp, n, tp,
                                         table.stride(0), table.shape[1], table.shape[0]), ctx.h)

    def attend(self, layer: int, q, table, lens, max_len: int, scale: float | None = None, out=None, weights=None,
               weights_out=None):
        """Attention of q [n_seqs, n_head, head_dim], one new token per
        sequence, over its first lens[b] <= max_len positions; returns out of
        q's shape. scale: 1 / sqrt(head_dim) unless given. With weights
        and/or weights_out ([n_seqs, n_kv_head, >= max_len], weights_out =
        weights for in place), weights_out = weights + the softmax weights
        summed over each kv head's query heads."""
        import torch

        ctx = self.ctx
        qp = _check(ctx, "q", q, torch.float32, 3, 2)
        n, n_head = q.shape[0], q.shape[1]
        _shape("q", q, (n, n_head, self.head_dim))
        if out is None:
            out = torch.empty((n, n_head, self.head_dim), dtype=torch.float32, device=q.device)
        op = _check(ctx, "out", out, torch.float32, 3, 2)
        _shape("out", out, q.shape)
        tp, lp = _check(ctx, "table", table, torch.int32, 2), _check(ctx, "lens", lens, torch.int32, 1)
        _shape("lens", lens, (n,))
        if table.shape[0] != n:
            raise ValueError("table and q must have a row per sequence")
        wp = wop = None
        stride = 0
        if weights is not None and weights_out is None:
            raise ValueError("weights without weights_out")
        if weights_out is not None:
            wop = _check(ctx, "weights_out", weights_out, torch.float32, 3)
            stride = weights_out.stride(1)
            for name, w in (("weights", weights), ("weights_out", weights_out)):
                if w is None:
                    continue
                p = _check(ctx, name, w, torch.float32, 3)
                if tuple(w.shape[:2]) != (n, self.n_kv_head) or w.shape[2] < max_len:
                    raise ValueError(f"{name} must be [{n}, {self.n_kv_head}, >= {max_len}]")
                if w.stride(1) != stride or (n > 1 and w.stride(0) != stride * self.n_kv_head):
                    raise ValueError("weights and weights_out must have the same evenly spaced rows")
                if name == "weights":
                    wp = p
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)
        with _Ordered(ctx):
            check(lib().llmq_paged_attend(ctx.h, self.h, layer, qp, q.stride(0), op, out.stride(0), n, n_head, tp,
                                          table.stride(0), table.shape[1], lp, max_len, scale, wp, wop, stride), ctx.h)
        return out

    def evict(self, table, lens, max_len: int, weights, budget: int, dst_table, sinks: int = 0, recent: int = 0,
              layer0: int = 0, n_layers: int | None = None):
        """Bounds every (layer, sequence, head) to `budget` positions: the
        first `sinks`, the last `recent`, and those of the largest weights
        [n_layers, n_seqs, n_kv_head, >= max_len]; their rows move in order to
        dst_table's pages, which must not be the source's. Returns (kept
        positions int32 [n_layers, n_seqs, n_kv_head, budget], -1 past the
        kept; their weights, 0 past them; the new lengths int32 [n_seqs])."""
        import torch

        ctx, n = self.ctx, table.shape[0]
        n_layers = self.n_layer - layer0 if n_layers is None else n_layers
        tp, lp = _check(ctx, "table", table, torch.int32, 2), _check(ctx, "lens", lens, torch.int32, 1)
        dp = _check(ctx, "dst_table", dst_table, torch.int32, 2)
        _shape("lens", lens, (n,))
        if dst_table.shape[0] != n:
            raise ValueError("table and dst_table must have a row per sequence")
        wp = _check(ctx, "weights", weights, torch.float32, 4)
        if tuple(weights.shape[:3]) != (n_layers, n, self.n_kv_head) or weights.shape[3] < max_len:
            raise ValueError(f"weights must be [{n_layers}, {n}, {self.n_kv_head}, >= {max_len}]")
        ws = weights.stride(2)
        if (n > 1 and weights.stride(1) != ws * self.n_kv_head) or (
                n_layers > 1 and weights.stride(0) != ws * self.n_kv_head * n):
            raise ValueError("weights must have evenly spaced rows")
        if budget <= 0:
            raise ValueError("budget must be positive")
        rows = (n_layers, n, self.n_kv_head, budget)
        kept = torch.empty(rows, dtype=torch.int32, device=weights.device)
        wout = torch.empty(rows, dtype=torch.float32, device=weights.device)
        lens_out = torch.empty(n, dtype=torch.int32, device=weights.device)
        with _Ordered(ctx):
            check(lib().llmq_paged_evict(ctx.h, self.h, layer0, n_layers, n, tp, table.stride(0), table.shape[1], lp, max_len,
                                         wp, ws, budget, sinks, recent, dp, dst_table.stride(0), dst_table.shape[1],
                                         kept.data_ptr(), wout.data_ptr(), budget, lens_out.data_ptr()), ctx.h)
        return kept, wout, lens_out

    def free(self):
        """Releases the pool; its views must not be used any more."""
        self.k = self.v = self.ks = self.vs = None
        self._storage.free()
        self.h = None


class _Storage:
    """Owns a llmq_paged handle."""

    def __init__(self, ctx: Context, h):
        self.ctx, self.h = ctx, h

    def free(self):
        if self.h:
            lib().llmq_paged_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class _Rules(C.Structure):
    _fields_ = [("repetition", C.c_void_p), ("presence", C.c_void_p), ("frequency", C.c_void_p), ("ids", C.c_void_p),
                ("n_ids", C.c_void_p), ("n_prompt", C.c_void_p), ("ids_stride", C.c_longlong),
                ("max_ids", C.c_int), ("n_bias", C.c_int),
                ("bias_offsets", C.c_void_p), ("bias_ids", C.c_void_p), ("bias_values", C.c_void_p),
                ("mask", C.c_void_p), ("mask_stride", C.c_longlong)]


@dataclass
class LogitRules:
    """What may change the logits of n rows; None leaves a rule out.

    ids int32 [n, m] with n_ids int32 [n]: each row's history, of which the
    first n_prompt int32 [n] tokens (None: none) are the prompt. repetition,
    presence, frequency float32 [n]: the penalties. bias: (offsets int32
    [n + 1], ids int32, ascending in a row, values float32). mask int32 [n,
    >= ceil(V / 32)]: bit t % 32 of word t // 32 allows token t."""

    repetition: object = None
    presence: object = None
    frequency: object = None
    ids: object = None
    n_ids: object = None
    n_prompt: object = None
    bias: tuple | None = None
    mask: object = None

    def _struct(self, ctx: Context, n: int, V: int) -> _Rules:
        import torch

        r = _Rules()
        for name, dtype in (("repetition", torch.float32), ("presence", torch.float32), ("frequency", torch.float32),
                            ("n_ids", torch.int32), ("n_prompt", torch.int32)):
            t = getattr(self, name)
            if t is not None:
                setattr(r, name, _check(ctx, name, t, dtype, 1))
                _shape(name, t, (n,))
        if self.ids is not None:
            if self.ids.shape[0] != n:
                raise ValueError("ids must have a row per row of logits")
            # an empty tensor has no address: any valid one will do for no elements
            r.ids = _check(ctx, "ids", self.ids, torch.int32, 2) or r.n_ids
            r.ids_stride, r.max_ids = self.ids.stride(0), self.ids.shape[1]
        if self.bias is not None:
            off, ids, val = self.bias
            r.bias_offsets = _check(ctx, "bias offsets", off, torch.int32, 1)
            r.bias_ids = _check(ctx, "bias ids", ids, torch.int32, 1) or r.bias_offsets
            r.bias_values = _check(ctx, "bias values", val, torch.float32, 1) or r.bias_offsets
            _shape("bias offsets", off, (n + 1,))
            _shape("bias values", val, ids.shape)
            r.n_bias = ids.numel()
        if self.mask is not None:
            r.mask = _check(ctx, "mask", self.mask, torch.int32, 2)
            if self.mask.shape[0] != n or self.mask.shape[1] < (V + 31) // 32:
                raise ValueError(f"mask must be [{n}, >= {(V + 31) // 32}]")
            r.mask_stride = self.mask.stride(0)
        return r


def process_logits(ctx: Context, logits, rules: LogitRules, out=None, argmax=None):
    """The rules on logits [n, V]: returns (out [n, V], argmax int32 [n]: the
    first index of each row's largest logit, -1 where nothing is left). out
    may be logits."""
    import torch

    lp = _check(ctx, "logits", logits, torch.float32, 2)
    n, V = logits.shape
    if out is None:
        out = torch.empty((n, V), dtype=torch.float32, device=logits.device)
    op = _check(ctx, "out", out, torch.float32, 2)
    _shape("out", out, (n, V))
    if argmax is None:
        argmax = torch.empty(n, dtype=torch.int32, device=logits.device)
    ap = _check(ctx, "argmax", argmax, torch.int32, 1)
    _shape("argmax", argmax, (n,))
    r = rules._struct(ctx, n, V)
    with _Ordered(ctx):
        check(lib().llmq_process_logits(ctx.h, lp, logits.stride(0), op, out.stride(0), n, V, C.byref(r), ap), ctx.h)
    return out, argmax
