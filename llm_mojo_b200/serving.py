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
from dataclasses import dataclass

import torch

from ._lib import KV_BF16, KV_F32, KV_QUANT8, OK, check, lib
from .tensor import Context

F32, I32 = torch.float32, torch.int32

KINDS = {"int8": KV_QUANT8, "bf16": KV_BF16, "f32": KV_F32}


def _check(ctx: Context, name: str, t, dtype, ndim: int, inner: int = 1):
    """t as the call takes it: on the context's device, `dtype`, `ndim`
    dimensions of which the last `inner` are contiguous. Returns its address."""
    if t.dtype is not dtype or t.dim() != ndim or t.get_device() != ctx.device or not (
            t.is_contiguous() or _rows_contiguous(t, inner)):
        raise ValueError(f"{name} must be {dtype} on cuda:{ctx.device} with {ndim} dimensions, the last {inner} "
                         f"contiguous; not {t.dtype} on {t.device}, {tuple(t.shape)} with strides {t.stride()}")
    return t.data_ptr()


def _rows_contiguous(t, inner: int) -> bool:
    want = 1
    for n, stride in zip(reversed(t.shape[-inner:]), reversed(t.stride()[-inner:])):
        if n != 1 and stride != want:
            return False
        want *= n
    return True


def _row_stride(name: str, t) -> int:
    """The distance of t's rows [..., row] from one another, which must be the
    same over all leading dimensions; a dimension of one has no say."""
    if t.is_contiguous():
        return t.shape[-1]
    step, rows = None, 1
    for n, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n != 1:
            if step is None:
                step = stride
            elif stride != step * rows:
                raise ValueError(f"{name} must have evenly spaced rows")
        rows *= n
    return t.shape[-1] if step is None else step


def _shape(name: str, t, want):
    if t.shape != want:
        raise ValueError(f"{name} must be {tuple(want)}, not {tuple(t.shape)}")


def _call(ctx: Context, fn, *args):
    """fn(ctx, *args) in order with torch's current stream."""
    if ctx.on_torch_stream():
        status = fn(ctx.h, *args)
        if status != OK:
            check(status, ctx.h)
    else:
        torch.cuda.current_stream(ctx.device).synchronize()
        check(fn(ctx.h, *args), ctx.h)
        ctx.sync()


class PagedKVCache:
    """The pages of one cache, for all its sequences: kind 'int8' (codes with
    a float32 scale per position and head, QuantKV[8]'s rule), 'bf16' or
    'f32'. k and v are the pool, [n_layer, n_pages, n_kv_head, page_size,
    head_dim]; ks and vs its scales (None without): tensors of torch's
    allocator, not cleared.

    A page table (int32 [n_seqs, n]) gives the page of each run of page_size
    positions; an entry outside the pool (-1) is no page."""

    def __init__(self, ctx: Context, kind: str, n_layer: int, n_pages: int, page_size: int, n_kv_head: int,
                 head_dim: int):
        if kind not in KINDS:
            raise ValueError(f"unknown paged cache kind {kind}")
        self.ctx, self.kind = ctx, kind
        self.n_layer, self.n_pages, self.page_size = n_layer, n_pages, page_size
        self.n_kv_head, self.head_dim, self.scale = n_kv_head, head_dim, 1.0 / max(head_dim, 1) ** 0.5
        if min(n_layer, n_pages, page_size, n_kv_head, head_dim) <= 0 or head_dim > 128 or (
                n_layer * n_pages * n_kv_head * page_size * head_dim > 1 << 39):
            # no such buffers: the library says why
            check(lib().llmq_paged_create(ctx.h, KINDS[kind], n_layer, n_pages, page_size, n_kv_head, head_dim,
                                          C.byref(C.c_void_p())), ctx.h)
        shape = (n_layer, n_pages, n_kv_head, page_size, head_dim)
        at = dict(device=f"cuda:{ctx.device}")
        dtype = {"int8": torch.int8, "bf16": torch.bfloat16, "f32": F32}[kind]
        self.k, self.v = torch.empty(shape, dtype=dtype, **at), torch.empty(shape, dtype=dtype, **at)
        self.ks = self.vs = None
        if kind == "int8":
            self.ks, self.vs = torch.empty(shape[:-1], dtype=F32, **at), torch.empty(shape[:-1], dtype=F32, **at)
        # the buffers again: k and the others are the caller's to keep or drop
        self._buffers = [t for t in (self.k, self.v, self.ks, self.vs) if t is not None]
        ptr = [t.data_ptr() if t is not None else None for t in (self.k, self.v, self.ks, self.vs)]
        h = C.c_void_p()
        check(lib().llmq_paged_create_in(ctx.h, KINDS[kind], n_layer, n_pages, page_size, n_kv_head, head_dim, *ptr,
                                         C.byref(h)), ctx.h)
        self.h = h
        self._store, self._attend = lib().llmq_paged_store, lib().llmq_paged_attend
        self._evict = lib().llmq_paged_evict

    def store(self, layer: int, k, v, pos, table, seq=None):
        """Stores rows k, v [n, n_kv_head, head_dim] (any row stride: the
        columns of a projection will do) at positions pos [n] of sequences seq
        [n] (None: row r is sequence r). A negative position is skipped."""
        ctx, n = self.ctx, k.shape[0]
        kp, vp = _check(ctx, "k", k, F32, 3, 2), _check(ctx, "v", v, F32, 3, 2)
        rows = (n, self.n_kv_head, self.head_dim)
        _shape("k", k, rows)
        _shape("v", v, rows)
        pp = _check(ctx, "pos", pos, I32, 1)
        _shape("pos", pos, (n,))
        sp = None
        if seq is not None:
            sp = _check(ctx, "seq", seq, I32, 1)
            _shape("seq", seq, (n,))
        tp = _check(ctx, "table", table, I32, 2)
        _call(ctx, self._store, self.h, layer, kp, k.stride(0), vp, v.stride(0), sp, pp, n, tp,
              table.stride(0), table.shape[1], table.shape[0])

    def attend(self, layer: int, q, table, lens, max_len: int, scale: float | None = None, out=None, weights=None,
               weights_out=None):
        """Attention of q [n_seqs, n_head, head_dim], one new token per
        sequence, over its first lens[b] <= max_len positions; returns out of
        q's shape. scale: 1 / sqrt(head_dim) unless given. With weights
        and/or weights_out ([n_seqs, n_kv_head, >= max_len], of one layout;
        weights_out = weights for in place), weights_out = weights + the
        softmax weights summed over each kv head's query heads."""
        ctx = self.ctx
        qp = _check(ctx, "q", q, F32, 3, 2)
        n, n_head, dim = q.shape
        if dim != self.head_dim:
            raise ValueError(f"q must have {self.head_dim} dimensions a head, not {dim}")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
            op = out.data_ptr()
        else:
            op = _check(ctx, "out", out, F32, 3, 2)
            _shape("out", out, q.shape)
        tp, lp = _check(ctx, "table", table, I32, 2), _check(ctx, "lens", lens, I32, 1)
        if lens.shape[0] != n or table.shape[0] != n:
            raise ValueError("table, lens and q must have a row per sequence")
        wp = wop = None
        stride = 0
        if weights_out is None:
            if weights is not None:
                raise ValueError("weights without weights_out")
        else:
            wop = _check(ctx, "weights_out", weights_out, F32, 3)
            stride = _row_stride("weights_out", weights_out)
            shape = weights_out.shape
            if shape[0] != n or shape[1] != self.n_kv_head or shape[2] < max_len:
                raise ValueError(f"weights_out must be [{n}, {self.n_kv_head}, >= {max_len}]")
            if weights is not None:
                wp = _check(ctx, "weights", weights, F32, 3)
                if weights.shape != shape or _row_stride("weights", weights) != stride:
                    raise ValueError("weights must have the shape and strides of weights_out")
        _call(ctx, self._attend, self.h, layer, qp, q.stride(0), op, out.stride(0), n, n_head, tp,
              table.stride(0), table.shape[1], lp, max_len, self.scale if scale is None else scale, wp, wop, stride)
        return out

    def evict(self, table, lens, max_len: int, weights, budget: int, dst_table, sinks: int = 0, recent: int = 0,
              layer0: int = 0, n_layers: int | None = None):
        """Bounds every (layer, sequence, head) to `budget` positions: the
        first `sinks`, the last `recent`, and those of the largest weights
        [n_layers, n_seqs, n_kv_head, >= max_len]; their rows move in order to
        dst_table's pages, which must not be the source's. Returns (kept
        positions int32 [n_layers, n_seqs, n_kv_head, budget], -1 past the
        kept; their weights, 0 past them; the new lengths int32 [n_seqs], -1
        for a sequence that would keep a position without a page: it is
        refused, and attended to with that length it is empty)."""
        ctx, n = self.ctx, table.shape[0]
        n_layers = self.n_layer - layer0 if n_layers is None else n_layers
        tp, lp = _check(ctx, "table", table, I32, 2), _check(ctx, "lens", lens, I32, 1)
        dp = _check(ctx, "dst_table", dst_table, I32, 2)
        _shape("lens", lens, (n,))
        if dst_table.shape[0] != n:
            raise ValueError("table and dst_table must have a row per sequence")
        wp = _check(ctx, "weights", weights, F32, 4)
        if tuple(weights.shape[:3]) != (n_layers, n, self.n_kv_head) or weights.shape[3] < max_len:
            raise ValueError(f"weights must be [{n_layers}, {n}, {self.n_kv_head}, >= {max_len}]")
        ws = _row_stride("weights", weights)
        if budget <= 0:
            raise ValueError("budget must be positive")
        rows = (n_layers, n, self.n_kv_head, budget)
        kept, wout, lens_out = lens.new_empty(rows), weights.new_empty(rows), torch.empty_like(lens)
        _call(ctx, self._evict, self.h, layer0, n_layers, n, tp, table.stride(0), table.shape[1], lp, max_len,
              wp, ws, budget, sinks, recent, dp, dst_table.stride(0), dst_table.shape[1], kept.data_ptr(),
              wout.data_ptr(), budget, lens_out.data_ptr())
        return kept, wout, lens_out

    def free(self):
        """Gives the buffers back to torch once the context's stream is done
        with them."""
        if getattr(self, "h", None):
            if self.ctx.h:
                self.ctx.sync()
            lib().llmq_paged_free(self.h)
            self.h = None
        self.k = self.v = self.ks = self.vs = None
        self._buffers = []

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
        r = _Rules()

        def per_row(name, t, dtype):
            p = _check(ctx, name, t, dtype, 1)
            if t.shape[0] != n:
                raise ValueError(f"{name} must have a value per row of logits")
            return p

        if self.repetition is not None:
            r.repetition = per_row("repetition", self.repetition, F32)
        if self.presence is not None:
            r.presence = per_row("presence", self.presence, F32)
        if self.frequency is not None:
            r.frequency = per_row("frequency", self.frequency, F32)
        if self.n_ids is not None:
            r.n_ids = per_row("n_ids", self.n_ids, I32)
        if self.n_prompt is not None:
            r.n_prompt = per_row("n_prompt", self.n_prompt, I32)
        if self.ids is not None:
            if self.ids.shape[0] != n:
                raise ValueError("ids must have a row per row of logits")
            # an empty tensor has no address: any valid one will do for no elements
            r.ids = _check(ctx, "ids", self.ids, I32, 2) or r.n_ids
            r.ids_stride, r.max_ids = self.ids.stride(0), self.ids.shape[1]
        if self.bias is not None:
            off, ids, val = self.bias
            r.bias_offsets = _check(ctx, "bias offsets", off, I32, 1)
            r.bias_ids = _check(ctx, "bias ids", ids, I32, 1) or r.bias_offsets
            r.bias_values = _check(ctx, "bias values", val, F32, 1) or r.bias_offsets
            _shape("bias offsets", off, (n + 1,))
            _shape("bias values", val, ids.shape)
            r.n_bias = ids.shape[0]
        if self.mask is not None:
            r.mask = _check(ctx, "mask", self.mask, I32, 2)
            if self.mask.shape[0] != n or self.mask.shape[1] < (V + 31) // 32:
                raise ValueError(f"mask must be [{n}, >= {(V + 31) // 32}]")
            r.mask_stride = self.mask.stride(0)
        return r


def process_logits(ctx: Context, logits, rules: LogitRules, out=None, argmax=None):
    """The rules on logits [n, V]: returns (out [n, V], argmax int32 [n]: the
    first index of each row's largest logit, -1 where nothing is left). out
    may be logits."""
    lp = _check(ctx, "logits", logits, F32, 2)
    n, V = logits.shape
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((n, V))
        op = out.data_ptr()
    else:
        op = _check(ctx, "out", out, F32, 2)
        _shape("out", out, (n, V))
    if argmax is None:
        argmax = torch.empty(n, dtype=I32, device=logits.device)
        ap = argmax.data_ptr()
    else:
        ap = _check(ctx, "argmax", argmax, I32, 1)
        _shape("argmax", argmax, (n,))
    _call(ctx, lib().llmq_process_logits, lp, logits.stride(0), op, out.stride(0), n, V,
          C.byref(rules._struct(ctx, n, V)), ap)
    return out, argmax
