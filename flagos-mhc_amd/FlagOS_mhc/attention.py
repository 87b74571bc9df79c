"""Attention of an mHC model's attention sublayer, forward and backward.

    out_i = sum_j softmax_j(scale q_i . k_j) v_j

over the keys j of i's sequence, under ``causal`` those up to its own place:
where a sequence has Lq queries and Lk keys, the queries are its last Lq
positions, so j <= i + Lk - Lq.  Query heads in groups share a key head: head
h goes with key head h / (H / Hk).

Queries are packed rows (T, H, d) with the sequences' starts in cu_seqlens, or
equally long sequences (B, S, H, d) ((T, H, d) without cu_seqlens is one
sequence); keys and values likewise, a batch of them with lengths_k: a cache
of which each sequence uses its first rows.  Prompts, training batches and
single tokens over a cache are all this call.

fp32 with d up to 128, bf16 and fp16 up to 256.  Scores, maxima and sums are
fp32; the weights exp(..), and in the backward the gradients of the scores, are
rounded to the operands' type for the product that follows, in fp16 times powers
of two that leave them all bits: a forward's weights down to 2^-21 of their
query's largest, a backward's to 2^-28, and the scores' gradients to 2^-22 of the
largest of their query (grad_q) or key (grad_k).  q, k, v may be views with any
strides of their rows and heads; rows that are not at multiples of 16 bytes, or
d that is not whole 16 bytes, are copied in every call.  The reference has no
such operator: its model code runs PyTorch's.
"""

from __future__ import annotations

import functools
import math
import struct

import torch

from . import _lib

_ARGS = struct.Struct("3P9q3P2q6ifi")  # mhc_attention_args (include/mhc_amd.h)
_STRIDES = struct.Struct("3q")
_MAX_ROW_BYTES = 1 << 24
_MAX_SCALE = torch.finfo(torch.float32).max * math.log(2.0)  # scale * log2(e) is a fp32 number
_INTS = (torch.int32, torch.int64)


def _rows(t, shape, es):
    """(t, its address, (sequence, row, head) strides): t as the kernels take it,
    a copy where its strides or address are not whole 16 bytes."""
    H, d = shape[-2], shape[-1]
    at = t.data_ptr()
    if t.is_contiguous():
        if not at & 15 and H * d * es <= _MAX_ROW_BYTES:
            return t, at, (shape[1] * H * d if len(shape) == 4 else 0, H * d, d)
    else:
        st = t.stride()
        row = st[-3] if shape[-3] > 1 else H * d
        head = st[-2] if H > 1 else d
        batch = st[0] if len(shape) == 4 and shape[0] > 1 else 0
        if not ((st[-1] != 1 and d > 1) or (row | head | batch) & (16 // es - 1) or at & 15 or row < d
                or row * es > _MAX_ROW_BYTES):
            return t, at, (batch, row, head)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), (shape[1] * H * d if len(shape) == 4 else 0, H * d, d)


@functools.lru_cache(maxsize=1024)
def _workspace_size(name, dev_index, packed_q, packed_k, *sizes):
    """A *_workspace_size query: a function of the sizes and the device alone."""
    rows_q, rows_k, B, H, Hk, wide, code = sizes
    row = wide  # (the strides have to pass the checks, no more)
    args = _ARGS.pack(16, 16, 16, 0, row, wide, 0, row, wide, 0, row, wide, 16 if packed_q else 0, 16 if packed_k else 0, 0,
                      rows_q, rows_k, B, H, Hk, wide, code, 1, 1.0, 0)
    with torch.cuda.device(dev_index):
        return int(getattr(_lib.load(), name)(args))


class _Call:
    """The checked operands of a call."""

    __slots__ = ("keep", "H", "Hk", "d", "wide", "es", "code", "rows_q", "rows_k", "args", "sizes")

    def __init__(self, what, q, k, v, cu_q, cu_k, lengths, causal, scale):
        dt = q.dtype
        code = self.code = _lib.dtype_code(what, dt)
        if k.dtype is not dt or v.dtype is not dt:
            raise ValueError(f"{what}: q is {dt}, k {k.dtype} and v {v.dtype}, expected one type")
        qs, ks = q.shape, k.shape
        nq, nk = len(qs), len(ks)
        if nq not in (3, 4) or nk not in (3, 4) or v.shape != ks or ks[-1] != qs[-1]:
            raise ValueError(f"{what}: q {tuple(qs)}, k {tuple(ks)} and v {tuple(v.shape)} do not fit")
        H, d, Hk = qs[-2], qs[-1], ks[-2]
        if H < 1 or Hk < 1 or H % Hk or d < 1:
            raise ValueError(f"{what}: {H} query heads of {d} in groups of {Hk} key heads")
        if d > (128 if code == 0 else 256):
            raise NotImplementedError(f"{what}: head width {d} not supported (at most 256, in fp32 128)")
        if scale is None:
            scale = d ** -0.5
        elif not 0.0 < scale <= _MAX_SCALE:
            raise ValueError(f"{what}: scale {scale}, expected a positive number of at most {_MAX_SCALE:.4g}")
        at_q = at_k = at_n = 0
        if cu_q is not None:
            if nq != 3:
                raise ValueError(f"{what}: cu_seqlens goes with packed rows (T, H, d), q is {tuple(qs)}")
            if cu_k is None and nk == 3 and lengths is None:
                if ks[0] != qs[0]:
                    raise ValueError(f"{what}: {ks[0]} packed keys for {qs[0]} queries need cu_seqlens_k")
                cu_k = cu_q
            same = cu_k is cu_q
            cu_q = _lib.cu_operand(what, "cu_seqlens", cu_q)
            if same:
                cu_k = cu_q
            B = cu_q.shape[0] - 1
            at_q = cu_q.data_ptr()
        else:
            B = qs[0] if nq == 4 else 1
        if cu_k is not None:
            if nk != 3 or lengths is not None:
                raise ValueError(f"{what}: cu_seqlens_k goes with packed keys (T, Hk, d) and no lengths_k, k is {tuple(ks)}")
            if cu_k is not cu_q:
                cu_k = _lib.cu_operand(what, "cu_seqlens_k", cu_k)
            Bk = cu_k.shape[0] - 1
            at_k = cu_k.data_ptr()
        else:
            Bk = ks[0] if nk == 4 else 1
        if Bk != B:
            raise ValueError(f"{what}: {B} sequences of queries and {Bk} of keys")
        if lengths is not None:
            if lengths.dim() != 1 or lengths.shape[0] != B or lengths.dtype not in _INTS:
                raise ValueError(f"{what}: lengths_k of shape {tuple(lengths.shape)} and {lengths.dtype} for {B} sequences")
            if lengths.dtype is not torch.int32 or not lengths.is_contiguous():
                lengths = _lib.operand(lengths, (B,), torch.int32)
            at_n = lengths.data_ptr()
        es = self.es = 4 if code == 0 else 2
        wide = self.wide = -(-d * es // 16) * 16 // es  # d in whole 16 bytes
        self.H, self.Hk, self.d = H, Hk, d
        if wide == d:
            q, pq, qst = _rows(q, qs, es)
            k, pk, kst = _rows(k, ks, es)
            v, pv, vst = _rows(v, ks, es)
        else:
            (q, pq, qst), (k, pk, kst), (v, pv, vst) = self.take(q), self.take(k), self.take(v)
        rows_q = self.rows_q = qs[0] if nq == 3 else qs[0] * qs[1]
        rows_k = self.rows_k = ks[0] if nk == 3 else ks[0] * ks[1]
        self.keep = (q, k, v, cu_q, cu_k, lengths)  # as long as their addresses are used
        self.sizes = (at_q != 0, at_k != 0, rows_q, rows_k, B, H, Hk, wide, code)
        self.args = _ARGS.pack(pq, pk, pv, *qst, *kst, *vst, at_q, at_k, at_n, rows_q, rows_k, B, H, Hk, wide, code,
                               1 if causal else 0, scale, 0)

    def take(self, t):
        """_rows of a tensor in the call's width."""
        if self.wide != self.d:
            t = torch.nn.functional.pad(t, (0, self.wide - self.d))
        return _rows(t, t.shape, self.es)

    def empty(self, like):
        if self.wide == self.d:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        return like.new_empty(like.shape[:-1] + (self.wide,))

    def trim(self, t):
        return t if self.wide == self.d else t[..., :self.d].contiguous()

    def workspace(self, name, dev_index, like):
        n = _workspace_size(name, dev_index, *self.sizes)
        return (like.new_empty(n, dtype=torch.uint8), n) if n else (None, 0)


def attention(q, k, v, cu_seqlens=None, *, cu_seqlens_k=None, lengths_k=None, causal=True, scale=None,
              need_backward=False):
    """Attention on the HIP device.  Returns a dict with out (q's shape and
    dtype) and, with ``need_backward``, lse (H, rows of q) fp32.

    q (T, H, d) with cu_seqlens (B + 1,) int32 on the device, its first entry 0,
    or (B, S, H, d); k, v (Tk, Hk, d) with cu_seqlens_k (by default
    cu_seqlens), or (B, Sk, Hk, d), of which lengths_k (B,) rows count (by
    default all; rows past them are not read).  scale > 0, by default d^-1/2.
    Queries that see no key, and rows behind the last packed sequence, get out
    0 (lse -infinity).  Nothing is copied to the host: the starts and lengths
    may change between replays of a captured graph."""
    what = "attention"
    _lib.require_device(what, q, k, v, cu_seqlens, cu_seqlens_k, lengths_k)
    c = _Call(what, q, k, v, cu_seqlens, cu_seqlens_k, lengths_k, causal, scale)
    out = c.empty(q)
    res = {"out": out}
    lse = None
    if need_backward:
        lse = res["lse"] = q.new_empty((c.H, c.rows_q), dtype=torch.float32)
    if c.rows_q > 0:
        dev = q.get_device()
        ws, n = c.workspace("mhc_attention_fwd_workspace_size", dev, q)
        _lib.call(what, _lib.load().mhc_attention_fwd, dev, c.args, out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), n)
    if c.wide != c.d:
        res["out"] = c.trim(out)
    return res


def attention_backward(grad_out, q, k, v, out, lse, cu_seqlens=None, *, cu_seqlens_k=None, lengths_k=None, causal=True,
                       scale=None, need_kv=True):
    """(grad_q, grad_k, grad_v) from the forward's out and lse, in the shapes
    and dtype of q, k and v; the last two are None with ``need_kv=False``.  Rows
    of no sequence, and of a cache past its lengths, get 0.  Deterministic."""
    what = "attention_backward"
    _lib.require_device(what, grad_out, q, k, v, out, lse, cu_seqlens, cu_seqlens_k, lengths_k)
    c = _Call(what, q, k, v, cu_seqlens, cu_seqlens_k, lengths_k, causal, scale)
    if grad_out.shape != q.shape or out.shape != q.shape or out.dtype is not q.dtype:
        raise ValueError(f"{what}: grad_out {tuple(grad_out.shape)} and out {tuple(out.shape)} {out.dtype} for q "
                         f"{tuple(q.shape)} {q.dtype}")
    if tuple(lse.shape) != (c.H, c.rows_q) or lse.dtype is not torch.float32:
        raise ValueError(f"{what}: lse of shape {tuple(lse.shape)} and {lse.dtype}, expected {(c.H, c.rows_q)} of float32")
    if not lse.is_contiguous():
        lse = lse.contiguous()
    go, at_go, gst = c.take(grad_out if grad_out.dtype is q.dtype else grad_out.to(q.dtype))
    o, at_o, _ = c.take(out if out.is_contiguous() else out.contiguous())
    dq, dk, dv = c.empty(q), c.empty(k) if need_kv else None, c.empty(v) if need_kv else None
    if c.rows_q > 0 or (need_kv and c.rows_k > 0):
        dev = q.get_device()
        if need_kv:
            ws, n = c.workspace("mhc_attention_bwd_workspace_size", dev, q)
        else:
            n = -(-c.H * c.rows_q * 4 // 256) * 256
            ws = q.new_empty(n, dtype=torch.uint8)
        _lib.call(what, _lib.load().mhc_attention_bwd, dev, c.args, at_go, _STRIDES.pack(*gst), at_o, lse.data_ptr(),
                  dq.data_ptr(), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(ws), n)
    if c.wide != c.d:
        dq, dk, dv = (None if t is None else c.trim(t) for t in (dq, dk, dv))
    return dq, dk, dv


def attention_ref(q, k, v, cu_seqlens=None, *, cu_seqlens_k=None, lengths_k=None, causal=True, scale=None):
    """The same in PyTorch, fp32 math, cast to q's dtype, sequence by sequence
    (reads the starts and lengths on the host)."""
    d, G = q.shape[-1], q.shape[-2] // k.shape[-2]
    scale = d ** -0.5 if scale is None else scale
    cu_k = cu_seqlens if cu_seqlens_k is None and cu_seqlens is not None and k.dim() == 3 and lengths_k is None else cu_seqlens_k

    def parts(t, cu, lengths=None):
        if cu is not None:
            at = [0] + cu.tolist()[1:]
            return [t[a:b] for a, b in zip(at, at[1:])]
        t = t if t.dim() == 4 else t[None]
        return list(t) if lengths is None else [s[:n] for s, n in zip(t, lengths.tolist())]

    outs = []
    for qi, ki, vi in zip(parts(q, cu_seqlens), parts(k, cu_k, lengths_k), parts(v, cu_k, lengths_k)):
        n, m = qi.shape[0], ki.shape[0]
        qf, kf, vf = (t.float().transpose(0, 1) for t in (qi, ki.repeat_interleave(G, 1), vi.repeat_interleave(G, 1)))
        score = (qf @ kf.transpose(1, 2)) * scale
        hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
        if causal:
            hidden = torch.arange(m, device=q.device)[None] > torch.arange(n, device=q.device)[:, None] + (m - n)
        score = score.masked_fill(hidden, -math.inf)
        p = torch.softmax(score, -1).masked_fill(hidden.all(-1)[:, None] if m else hidden, 0.0)
        outs.append((p @ vf).transpose(0, 1).to(q.dtype))
    if cu_seqlens is None:
        return torch.stack(outs).reshape(q.shape) if outs else torch.zeros_like(q)
    rest = q.shape[0] - sum(o.shape[0] for o in outs)
    return torch.cat([*outs, q.new_zeros((rest, *q.shape[1:]))])


class AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens=None, cu_seqlens_k=None, lengths_k=None, causal=True, scale=None):
        f = attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k, lengths_k=lengths_k, causal=causal, scale=scale,
                      need_backward=True)
        ctx.save_for_backward(q, k, v, f["out"], f["lse"], cu_seqlens, cu_seqlens_k, lengths_k)
        ctx.args = dict(causal=causal, scale=scale)
        return f["out"]

    @staticmethod
    def backward(ctx, grad_out):
        q, k, v, out, lse, cu, cu_k, lengths = ctx.saved_tensors
        grads = attention_backward(grad_out, q, k, v, out, lse, cu, cu_seqlens_k=cu_k, lengths_k=lengths, **ctx.args,
                                   need_kv=any(ctx.needs_input_grad[1:3]))
        return (*_lib.first_order("attention", grads, grad_out, q, k, v), None, None, None, None, None)


def attention_fn(q, k, v, cu_seqlens=None, *, cu_seqlens_k=None, lengths_k=None, causal=True, scale=None):
    """Autograd-aware attention: out.  Without gradients to take, nothing is
    saved."""
    if not _lib.needs_autograd(q, k, v):
        return attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k, lengths_k=lengths_k, causal=causal,
                         scale=scale)["out"]
    return AttentionFn.apply(q, k, v, cu_seqlens, cu_seqlens_k, lengths_k, causal, scale)


def projected_width(what, heads, w_q, w_k, w_v):
    """The head width of projections (heads * d, D), (heads_k * d, D) twice."""
    if heads < 1 or w_q.dim() != 2 or w_q.shape[0] % heads or w_q.shape[0] < heads:
        raise ValueError(f"{what}: w_q of shape {tuple(w_q.shape)} for {heads} heads")
    d = w_q.shape[0] // heads
    if w_k.dim() != 2 or w_k.shape[0] % d or w_k.shape[0] < d or w_v.shape != w_k.shape:
        raise ValueError(f"{what}: w_k of shape {tuple(w_k.shape)} and w_v of {tuple(w_v.shape)} for heads of {d}")
    return d
