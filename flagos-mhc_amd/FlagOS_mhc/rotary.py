"""Rotary positions of an attention sublayer's queries and keys, forward and
backward.

    (a, b) -> amplitude (a cos w - b sin w, a sin w + b cos w),  w = position * freqs[i]

for the pairs of a head's first r = 2 len(freqs) elements: (i, i + r/2) in the
"half" layout, (2i, 2i + 1) in the "interleaved" one; elements past r are
copied.  ``rotary_frequencies`` gives freqs, and the amplitude, of the usual
ways to stretch positions.  Angles are reduced in 64 bits, products are fp32.
The reference has no such operator: its model code runs PyTorch's.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib

#: layouts and their codes (include/mhc_amd.h)
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, turns=(1.0, 32.0),
                       device="cuda"):
    """(freqs, amplitude) for ``rotary``: freqs (rotary_dim / 2,) float64 on
    `device`, radians a position, base^(-2i / rotary_dim).  ``scaling``, by
    ``factor`` > 0:
      None      as they are
      "linear"  positions divided by factor
      "ntk"     base * factor^(r / (r - 2)): the slowest pair is stretched by factor, the fastest stays
      "yarn"    pairs that turn less than turns[0] times over original_length positions are stretched by
                factor, those above turns[1] stay, in between by a linear share of their turns;
                amplitude 0.1 ln(factor) + 1 (factor > 1).  (Some model code shares linearly in the
                pair's index: weights trained so need such freqs, which ``rotary`` takes as well)
    """
    what = "rotary_frequencies"
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"{what}: rotary_dim {rotary_dim}, expected an even number of at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"{what}: scaling {scaling!r}, expected one of {SCALINGS}")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"{what}: base {base} and factor {factor}, expected positive numbers")
    if scaling == "ntk" and r > 2:
        base = base * factor ** (r / (r - 2))
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    amplitude = 1.0
    if scaling == "linear":
        f = [v / factor for v in f]
    elif scaling == "yarn":
        low, high = turns
        if not original_length or original_length < 1 or not 0 <= low < high:
            raise ValueError(f"{what}: original_length {original_length} and turns {turns} for yarn")
        keep = [min(1.0, max(0.0, (original_length * v / (2 * math.pi) - low) / (high - low))) for v in f]
        f = [v * s + v / factor * (1 - s) for v, s in zip(f, keep)]
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return torch.tensor(f, dtype=torch.float64, device=device), amplitude


_ARGS = struct.Struct("7P4q2qf8i")  # mhc_rotary_args (include/mhc_amd.h)


def _strided(t, shape):
    """(t, row stride, head stride): t (..., H, d) with its rows one stride apart
    and a head's elements side by side; a copy where it is not so."""
    if not t.is_contiguous():
        st = t.stride()
        if st[-1] == 1 or shape[-1] == 1:
            row = 0
            rows = 1  # of the dimensions seen so far
            for n, s in zip(reversed(shape[:-2]), reversed(st[:-2])):
                if n == 1:
                    continue
                if rows == 1:
                    row = s
                elif s != row * rows:
                    break
                rows *= n
            else:
                return t, row, st[-2]
        t = t.contiguous()
    return t, shape[-2] * shape[-1], shape[-1]


def _run(what, q, k, freqs, positions, cu_seqlens, layout, amplitude, inverse):
    _lib.require_device(what, q, k, freqs, positions, cu_seqlens)
    dt = q.dtype
    code = _lib.dtype_code(what, dt)
    if layout not in LAYOUTS:
        raise ValueError(f"{what}: layout {layout!r}, expected one of {tuple(LAYOUTS)}")
    shape = q.shape
    if len(shape) < 3:
        raise ValueError(f"{what}: q of shape {tuple(shape)}, expected (..., heads, d) with a dimension of tokens")
    H, d = shape[-2], shape[-1]
    if H < 1 or d < 1:
        raise ValueError(f"{what}: q of shape {tuple(shape)} has no heads")
    T = q.numel() // (H * d)
    Hk = 0
    if k is not None:
        ks = k.shape
        if len(ks) != len(shape) or ks[:-2] != shape[:-2] or ks[-1] != d or k.dtype is not dt:
            raise ValueError(f"{what}: k of shape {tuple(ks)} and {k.dtype} for q of {tuple(shape)} and {dt}")
        Hk = ks[-2]
        if Hk < 1:
            raise ValueError(f"{what}: k of shape {tuple(ks)} has no heads")
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or 2 * freqs.shape[0] > d:
        raise ValueError(f"{what}: freqs of shape {tuple(freqs.shape)} and {freqs.dtype}, expected float64 and at most {d // 2}")
    if not freqs.is_contiguous():
        freqs = freqs.contiguous()
    at_p = at_cu = wide = B = 0
    if positions is not None:
        if cu_seqlens is not None:
            raise ValueError(f"{what}: positions and cu_seqlens")
        wide = positions.dtype is torch.int64
        if not (wide or positions.dtype is torch.int32) or positions.numel() != T:
            raise ValueError(f"{what}: positions of shape {tuple(positions.shape)} and {positions.dtype}, expected "
                             f"{T} of int32 or int64")
        if positions.dim() > 1:
            at = [n for n in positions.shape if n != 1]
            if len(at) > 1 and at != [n for n in shape[:-2] if n != 1]:
                raise ValueError(f"{what}: positions of shape {tuple(positions.shape)} for rows {tuple(shape[:-2])}")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        at_p = positions.data_ptr()
    elif cu_seqlens is not None:
        if len(shape) != 3:
            raise ValueError(f"{what}: cu_seqlens goes with packed rows (T, heads, d), q is {tuple(shape)}")
        cu_seqlens = _lib.cu_operand(what, "cu_seqlens", cu_seqlens)
        at_cu, B = cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1
    qs, q_row, q_head = _strided(q, shape)
    qo = torch.empty_like(qs, memory_format=torch.contiguous_format)
    at_k = at_ko = k_row = k_head = 0
    ko = None
    if k is not None:
        ks, k_row, k_head = _strided(k, ks)
        ko = torch.empty_like(ks, memory_format=torch.contiguous_format)
        at_k, at_ko = ks.data_ptr(), ko.data_ptr()
    if T > 0:
        args = _ARGS.pack(qs.data_ptr(), at_k, qo.data_ptr(), at_ko, freqs.data_ptr(), at_p, at_cu, q_row, q_head, k_row, k_head,
                          T, shape[-3], amplitude, B, code, H, Hk, d, 2 * freqs.shape[0], LAYOUTS[layout],
                          wide | inverse << 1)
        _lib.call(what, _lib.load().mhc_rotary, q.get_device(), args)
    return qo, ko


def rotary(q, k, freqs, positions=None, *, cu_seqlens=None, layout="half", amplitude=1.0):
    """Rotary positions on the HIP device, for q (..., H, d) and k (..., Hk, d)
    (or None) of one call: new tensors (q, k), k's None if it is.

    A row's position is positions[t] (int32 or int64, any sign; one a row, flat
    or in the shape of the dimensions before the heads), else, with cu_seqlens
    (B + 1,) of packed rows (T, H, d), its place in its sequence, else its place
    along the dimension before the heads."""
    return _run("rotary", q, k, freqs, positions, cu_seqlens, layout, amplitude, 0)


def rotary_backward(grad_q, grad_k, freqs, positions=None, *, cu_seqlens=None, layout="half", amplitude=1.0):
    """Gradients of q and k: the gradients rotated back."""
    return _run("rotary_backward", grad_q, grad_k, freqs, positions, cu_seqlens, layout, amplitude, 1)


def rotary_ref(x, freqs, positions, layout="half", amplitude=1.0):
    """The same in PyTorch for one tensor (..., H, d) and positions of its
    leading dimensions: angles in 64 bits, products fp32, cast to x's dtype."""
    w = positions.double()[..., None] * freqs.double()
    cos, sin = ((f(w) * amplitude).float()[..., None, :] for f in (torch.cos, torch.sin))
    r = 2 * freqs.numel()
    xf = x.float()
    half = layout == "half"
    a, b = (xf[..., :r // 2], xf[..., r // 2:r]) if half else (xf[..., 0:r:2], xf[..., 1:r:2])
    pair = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(pair, -1) if half else torch.stack(pair, -1).flatten(-2)
    return torch.cat((turned, xf[..., r:]), -1).to(x.dtype)


class RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, freqs, positions, cu_seqlens, layout, amplitude):
        ctx.save_for_backward(freqs, positions, cu_seqlens)
        ctx.args = (layout, amplitude)
        ctx.set_materialize_grads(False)
        qo, ko = rotary(q, k, freqs, positions, cu_seqlens=cu_seqlens, layout=layout, amplitude=amplitude)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, grad_q, grad_k=None):
        freqs, positions, cu = ctx.saved_tensors
        need = ctx.needs_input_grad
        gq, gk = (g if n else None for g, n in zip((grad_q, grad_k), need))
        # (linear: the backward of the backward is the same rotation again, forward)
        out = _back(gq, gk, freqs, positions, cu, *ctx.args)
        return (*out, None, None, None, None, None)


class _RotaryBackFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gq, gk, freqs, positions, cu_seqlens, layout, amplitude):
        ctx.save_for_backward(freqs, positions, cu_seqlens)
        ctx.args = (layout, amplitude)
        q, k = rotary_backward(gq, gk, freqs, positions, cu_seqlens=cu_seqlens, layout=layout, amplitude=amplitude)
        return q if gk is None else (q, k)

    @staticmethod
    def backward(ctx, q, k=None):
        freqs, positions, cu = ctx.saved_tensors
        return (*_pair(RotaryFn.apply, q, k, freqs, positions, cu, *ctx.args), None, None, None, None, None)


def _pair(fn, q, k, *args):
    """fn of either or both of q and k: (q', k'), None for what is None."""
    if q is None and k is None:
        return None, None
    if q is None:
        return None, fn(k, None, *args)
    return (fn(q, None, *args), None) if k is None else fn(q, k, *args)


def _back(gq, gk, *args):
    return _pair(_RotaryBackFn.apply, gq, gk, *args)


def refuse_trained(asked):
    """freqs' own gradient is not computed: asked for, it is an error, not None."""
    if asked:
        raise NotImplementedError("rotary: freqs requires a gradient, which is not computed (freqs.detach() needs none)")


def rotary_fn(q, k, freqs, positions=None, *, cu_seqlens=None, layout="half", amplitude=1.0):
    """Autograd-aware rotary: (q, k).  freqs that require a gradient are refused."""
    refuse_trained(freqs.requires_grad and torch.is_grad_enabled())
    if not _lib.needs_autograd(q, k, freqs):
        return rotary(q, k, freqs, positions, cu_seqlens=cu_seqlens, layout=layout, amplitude=amplitude)
    out = RotaryFn.apply(q, k, freqs, positions, cu_seqlens, layout, amplitude)
    return (out, None) if k is None else out
