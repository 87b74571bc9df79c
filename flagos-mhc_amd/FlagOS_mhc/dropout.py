"""Dropout whose mask is computed from the element's index and never stored.

Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
easy as 1, 2, 3", SC 2011) with key = seed and counter = (index of the
element's group of 8, offset) gives each element 16 bits; it is kept where
they are at least t = round(p * 65536) and then multiplied by
65536 / (65536 - t), so p acts in steps of 2^-16.  The index runs over the
tensor's elements in row-major order, whatever its strides.  The backward is
the same call on the gradient.  A program gives every call of a step its own
offset (or seed); with ``state``, an int64 tensor (seed, offset) on the
device, a captured graph reads them when it is replayed; seed and offset are
then not looked at, so calls that share a state share their mask: give each
layer a state of its own.
"""

from __future__ import annotations

import math

import torch

from . import _lib

_M64 = (1 << 64) - 1


def _apply(what, x, p, seed, offset, state):
    _lib.require_device(what, x, state)
    code = _lib.dtype_code(what, x.dtype)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p={p} is no probability")
    if state is not None and (state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous()):
        raise ValueError(f"{what}: state must be a contiguous int64 tensor (seed, offset) on {x.device}")
    xf = x.contiguous()
    y = torch.empty_like(xf)
    n = xf.numel()
    if n:
        _lib.call(what, _lib.load().mhc_dropout, x.get_device(), xf.data_ptr(), y.data_ptr(), n, code, p,
                  int(seed) & _M64, int(offset) & _M64, _lib.ptr(state))
    return y


def dropout(x, p, seed=0, offset=0, state=None):
    """Dropout on the HIP device, in x's shape and dtype."""
    return _apply("dropout", x, p, seed, offset, state)


def dropout_backward(grad_y, p, seed=0, offset=0, state=None):
    """x's gradient: grad_y under the forward's mask and factor."""
    return _apply("dropout_backward", grad_y, p, seed, offset, state)


def philox_ref(groups, seed, offset):
    """(groups, 4) int64: the Philox4x32-10 words of the first `groups` groups."""
    m32 = 0xFFFFFFFF
    i = torch.arange(groups, dtype=torch.int64)
    c = [i & m32, i >> 32, torch.full_like(i, offset & m32), torch.full_like(i, (offset >> 32) & m32)]
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # wrap modulo 2^64: every bit stays
        c = [((p1 >> 32) & m32) ^ c[1] ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c[3] ^ k1, p0 & m32]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return torch.stack(c, -1)


def dropout_ref(x, p, seed=0, offset=0):
    """The same in PyTorch."""
    n, t = x.numel(), int(math.floor(float(p) * 65536.0 + 0.5))
    words = philox_ref((n + 7) // 8, int(seed) & _M64, int(offset) & _M64)
    keep = (torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:n] >= t).to(x.device).reshape(x.shape)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype)


class DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed=0, offset=0, state=None):
        # the state the mask came from: a program moves its own on before the backward
        ctx.state = None if state is None else state.clone()
        ctx.args = (p, seed, offset)
        return dropout(x, p, seed, offset, ctx.state)

    @staticmethod
    def backward(ctx, grad_y):
        # linear: where a graph of the backward is asked for, the gradient is dropout_fn of grad_y
        fn = dropout_fn if torch.is_grad_enabled() else dropout_backward
        return fn(grad_y, *ctx.args, ctx.state), None, None, None, None


def dropout_fn(x, p, seed=0, offset=0, state=None):
    """Autograd-aware dropout: y."""
    return DropoutFn.apply(x, p, seed, offset, state)
