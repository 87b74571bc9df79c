"""Gated feed-forward block, forward and backward.

    gate = x w_gate^T,  up = x w_up^T,  hidden = act(gate) * up,  out = hidden w_down^T

x is (..., D), w_gate and w_up (F, D), w_down (O, F) as torch.nn.Linear keeps
its weights; out is (..., O).  All have one dtype (fp32, bf16 or fp16);
products accumulate in fp32 and hidden is rounded to that dtype between
them, as the gradients of gate and up are in the backward: results carry one
rounding more than with fp32 between the products, and in fp16 a hidden above
65504 is infinite.  Operands that are not contiguous, or whose address is no
multiple of 16 bytes, are copied in every call.  In an mHC layer x is the norm of ``mhc_pre_clamp_sinkhorn``'s y and
out the h_out of ``mhc_post``.  The reference has no such operator: its
model code runs PyTorch's.
"""

from __future__ import annotations

import math

import torch

from . import _lib

#: activation names and their codes (include/mhc_amd.h)
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def hidden_width(F: int) -> int:
    """Columns of the saved hidden: F rounded up to 8, those past F zero."""
    return (F + 7) // 8 * 8


def _aligned(t, shape, dtype):
    """t as _lib.operand gives it, at a 16-byte aligned address."""
    t = _lib.operand(t, shape, dtype)
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() & 15 else t


def _check(what, x, w_gate, w_up, w_down, activation):
    """(T, D, F, O, dtype code, activation code) of a call."""
    code = _lib.dtype_code(what, x.dtype)
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation {activation!r}, expected one of {tuple(ACTIVATIONS)}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError(f"{what}: x of {x.dim()}, w_gate of {w_gate.dim()} and w_down of {w_down.dim()} dimensions")
    F, D = w_gate.shape
    O = w_down.shape[0]
    if x.shape[-1] != D or tuple(w_up.shape) != (F, D) or w_down.shape[1] != F:
        raise ValueError(f"{what}: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and "
                         f"w_down {tuple(w_down.shape)} do not fit (..., D), (F, D), (F, D), (O, F)")
    if min(D, F, O) < 1:
        raise ValueError(f"{what}: empty weights (D={D}, F={F}, O={O})")
    for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if w.dtype != x.dtype:
            raise ValueError(f"{what}: {name} is {w.dtype}, x {x.dtype}")
    return math.prod(x.shape[:-1]), D, F, O, code, ACTIVATIONS[activation]


def gated_ffn(x, w_gate, w_up, w_down, activation="silu", need_backward=False):
    """The block on the HIP device.  Returns a dict with out (..., O) in x's
    dtype; with ``need_backward`` also gate and up (T, F) fp32 and hidden
    (T, F rounded up to 8) in x's dtype."""
    what = "gated_ffn"
    _lib.require_device(what, x, w_gate, w_up, w_down)
    T, D, F, O, code, act = _check(what, x, w_gate, w_up, w_down, activation)
    dev = x.device
    out = torch.empty(tuple(x.shape[:-1]) + (O,), dtype=x.dtype, device=dev)
    gate = up = hidden = None
    if need_backward:
        gate = torch.empty((T, F), dtype=torch.float32, device=dev)
        up = torch.empty((T, F), dtype=torch.float32, device=dev)
        hidden = torch.empty((T, hidden_width(F)), dtype=x.dtype, device=dev)
    if T > 0:
        xf = _aligned(x, (T, D), x.dtype)
        wg, wu = _aligned(w_gate, (F, D), x.dtype), _aligned(w_up, (F, D), x.dtype)
        wd = _aligned(w_down, (O, F), x.dtype)
        query = "mhc_gated_ffn_fwd_save_workspace_size" if need_backward else "mhc_gated_ffn_fwd_workspace_size"
        ws, ws_bytes = _lib.workspace(query, dev, T, D, F, O, code)
        _lib.call(what, _lib.load().mhc_gated_ffn_fwd, x.get_device(), xf.data_ptr(), wg.data_ptr(), wu.data_ptr(),
                  wd.data_ptr(), code, act, out.data_ptr(), _lib.ptr(gate), _lib.ptr(up), _lib.ptr(hidden),
                  ws.data_ptr(), ws_bytes, T, D, F, O)
    result = {"out": out}
    if need_backward:
        result.update(gate=gate, up=up, hidden=hidden)
    return result


def gated_ffn_backward(grad_out, x, w_gate, w_up, w_down, gate, up, hidden, activation="silu",
                       need_weights=True):
    """(grad_x, grad_w_gate, grad_w_up, grad_w_down) in the dtype of x, from the
    forward's gate, up and hidden; the last three are None with
    ``need_weights=False``.  Deterministic."""
    what = "gated_ffn_backward"
    _lib.require_device(what, grad_out, x, w_gate, w_up, w_down, gate, up, hidden)
    T, D, F, O, code, act = _check(what, x, w_gate, w_up, w_down, activation)
    if tuple(grad_out.shape) != tuple(x.shape[:-1]) + (O,):
        raise ValueError(f"{what}: grad_out of shape {tuple(grad_out.shape)}, expected {tuple(x.shape[:-1]) + (O,)}")
    for name, t in (("gate", gate), ("up", up)):
        if tuple(t.shape) != (T, F):
            raise ValueError(f"{what}: {name} of shape {tuple(t.shape)}, expected {(T, F)}")
    if tuple(hidden.shape) != (T, hidden_width(F)) or hidden.dtype != x.dtype:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} {hidden.dtype}, expected {(T, hidden_width(F))} {x.dtype}")
    dev = x.device
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    alloc = torch.empty if T > 0 else torch.zeros
    gwg = gwu = gwd = None
    if need_weights:
        gwg, gwu = (alloc((F, D), dtype=x.dtype, device=dev) for _ in range(2))
        gwd = alloc((O, F), dtype=x.dtype, device=dev)
    if T > 0:
        xf, go = _aligned(x, (T, D), x.dtype), _aligned(grad_out, (T, O), x.dtype)
        wg, wu = _aligned(w_gate, (F, D), x.dtype), _aligned(w_up, (F, D), x.dtype)
        wd = _aligned(w_down, (O, F), x.dtype)
        g, u = _aligned(gate, (T, F), torch.float32), _aligned(up, (T, F), torch.float32)
        h = _aligned(hidden, hidden.shape, x.dtype)
        ws, ws_bytes = _lib.workspace("mhc_gated_ffn_bwd_workspace_size", dev, T, D, F, O, code)
        _lib.call(what, _lib.load().mhc_gated_ffn_bwd, x.get_device(), go.data_ptr(), xf.data_ptr(), wg.data_ptr(),
                  wu.data_ptr(), wd.data_ptr(), g.data_ptr(), u.data_ptr(), h.data_ptr(), code, act, gx.data_ptr(),
                  _lib.ptr(gwg), _lib.ptr(gwu), _lib.ptr(gwd), ws.data_ptr(), ws_bytes, T, D, F, O)
    return gx, gwg, gwu, gwd


def activation_ref(name, g):
    """act(g) in PyTorch."""
    if name == "silu":
        return torch.nn.functional.silu(g)
    if name == "relu":
        return torch.relu(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if name == "gelu_tanh" else "none")


def gated_ffn_ref(x, w_gate, w_up, w_down, activation="silu"):
    """The same in PyTorch, fp32 math, cast to x's dtype (autograd-aware)."""
    xf = x.float()
    h = activation_ref(activation, xf @ w_gate.float().t()) * (xf @ w_up.float().t())
    return (h @ w_down.float().t()).to(x.dtype)


class GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation="silu"):
        f = gated_ffn(x, w_gate, w_up, w_down, activation, need_backward=True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, f["gate"], f["up"], f["hidden"])
        ctx.activation = activation
        return f["out"]

    @staticmethod
    def backward(ctx, grad_out):
        grads = gated_ffn_backward(grad_out, *ctx.saved_tensors, activation=ctx.activation,
                                   need_weights=any(ctx.needs_input_grad[1:4]))
        return (*_lib.first_order("gated_ffn", grads, grad_out, *ctx.saved_tensors[:4]), None)


def gated_ffn_fn(x, w_gate, w_up, w_down, activation="silu"):
    """Autograd-aware gated_ffn: out.  Without gradients to take, nothing is
    saved."""
    if not _lib.needs_autograd(x, w_gate, w_up, w_down):
        return gated_ffn(x, w_gate, w_up, w_down, activation)["out"]
    return GatedFfnFn.apply(x, w_gate, w_up, w_down, activation)
