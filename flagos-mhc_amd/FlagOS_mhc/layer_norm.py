"""Layer norm of the sublayer's input, forward and backward.

    mean = sum x / D,  rstd = (sum (x - mean)^2 / D + eps)^-1/2
    y = (x - mean) * rstd * weight + bias

x is (..., D); weight and bias are (D,) in x's dtype or fp32 (any other
dtype is converted to fp32), either may be None.  Sums are fp32.  In an mHC
layer x is the y of ``mhc_pre_clamp_sinkhorn`` and the result goes to the
attention or feed-forward block.  The reference has no such operator: its
model code runs PyTorch's.
"""

from __future__ import annotations

import torch

from . import _lib


_F32 = torch.float32


def _rows(what, x):
    """(rows, their length, dtype code) of x."""
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: x of shape {tuple(shape)} has no last dimension to normalise")
    D = shape[-1]
    return x.numel() // D, D, _lib.dtype_code(what, x.dtype)


def _param(what, name, p, x, D):
    """weight or bias as the kernel takes it: (D,), x's dtype or fp32."""
    if p.numel() != D:
        raise ValueError(f"{what}: {name} has {p.numel()} elements, x's rows {D}")
    dt = p.dtype
    if (dt is _F32 or dt is x.dtype) and p.is_contiguous():
        return p
    return _lib.operand(p, (D,), dt if dt is x.dtype else _F32)


def _params(what, x, D, weight, bias):
    w = None if weight is None else _param(what, "weight", weight, x, D)
    b = None if bias is None else _param(what, "bias", bias, x, D)
    if w is None:
        dt = x.dtype if b is None else b.dtype
    else:
        dt = w.dtype
        if b is not None and b.dtype is not dt:
            w, b, dt = w.float(), b.float(), _F32
    return w, b, _lib.DTYPE_CODE[dt]


def layer_norm(x, weight=None, bias=None, eps=1e-5, need_backward=False):
    """Layer norm on the HIP device.  Returns a dict with y (x's shape and
    dtype); with ``need_backward`` also mean and rstd (rows,) fp32."""
    what = "layer_norm"
    _lib.require_device(what, x, weight, bias)
    T, D, code = _rows(what, x)
    w, b, wcode = _params(what, x, D, weight, bias)
    xf = x.contiguous()
    y = torch.empty_like(xf)
    out = {"y": y}
    mean = rstd = None
    if need_backward:
        mean = out["mean"] = torch.empty(T, dtype=_F32, device=x.device)
        rstd = out["rstd"] = torch.empty_like(mean)
    if T > 0:
        _lib.call(what, _lib.load().mhc_layer_norm_fwd, x.get_device(), xf.data_ptr(), code, _lib.ptr(w), _lib.ptr(b),
                  wcode, eps, y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd), T, D)
    return out


def layer_norm_backward(grad_y, x, weight, mean, rstd, need_params=True):
    """(grad_x, grad_weight, grad_bias): grad_x in x's shape and dtype, the
    other two (D,) fp32 (None with ``need_params=False``).  Deterministic."""
    what = "layer_norm_backward"
    _lib.require_device(what, grad_y, x, weight, mean, rstd)
    T, D, code = _rows(what, x)
    if grad_y.shape != x.shape:
        raise ValueError(f"{what}: grad_y of shape {tuple(grad_y.shape)} for x of shape {tuple(x.shape)}")
    if mean.numel() != T or rstd.numel() != T:
        raise ValueError(f"{what}: {mean.numel()} means and {rstd.numel()} rstds for {T} rows")
    w, _, wcode = _params(what, x, D, weight, None)
    xf = x.contiguous()
    gy = grad_y if grad_y.dtype is x.dtype and grad_y.is_contiguous() else _lib.operand(grad_y, x.shape, x.dtype)
    mu = mean if mean.dtype is _F32 and mean.is_contiguous() else _lib.operand(mean, (T,), _F32)
    rs = rstd if rstd.dtype is _F32 and rstd.is_contiguous() else _lib.operand(rstd, (T,), _F32)
    gx = torch.empty_like(xf)
    gw = gb = ws = None
    ws_bytes = 0
    if need_params:
        gw = (torch.empty if T else torch.zeros)(D, dtype=_F32, device=x.device)
        gb = torch.empty_like(gw) if T else torch.zeros_like(gw)
    if T > 0:
        if need_params:
            ws, ws_bytes = _lib.workspace("mhc_layer_norm_bwd_workspace_size", x.device, T, D, code)
        _lib.call(what, _lib.load().mhc_layer_norm_bwd, x.get_device(), gy.data_ptr(), xf.data_ptr(), code, _lib.ptr(w),
                  wcode, mu.data_ptr(), rs.data_ptr(), gx.data_ptr(), _lib.ptr(gw), _lib.ptr(gb), _lib.ptr(ws),
                  ws_bytes, T, D)
    return gx, gw, gb


def layer_norm_ref(x, weight=None, bias=None, eps=1e-5):
    """The same in PyTorch, fp32 math, cast to x's dtype."""
    xf = x.float()
    xc = xf - xf.mean(-1, keepdim=True)
    y = xc * torch.rsqrt(xc.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps=1e-5):
        out = layer_norm(x, weight, bias, eps, need_backward=True)
        ctx.save_for_backward(x, weight, out["mean"], out["rstd"])
        ctx.dtypes = tuple(None if p is None else (p.shape, p.dtype) for p in (weight, bias))
        return out["y"]

    @staticmethod
    def backward(ctx, grad_y):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gx, gw, gb = layer_norm_backward(grad_y, x, weight, mean, rstd, need_params=need)
        gw, gb = (g.reshape(d[0]).to(d[1]) if d is not None and need else None for g, d in zip((gw, gb), ctx.dtypes))
        return (*_lib.first_order("layer_norm", (gx, gw, gb), grad_y, x, weight), None)


def layer_norm_fn(x, weight=None, bias=None, eps=1e-5):
    """Autograd-aware layer_norm: y.  Without gradients to take, nothing is
    saved."""
    if not _lib.needs_autograd(x, weight, bias):
        return layer_norm(x, weight, bias, eps)["y"]
    return LayerNormFn.apply(x, weight, bias, eps)
