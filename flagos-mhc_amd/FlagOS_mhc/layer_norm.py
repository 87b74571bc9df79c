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


def _rows(what, x):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x of shape {tuple(x.shape)} has no last dimension to normalise")
    D = x.shape[-1]
    return x.numel() // D, D


def _param(what, name, p, x):
    """weight or bias as the kernel takes it: (D,), x's dtype or fp32."""
    if p is None:
        return None
    if p.numel() != x.shape[-1]:
        raise ValueError(f"{what}: {name} has {p.numel()} elements, x's rows {x.shape[-1]}")
    if p.device != x.device:
        raise ValueError(f"{what}: {name} is on {p.device}, x on {x.device}")
    return _lib.operand(p, (p.numel(),), p.dtype if p.dtype == x.dtype else torch.float32)


def _params(what, x, weight, bias):
    w, b = _param(what, "weight", weight, x), _param(what, "bias", bias, x)
    if w is not None and b is not None and w.dtype != b.dtype:
        w, b = w.float(), b.float()
    dt = w.dtype if w is not None else b.dtype if b is not None else x.dtype
    return w, b, _lib.DTYPE_CODE[dt]


def layer_norm(x, weight=None, bias=None, eps=1e-5, need_backward=False):
    """Layer norm on the HIP device.  Returns a dict with y (x's shape and
    dtype); with ``need_backward`` also mean and rstd (rows,) fp32."""
    what = "layer_norm"
    _lib.require_device(what, x, weight, bias)
    code = _lib.dtype_code(what, x.dtype)
    T, D = _rows(what, x)
    w, b, wcode = _params(what, x, weight, bias)
    xf = x.contiguous()
    y = torch.empty_like(xf, memory_format=torch.contiguous_format)
    out = {"y": y}
    mean = rstd = None
    if need_backward:
        mean, rstd = (torch.empty((T,), dtype=torch.float32, device=x.device) for _ in range(2))
        out.update(mean=mean, rstd=rstd)
    if T > 0:
        lib = _lib.load()
        with _lib.on_device(xf.device):
            rc = lib.mhc_layer_norm_fwd(xf.data_ptr(), code, _lib.ptr(w), _lib.ptr(b), wcode, float(eps),
                                        y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd), T, D, _lib.stream_of(xf))
        _lib.check(rc, what)
    return out


def layer_norm_backward(grad_y, x, weight, mean, rstd, need_params=True):
    """(grad_x, grad_weight, grad_bias): grad_x in x's shape and dtype, the
    other two (D,) fp32 (None with ``need_params=False``).  Deterministic."""
    what = "layer_norm_backward"
    _lib.require_device(what, grad_y, x, weight, mean, rstd)
    code = _lib.dtype_code(what, x.dtype)
    T, D = _rows(what, x)
    if grad_y.shape != x.shape:
        raise ValueError(f"{what}: grad_y of shape {tuple(grad_y.shape)} for x of shape {tuple(x.shape)}")
    if mean.numel() != T or rstd.numel() != T:
        raise ValueError(f"{what}: {mean.numel()} means and {rstd.numel()} rstds for {T} rows")
    w, _, wcode = _params(what, x, weight, None)
    xf = x.contiguous()
    gy = _lib.operand(grad_y, x.shape, xf.dtype)
    mu, rs = _lib.operand(mean, (T,), torch.float32), _lib.operand(rstd, (T,), torch.float32)
    dev = xf.device
    gx = torch.empty_like(xf, memory_format=torch.contiguous_format)
    gw = gb = None
    if T == 0:
        if need_params:
            gw, gb = (torch.zeros((D,), dtype=torch.float32, device=dev) for _ in range(2))
        return gx, gw, gb
    ws, ws_bytes = None, 0
    if need_params:
        gw, gb = (torch.empty((D,), dtype=torch.float32, device=dev) for _ in range(2))
        ws, ws_bytes = _lib.workspace("mhc_layer_norm_bwd_workspace_size", dev, T, D, code)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.mhc_layer_norm_bwd(gy.data_ptr(), xf.data_ptr(), code, _lib.ptr(w), wcode, mu.data_ptr(),
                                    rs.data_ptr(), gx.data_ptr(), _lib.ptr(gw), _lib.ptr(gb), _lib.ptr(ws),
                                    ws_bytes, T, D, _lib.stream_of(xf))
    _lib.check(rc, what)
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
        return gx, gw, gb, None


def layer_norm_fn(x, weight=None, bias=None, eps=1e-5):
    """Autograd-aware layer_norm: y."""
    return LayerNormFn.apply(x, weight, bias, eps)
