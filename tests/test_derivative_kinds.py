"""What the autograd-aware functions do with derivatives that they do not
have: forward-mode ones and second ones are refused, never dropped.  No GPU:
the kernel calls are replaced by ones that compute nothing."""

from __future__ import annotations

import sys

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from FlagOS_mhc import _lib, library as L, sublayer as S


class _NoKernels:
    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture(autouse=True)
def no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: _NoKernels())
    monkeypatch.setattr(_lib, "workspace", lambda *a: (torch.zeros(1, dtype=torch.uint8), 1))


X, W, V = torch.ones(4, 8), torch.ones(6, 8), torch.ones(8, 6)
VECTOR = torch.ones(8)

# the operator as a function of one input, and that input
INPUTS = {
    "layer_norm_fn x": (lambda t: S.layer_norm_fn(t), X),
    "layer_norm_fn weight": (lambda t: S.layer_norm_fn(X, t), VECTOR),
    "layer_norm_fn bias": (lambda t: S.layer_norm_fn(X, None, t), VECTOR),
    "gated_ffn_fn x": (lambda t: S.gated_ffn_fn(t, W, W, V), X),
    "gated_ffn_fn w_gate": (lambda t: S.gated_ffn_fn(X, t, W, V), W),
    "gated_ffn_fn w_up": (lambda t: S.gated_ffn_fn(X, W, t, V), W),
    "gated_ffn_fn w_down": (lambda t: S.gated_ffn_fn(X, W, W, t), V),
    "dropout_fn": (lambda t: S.dropout_fn(t, 0.5), X),
    "layer_norm_op x": (lambda t: L.layer_norm_op(t), X),
    "layer_norm_op bias": (lambda t: L.layer_norm_op(X, None, t), VECTOR),
    "gated_ffn_op x": (lambda t: L.gated_ffn_op(t, W, W, V), X),
    "gated_ffn_op w_down": (lambda t: L.gated_ffn_op(X, W, W, t), V),
    "dropout_op": (lambda t: L.dropout_op(t, 0.5), X),
    "mhc_post_op": (lambda t: L.mhc_post_op(t, X, X, X), X),
    "mhc_pre_clamp_sinkhorn_op": (lambda t: L.mhc_pre_clamp_sinkhorn_op(X, t, X, X), X),
    "mhc_post_pre_clamp_sinkhorn_op": (lambda t: L.mhc_post_pre_clamp_sinkhorn_op(X, X, X, t, X, X, X), X),
}


@pytest.mark.parametrize("name", INPUTS)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(name, grad_mode):
    fn, t = INPUTS[name]
    with torch.set_grad_enabled(grad_mode), fwAD.dual_level():
        dual = fwAD.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward"):
            fn(dual)


@pytest.mark.parametrize("name", INPUTS)
def test_jvp_transform_is_refused(name):
    fn, t = INPUTS[name]
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(fn, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("fn", [lambda t: S.layer_norm_fn(t), lambda t: S.gated_ffn_fn(t, W, W, V),
                                lambda t: L.layer_norm_op(t), lambda t: L.gated_ffn_op(t, W, W, V),
                                lambda t: L.dropout_op(t, 0.5)])
def test_tensors_without_a_tangent_pass(fn):
    """.. at a level where others have one."""
    with fwAD.dual_level():
        fwAD.make_dual(X, X)
        assert fn(X).shape == X.shape and not fn(X).requires_grad


# each differentiable input of the operators whose second derivative depends on it
SECOND = [n for n in INPUTS if n.startswith(("layer_norm", "gated_ffn")) and "bias" not in n]


@pytest.mark.parametrize("name", SECOND)
def test_second_derivatives_are_refused(name):
    """.. also where the output's gradient is a constant, as after sum(), and
    beside another term of the loss."""
    fn, t = INPUTS[name]
    t = t.clone().requires_grad_(True)
    for grad_out in (None, torch.ones_like(fn(t)).requires_grad_(True)):
        y = fn(t)
        g, = torch.autograd.grad(y.sum() if grad_out is None else y, t, grad_out, create_graph=True)
        assert g.shape == t.shape and g.requires_grad
        with pytest.raises(RuntimeError, match="second derivatives|no autograd formula|autograd formula"):
            (g.sum() + t.sum()).backward()
    # first derivatives, with a graph of the backward or without
    for create in (True, False):
        assert torch.autograd.grad(fn(t).sum(), t, create_graph=create)[0].requires_grad == create


@pytest.mark.parametrize("fn", [S.dropout_fn, L.dropout_op])
def test_dropout_is_differentiable_twice(fn, monkeypatch):
    """Linear in x: the gradient of its gradient with respect to grad_y is the mask and factor again."""
    # (as the kernel: no graph of its own)
    apply = torch.no_grad()(lambda x, p, seed=0, offset=0, state=None: S.dropout_ref(x, p, seed, offset))
    for module in ("dropout", "library"):
        monkeypatch.setattr(sys.modules[f"FlagOS_mhc.{module}"], "dropout", apply)
    monkeypatch.setattr(sys.modules["FlagOS_mhc.dropout"], "dropout_backward", apply)
    x, c = torch.ones(5, 9, requires_grad=True), torch.full((5, 9), 2.0, requires_grad=True)
    g, = torch.autograd.grad((fn(x, 0.5, 3, 4) * c).sum(), x, create_graph=True)
    mask = S.dropout_ref(torch.ones(5, 9), 0.5, 3, 4)
    assert torch.equal(g.detach(), 2 * mask)
    gc, = torch.autograd.grad(g.sum(), c)
    assert torch.equal(gc, mask) and 0 < int((mask == 0).sum()) < mask.numel()


# ---- the mHC functions: N = 2 streams of width 4 ---------------------------------

T, N, D = 3, 2, 4
M = N * (N + 2)
STREAMS, H_RES, H_OUT, H_POST = torch.ones(T, N, D), torch.ones(T, N, N), torch.ones(T, D), torch.ones(T, N)
PHI, ALPHA, BASE = torch.ones(M, N * D), torch.ones(3), torch.ones(M)
PRE = {"y": H_OUT, "post_out": H_POST, "comb_frag": H_RES, "inv_rms": torch.ones(T), "mixes": torch.ones(T, M),
       "pre": torch.ones(T, N)}


@pytest.mark.parametrize("fn,inputs", [
    ("mhc_post_fn", (STREAMS, H_RES, H_OUT, H_POST)),
    ("mhc_pre_clamp_sinkhorn_fn", (STREAMS, PHI, ALPHA, BASE)),
    ("mhc_post_pre_clamp_sinkhorn_fn", (STREAMS, H_RES, H_OUT, H_POST, PHI, ALPHA, BASE))])
@pytest.mark.parametrize("summed", [True, False])
def test_mhc_second_derivatives_are_refused(fn, inputs, summed, monkeypatch):
    """.. with respect to every input; the operators are replaced by ones that
    return tensors of their results' shapes."""
    a = sys.modules["FlagOS_mhc.autograd"]
    like = lambda *ts: tuple(torch.zeros_like(t) for t in ts)
    out = lambda: {k: v.clone() for k, v in PRE.items()}
    monkeypatch.setattr(a, "mhc_post", lambda x, *r: torch.zeros_like(x))
    monkeypatch.setattr(a, "mhc_post_backward", lambda g, x, *r: like(x, *r))
    monkeypatch.setattr(a, "mhc_post_backward_sum", lambda g, g2, x, *r: like(x, *r))
    monkeypatch.setattr(a, "post_backward_sum_fused", lambda *s: summed)
    monkeypatch.setattr(a, "_pre_forward", lambda *r, **k: out())
    monkeypatch.setattr(a, "_pre_backward", lambda x, phi, alpha, base, *r, **k: like(x, phi, alpha, base))
    monkeypatch.setattr(a, "mhc_pre_clamp_sinkhorn_backward", lambda x, phi, alpha, base, *r, **k: like(x, phi, alpha, base))
    monkeypatch.setattr(a, "mhc_post_pre_clamp_sinkhorn", lambda x, *r, **k: (torch.zeros_like(x), out()))
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    run = lambda: (lambda y: y if isinstance(y, torch.Tensor) else sum(t.sum() for t in y))(getattr(a, fn)(*leaves))
    for i, t in enumerate(leaves):
        g, = torch.autograd.grad(run().sum(), t, create_graph=True)
        assert g.shape == t.shape and g.requires_grad
        with pytest.raises(RuntimeError, match="second derivatives"):
            (g.sum() + t.sum()).backward()
        assert not torch.autograd.grad(run().sum(), t)[0].requires_grad
