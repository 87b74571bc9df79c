"""Frozen weights: their gradients are neither computed nor allocated, through
the functions, the registered ops and the layer made of them, eager and compiled."""

from __future__ import annotations

import sys

import pytest
import torch

from FlagOS_mhc import library as L, sublayer as S
from test_sublayer_library import DEV, _gen, _layer_inputs

OPS = torch.ops.flagos_mhc


def test_meta_shapes_without_the_weights_gradients():
    with torch.device("meta"):
        x, w, r = torch.empty(6, 16, dtype=torch.bfloat16), torch.empty(16), torch.empty(6)
        assert [(tuple(t.shape), t.dtype) for t in OPS.layer_norm_backward(x, x, w, r, r, False)] == [
            ((6, 16), x.dtype), ((0,), torch.float32), ((0,), torch.float32)]
        wg, wd, g = (torch.empty(s, dtype=x.dtype) for s in ((24, 16), (8, 24), (6, 24)))
        got = OPS.gated_ffn_backward(torch.empty(6, 8, dtype=x.dtype), x, wg, wg, wd, g.float(), g.float(), g, "silu", False)
        assert [tuple(t.shape) for t in got] == [(6, 16), (0,), (0,), (0,)]


@pytest.mark.gpu
def test_opcheck_without_the_weights_gradients():
    g = _gen(1)
    r = lambda *s, to=torch.bfloat16: torch.randn(*s, device=DEV, generator=g).to(to)
    x, w = r(9, 40), r(40, to=torch.float32)
    _, mean, rstd = OPS.layer_norm(x, w, None, 1e-5)
    torch.library.opcheck(OPS.layer_norm_backward.default, (r(9, 40), x, w, mean, rstd, False))
    wg, wu, wd = r(56, 40), r(56, 40), r(24, 56)
    f = OPS.gated_ffn(x, wg, wu, wd, "gelu", True)
    torch.library.opcheck(OPS.gated_ffn_backward.default, (r(9, 24), x, wg, wu, wd, *f[1:], "gelu", False))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fn", "op", "compiled"])
@pytest.mark.parametrize("trained", [(), (4,), (5,), (6,), (8,), (4, 7)])
def test_frozen_weights(form, trained, monkeypatch):
    """The gradients that are wanted equal those with everything trained, and the
    kernels are asked for the others only where one of their group is wanted."""
    args = _layer_inputs(40, 4, 128, 200, seed=3)
    gy = torch.randn(40, 4, 128, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    asked = {}
    for name, module in (("layer_norm_backward", "layer_norm"), ("gated_ffn_backward", "gated_ffn")):
        def spy(*a, _run=getattr(S, name), _name=name, **k):
            out = _run(*a, **k)
            asked[_name] = out[1] is not None
            return out
        for m in (module, "library"):
            monkeypatch.setattr(sys.modules[f"FlagOS_mhc.{m}"], name, spy)
    fn = S.mhc_ffn_layer_fn if form == "fn" else L.mhc_ffn_layer_op
    if form == "compiled":
        torch._dynamo.reset()
        fn = torch.compile(fn, backend="aot_eager", fullgraph=True)

    def run(which):
        leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate(args)]
        fn(*leaves).backward(gy)
        return [t.grad for t in leaves]

    want = run(range(9))
    assert asked == {"layer_norm_backward": True, "gated_ffn_backward": True}
    got = run((0, *trained))
    assert asked == {"layer_norm_backward": any(i in (4, 5) for i in trained),
                     "gated_ffn_backward": any(i in (6, 7, 8) for i in trained)}
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b) if i in (0, *trained) else a is None, i


@pytest.mark.gpu
@pytest.mark.parametrize("fn", [S.mhc_ffn_layer_fn, L.mhc_ffn_layer_op])
def test_gradients_with_a_graph_of_the_backward(fn):
    """create_graph=True changes no gradient; the graph's use is refused."""
    args = _layer_inputs(20, 4, 64, 72, seed=5)
    gy = torch.randn(20, 4, 64, device=DEV, generator=_gen(6)).to(torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in args]
    want = torch.autograd.grad(fn(*leaves, dropout_p=0.1, seed=2), leaves, gy)
    got = torch.autograd.grad(fn(*leaves, dropout_p=0.1, seed=2), leaves, gy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for g in got:
        with pytest.raises(RuntimeError, match="second derivatives|autograd formula"):
            g.float().sum().backward(retain_graph=True)
