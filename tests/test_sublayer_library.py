"""The sublayer's operators as torch.ops.flagos_mhc.*, and the mHC feed-forward
layer they make: shapes on meta tensors (CPU); registration checks, the layer
through autograd, compiled, in captured graphs and against PyTorch (GPU)."""

from __future__ import annotations

import pytest
import torch

import FlagOS_mhc as m
import sublayer_ref as R
from FlagOS_mhc import library as L, sublayer as S

OPS = ("layer_norm", "layer_norm_backward", "gated_ffn", "gated_ffn_backward", "dropout")
DEV = "cuda"


def test_ops_registered():
    for name in OPS:
        assert hasattr(torch.ops.flagos_mhc, name), name


@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_meta_shapes(lead):
    T, D, F, O, bf = 6, 16, 21, 24, torch.bfloat16
    ops = torch.ops.flagos_mhc
    with torch.device("meta"):
        x, w = torch.empty(lead + (D,), dtype=bf), torch.empty(D)
        assert [(t.shape, t.dtype) for t in ops.layer_norm(x, w, None, 1e-5)] == [
            (x.shape, bf), ((T,), torch.float32), ((T,), torch.float32)]
        assert [(t.shape, t.dtype) for t in ops.layer_norm_backward(x, x, w, w, w)] == [
            (x.shape, bf), ((D,), torch.float32), ((D,), torch.float32)]
        wg, wd = torch.empty(F, D, dtype=bf), torch.empty(O, F, dtype=bf)
        got = ops.gated_ffn(x, wg, wg, wd, "silu", True)
        assert [(t.shape, t.dtype) for t in got] == [
            (lead + (O,), bf), ((T, F), torch.float32), ((T, F), torch.float32), ((T, 24), bf)]
        assert [tuple(t.shape) for t in ops.gated_ffn(x, wg, wg, wd, "silu", False)] == [lead + (O,), (0,), (0,), (0,)]
        grads = ops.gated_ffn_backward(got[0], x, wg, wg, wd, *got[1:], "silu")
        assert [t.shape for t in grads] == [x.shape, wg.shape, wg.shape, wd.shape]
        assert ops.dropout(x, 0.5, 1, 2).shape == x.shape


def test_cpu_tensors_refused():
    x = torch.randn(4, 8)
    for call in (lambda: L.layer_norm_op(x), lambda: L.gated_ffn_op(x, x, x, x.t()), lambda: L.dropout_op(x, 0.5)):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


# ---- GPU ---------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _layer_inputs(T, N, D, F, dtype=torch.bfloat16, seed=0):
    """x, phi, alpha, base, norm weight and bias, the block's weights."""
    g = _gen(seed)
    r = lambda *s, scale=1.0, to=dtype: (torch.randn(*s, device=DEV, generator=g) * scale).to(to)
    M, f32 = N * (N + 2), torch.float32
    return [r(T, N, D), r(M, N * D, scale=(N * D) ** -0.5), torch.tensor([0.5, 0.5, 1.0], device=DEV),
            r(M, scale=0.1, to=f32), 1 + r(D, scale=0.1, to=f32), r(D, scale=0.1, to=f32),
            r(F, D, scale=D ** -0.5), r(F, D, scale=D ** -0.5), r(D, F, scale=F ** -0.5)]


@pytest.mark.gpu
def test_opcheck():
    g = _gen(1)
    r = lambda *s, to=torch.bfloat16: torch.randn(*s, device=DEV, generator=g).to(to)
    x, w, b = r(9, 40).requires_grad_(True), r(40, to=torch.float32).requires_grad_(True), r(40)
    ops = torch.ops.flagos_mhc
    torch.library.opcheck(ops.layer_norm.default, (x, w, b.float(), 1e-5))
    y, mean, rstd = ops.layer_norm(x.detach(), w.detach(), None, 1e-5)
    torch.library.opcheck(ops.layer_norm_backward.default, (r(9, 40), x.detach(), w.detach(), mean, rstd))
    wg, wu, wd = r(56, 40), r(56, 40), r(24, 56)
    torch.library.opcheck(ops.gated_ffn.default, (x, wg.requires_grad_(True), wu, wd, "gelu", True))
    f = ops.gated_ffn(x.detach(), wg.detach(), wu, wd, "gelu", True)
    torch.library.opcheck(ops.gated_ffn_backward.default, (r(9, 24), x.detach(), wg.detach(), wu, wd, *f[1:], "gelu"))
    torch.library.opcheck(ops.dropout.default, (x, 0.25, -5, 7))
    torch.library.opcheck(ops.dropout.default, (x, 0.25, 0, 0, torch.tensor([3, 4], device=DEV)))


@pytest.mark.gpu
def test_layer_matches_its_parts_and_pytorch():
    """The layer's output and gradients equal those of the operators called one by
    one, and PyTorch's references in fp32 within the roundings between them."""
    T, N, D, F = 130, 4, 256, 704
    args = _layer_inputs(T, N, D, F)
    g = _gen(2)
    gy = torch.randn(T, N, D, device=DEV, generator=g).to(torch.bfloat16)
    kw = dict(activation="gelu_tanh", dropout_p=0.2, seed=5, offset=9, clamp_min=-10.0, clamp_max=10.0)

    leaves = [t.clone().requires_grad_(True) for t in args]
    out = S.mhc_ffn_layer_fn(*leaves, **kw)
    out.backward(gy)

    x, phi, alpha, base, nw, nb, wg, wu, wd = args
    pre = m.mhc_pre_clamp_sinkhorn(x, phi, alpha, base, need_backward=True, clamp_min=-10.0, clamp_max=10.0)
    n = S.layer_norm(pre["y"], nw, nb, need_backward=True)
    f = S.gated_ffn(n["y"], wg, wu, wd, "gelu_tanh", need_backward=True)
    h = S.dropout(f["out"], 0.2, 5, 9)
    assert torch.equal(out, m.mhc_post(x, pre["comb_frag"], h, pre["post_out"]))
    _, _, gh, _ = m.mhc_post_backward(gy, x, pre["comb_frag"], h, pre["post_out"])
    gn, *gw = S.gated_ffn_backward(S.dropout_backward(gh, 0.2, 5, 9), n["y"], wg, wu, wd, f["gate"], f["up"],
                                   f["hidden"], "gelu_tanh")
    _, gnw, gnb = S.layer_norm_backward(gn, pre["y"], nw, n["mean"], n["rstd"])
    for leaf, want in zip(leaves[4:], (gnw, gnb, *gw)):
        assert torch.equal(leaf.grad, want)

    # the sublayer in PyTorch, in fp32, from the same y
    y = pre["y"].float().requires_grad_(True)
    ref = S.dropout_ref(S.gated_ffn_ref(S.layer_norm_ref(y, nw, nb), wg.float(), wu.float(), wd.float(), "gelu_tanh"),
                        0.2, 5, 9)
    ref.backward(gh.float())
    # roundings to bf16 on the way: norm, hidden, out, dropped; the gradients of out, gate and up, norm, y
    eps = R.half_step(torch.bfloat16)
    assert float((h.float() - ref.detach()).norm() / ref.detach().norm()) <= 4 * eps
    gx_y, _, _ = S.layer_norm_backward(gn, pre["y"], nw, n["mean"], n["rstd"])
    assert float((gx_y.float() - y.grad).norm() / y.grad.norm()) <= 8 * eps


@pytest.mark.gpu
def test_registered_layer_compiles_and_matches():
    T, N, D, F = 70, 4, 128, 200
    args = _layer_inputs(T, N, D, F, seed=3)
    gy = torch.randn(T, N, D, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    kw = dict(dropout_p=0.3, seed=1 << 63, offset=3)

    def run(fn):
        leaves = [t.clone().requires_grad_(True) for t in args]
        out = fn(*leaves)
        out.backward(gy)
        return [out.detach()] + [t.grad for t in leaves]

    want = run(lambda *a: S.mhc_ffn_layer_fn(*a, **kw))
    torch._dynamo.reset()
    for fn in (lambda *a: L.mhc_ffn_layer_op(*a, **kw),
               torch.compile(lambda *a: L.mhc_ffn_layer_op(*a, **kw), backend="aot_eager", fullgraph=True)):
        got = run(fn)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            torch.testing.assert_close(a.float(), b.float(), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,F", [(1, 512, 1024), (40, 264, 520), (300, 255, 513)])
def test_graph_replay(T, D, F):
    """Forward and backward of the three operators in a captured graph, replayed
    with eager work in between, new inputs and a moving dropout state."""
    g = _gen(T)
    r = lambda *s, scale=1.0: (torch.randn(*s, device=DEV, generator=g) * scale).to(torch.bfloat16)
    x, gy, nw = r(T, D), r(T, D), r(D)
    wg, wu, wd = r(F, D, scale=D ** -0.5), r(F, D, scale=D ** -0.5), r(D, F, scale=F ** -0.5)
    state = torch.tensor([7, 0], device=DEV)

    def step():
        n = S.layer_norm(x, nw, None, need_backward=True)
        f = S.gated_ffn(n["y"], wg, wu, wd, need_backward=True)
        y = S.dropout(f["out"], 0.2, state=state)
        gn, *gw = S.gated_ffn_backward(S.dropout_backward(gy, 0.2, state=state), n["y"], wg, wu, wd, f["gate"],
                                       f["up"], f["hidden"])
        return [y, *S.layer_norm_backward(gn, x, nw, n["mean"], n["rstd"]), *gw]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    torch.cuda.synchronize()
    seen = []
    for rnd in range(4):
        state[1] = rnd
        if rnd == 2:
            x.copy_(r(T, D))
            gy.copy_(r(T, D))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, eager)):
            assert torch.equal(a, b), f"replay {rnd}: output {i} differs from eager"
        seen.append(captured[0].clone())
    assert not torch.equal(seen[0], seen[1])  # the mask moved with the state
