"""Rotary positions and attention as torch.ops.flagos_mhc.*, and the mHC
attention layer they make: shapes on meta tensors and derivatives that are not
there (CPU); registration checks, the layer through autograd, compiled, in
captured graphs and against PyTorch (GPU)."""

from __future__ import annotations

import sys
import types

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import FlagOS_mhc as m
import attention_ref as R
from FlagOS_mhc import _lib, library as L, sublayer as S

DEV = "cuda"


def test_meta_shapes():
    ops, bf = torch.ops.flagos_mhc, torch.bfloat16
    for lead in ((6,), (2, 3)):
        with torch.device("meta"):
            q, k, f = torch.empty(lead + (4, 64), dtype=bf), torch.empty(lead + (2, 64), dtype=bf), torch.empty(16)
            assert [(t.shape, t.dtype) for t in ops.rotary(q, k, f)] == [(q.shape, bf), (k.shape, bf)]
            assert [tuple(t.shape) for t in ops.rotary(q, None, f)] == [tuple(q.shape), (0,)]
            out, lse = ops.attention(q, k, k)
            assert (out.shape, out.dtype, tuple(lse.shape), lse.dtype) == (q.shape, bf, (4, 6), torch.float32)
            assert tuple(ops.attention(q, k, k, save=False)[1].shape) == (0,)
            assert [t.shape for t in ops.attention_backward(q, q, k, k, out, lse)] == [q.shape, k.shape, k.shape]


def test_cpu_tensors_refused():
    q = torch.randn(4, 2, 64)
    for call in (lambda: L.attention_op(q, q, q), lambda: L.rotary_op(q, q, torch.ones(4, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


def _on(index):
    return types.SimpleNamespace(is_cuda=True, device=torch.device("cuda", index), get_device=lambda: index)


CALLS = {
    "rotary": (lambda q, k, f, p: S.rotary(q, k, f, p), 4),
    "rotary cu_seqlens": (lambda q, k, f, c: S.rotary(q, k, f, cu_seqlens=c), 4),
    "attention": (lambda q, k, v, c, ck, n: S.attention(q, k, v, c, cu_seqlens_k=ck, lengths_k=n), 6),
    "attention_backward": (lambda g, q, k, v, o, l, c: S.attention_backward(g, q, k, v, o, l, c), 7),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, count) in CALLS.items() for i in range(count)])
def test_another_device_is_refused(name, at):
    fn, count = CALLS[name]
    with pytest.raises(ValueError, match="expected one device"):
        fn(*[_on(1 if i == at else 0) for i in range(count)])


@pytest.fixture
def no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(sys.modules["FlagOS_mhc.attention"], "_workspace_size", lambda *a: 0)


Q, K = torch.ones(4, 2, 8), torch.ones(4, 1, 8)
F = torch.ones(4, dtype=torch.float64)
INPUTS = {
    "rotary_fn q": (lambda t: S.rotary_fn(t, K, F)[0], Q),
    "rotary_fn k": (lambda t: S.rotary_fn(Q, t, F)[1], K),
    "rotary_op q": (lambda t: L.rotary_op(t, K, F)[0], Q),
    "attention_fn q": (lambda t: S.attention_fn(t, K, K), Q),
    "attention_fn k": (lambda t: S.attention_fn(Q, t, K), K),
    "attention_fn v": (lambda t: S.attention_fn(Q, K, t), K),
    "attention_op q": (lambda t: L.attention_op(t, K, K), Q),
    "attention_op v": (lambda t: L.attention_op(Q, K, t), K),
}


@pytest.mark.parametrize("name", INPUTS)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(no_kernels, name, grad_mode):
    fn, t = INPUTS[name]
    with torch.set_grad_enabled(grad_mode), fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            fn(fwAD.make_dual(t, torch.ones_like(t)))
        assert fn(t).shape == fn(t).shape


@pytest.mark.parametrize("name", [n for n in INPUTS if n.startswith("attention")])
def test_second_derivatives_are_refused(no_kernels, name):
    fn, t = INPUTS[name]
    t = t.clone().requires_grad_(True)
    for grad_out in (None, torch.ones(4, 2, 8).requires_grad_(True)):
        y = fn(t)
        g, = torch.autograd.grad(y.sum() if grad_out is None else y, t, grad_out, create_graph=True)
        assert g.shape == t.shape and g.requires_grad
        with pytest.raises(RuntimeError, match="second derivatives|no autograd formula|autograd formula"):
            (g.sum() + t.sum()).backward()


@pytest.mark.parametrize("fn", [S.rotary_fn, L.rotary_op])
def test_rotary_is_differentiable_twice(fn, monkeypatch):
    """Linear in q and k: the gradient of its gradient is the rotation again."""
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    pos = torch.arange(4)

    def run(sign):
        def apply(q, k, freqs, positions=None, *, cu_seqlens=None, layout="half", amplitude=1.0):
            with torch.no_grad():
                return tuple(None if t is None else S.rotary_ref(t, sign * freqs, pos, layout, amplitude) for t in (q, k))
        return apply

    for module in ("rotary", "library"):
        monkeypatch.setattr(sys.modules[f"FlagOS_mhc.{module}"], "rotary", run(1))
        monkeypatch.setattr(sys.modules[f"FlagOS_mhc.{module}"], "rotary_backward", run(-1))
    g = torch.Generator().manual_seed(1)
    r = lambda t: torch.randn(t.shape, generator=g)
    q, k = r(Q).requires_grad_(True), r(K).requires_grad_(True)
    c, d = r(Q).requires_grad_(True), r(K)
    a, b = fn(q, k, F)
    gq, gk = torch.autograd.grad((a * c).sum() + (b * d).sum(), (q, k), create_graph=True)
    torch.testing.assert_close(gq.detach(), S.rotary_ref(c.detach(), -F, pos))
    u = r(Q)
    gc, = torch.autograd.grad((gq * u).sum(), c)
    torch.testing.assert_close(gc, S.rotary_ref(u, F, pos))


def test_layer_checks(monkeypatch):
    w = torch.ones
    for heads, shapes in ((0, ((64, 8), (32, 8), (32, 8))), (3, ((64, 8), (32, 8), (32, 8))), (2, ((64, 8), (24, 8), (24, 8))),
                          (2, ((64, 8), (32, 8), (64, 8))), (2, ((0, 8), (32, 8), (32, 8)))):
        for layer in (S.mhc_attention_layer_fn, L.mhc_attention_layer_op):
            with pytest.raises(ValueError, match="mhc_attention_layer"):
                layer(None, None, None, None, None, None, *(w(s) for s in shapes), None, heads=heads)


# ---- GPU ---------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _layer_inputs(lead, N, D, H, Hk, d, dtype=torch.bfloat16, seed=0):
    """x, phi, alpha, base, norm weight and bias, w_q, w_k, w_v, w_out."""
    g = _gen(seed)
    r = lambda *s, scale=1.0, to=dtype: (torch.randn(*s, device=DEV, generator=g) * scale).to(to)
    M, f32 = N * (N + 2), torch.float32
    return [r(*lead, N, D), r(M, N * D, scale=(N * D) ** -0.5), torch.tensor([0.5, 0.5, 1.0], device=DEV),
            r(M, scale=0.1, to=f32), 1 + r(D, scale=0.1, to=f32), r(D, scale=0.1, to=f32),
            r(H * d, D, scale=D ** -0.5), r(Hk * d, D, scale=D ** -0.5), r(Hk * d, D, scale=D ** -0.5),
            r(D, H * d, scale=(H * d) ** -0.5)]


@pytest.mark.gpu
def test_opcheck():
    g = _gen(1)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g).to(torch.bfloat16)
    freqs, _ = S.rotary_frequencies(32)
    q, k, v = r(9, 4, 64).requires_grad_(True), r(9, 2, 64).requires_grad_(True), r(9, 2, 64)
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device=DEV)
    ops = torch.ops.flagos_mhc
    torch.library.opcheck(ops.rotary.default, (q, k, freqs, None, cu, "interleaved", 1.5, False))
    torch.library.opcheck(ops.rotary.default, (q, None, freqs, torch.arange(9, device=DEV)))
    torch.library.opcheck(ops.attention.default, (q, k, v, cu))
    torch.library.opcheck(ops.attention.default, (q, k, v, None, None, None, False, 0.2, True))
    out, lse = ops.attention(q.detach(), k.detach(), v, cu)
    torch.library.opcheck(ops.attention_backward.default, (r(9, 4, 64), q.detach(), k.detach(), v, out, lse, cu))


@pytest.mark.gpu
def test_layer_matches_its_parts_and_pytorch():
    """The layer's output and gradients equal those of the operators called one by
    one, and PyTorch's references in fp32 within the roundings between them."""
    T, N, D, H, Hk, d = 150, 4, 256, 6, 2, 64
    args = _layer_inputs((T,), N, D, H, Hk, d)
    cu = torch.tensor([0, 70, 70, 141, 150], dtype=torch.int32, device=DEV)
    freqs, amp = S.rotary_frequencies(32, scaling="yarn", factor=2.0, original_length=64)
    gy = torch.randn(T, N, D, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    kw = dict(dropout_p=0.2, seed=5, offset=9, clamp_min=-10.0, clamp_max=10.0)

    leaves = [t.clone().requires_grad_(True) for t in args]
    out = S.mhc_attention_layer_fn(*leaves, freqs, heads=H, cu_seqlens=cu, amplitude=amp, layout="interleaved", **kw)
    out.backward(gy)

    x, phi, alpha, base, nw, nb, wq, wk, wv, wo = args
    pre = m.mhc_pre_clamp_sinkhorn(x, phi, alpha, base, need_backward=True, clamp_min=-10.0, clamp_max=10.0)
    n = S.layer_norm(pre["y"], nw, nb, need_backward=True)
    q, k, v = ((n["y"] @ w.t()).view(T, -1, d) for w in (wq, wk, wv))
    rot = dict(cu_seqlens=cu, layout="interleaved", amplitude=amp)
    q, k = S.rotary(q, k, freqs, **rot)
    f = S.attention(q, k, v, cu, need_backward=True)
    h = S.dropout(f["out"].view(T, -1) @ wo.t(), 0.2, 5, 9)
    torch.testing.assert_close(out, m.mhc_post(x, pre["comb_frag"], h, pre["post_out"]), rtol=0, atol=0)
    _, _, gh, _ = m.mhc_post_backward(gy, x, pre["comb_frag"], h, pre["post_out"])
    go = S.dropout_backward(gh, 0.2, 5, 9)
    gf = (go @ wo).view(T, H, d)
    gq, gk, gv = S.attention_backward(gf, q, k, v, f["out"], f["lse"], cu)
    gq, gk = S.rotary_backward(gq, gk, freqs, **rot)
    # weights' gradients: the same products, in an order of the library's own
    for leaf, want in zip(leaves[6:], (gq, gk, gv, None)):
        w = go.t() @ f["out"].view(T, -1) if want is None else want.reshape(T, -1).t() @ n["y"]
        assert float((leaf.grad - w).float().norm() / w.float().norm()) <= 2 ** -8

    # the sublayer in PyTorch, in fp32, from the same y
    y = S.layer_norm_ref(pre["y"].float(), nw, nb)
    q, k, v = ((y @ w.float().t()).view(T, -1, d) for w in (wq, wk, wv))
    pos = torch.cat([torch.arange(c, device=DEV) for c in (70, 0, 71, 9)])
    q, k = (S.rotary_ref(t, freqs, pos, "interleaved", amp) for t in (q, k))
    ref = S.dropout_ref(S.attention_ref(q, k, v, cu).view(T, -1) @ wo.float().t(), 0.2, 5, 9)
    # roundings to bf16 on the way: norm, q, k, v, rotated, weights, out, projected, dropped
    assert float((h.float() - ref).norm() / ref.norm()) <= 9 * R.half_step(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(90,), (3, 30)])
def test_registered_layer_compiles_and_matches(lead):
    N, D, H, Hk, d = 4, 128, 4, 2, 32
    args = _layer_inputs(lead, N, D, H, Hk, d, seed=3)
    gy = torch.randn(*lead, N, D, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    freqs, _ = S.rotary_frequencies(32)
    cu = torch.tensor([0, 33, 90], dtype=torch.int32, device=DEV) if len(lead) == 1 else None
    kw = dict(heads=H, cu_seqlens=cu, dropout_p=0.3, seed=1 << 63, offset=3, scale=0.2)

    def run(fn):
        leaves = [t.clone().requires_grad_(True) for t in args]
        out = fn(*leaves)
        out.backward(gy)
        return [out.detach()] + [t.grad for t in leaves]

    want = run(lambda *a: S.mhc_attention_layer_fn(*a, freqs, **kw))
    torch._dynamo.reset()
    for fn in (lambda *a: L.mhc_attention_layer_op(*a, freqs, **kw),
               torch.compile(lambda *a: L.mhc_attention_layer_op(*a, freqs, **kw), backend="aot_eager", fullgraph=True)):
        got = run(fn)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            # (a compiled backward may take the library's products in another form)
            assert float((a.float() - b.float()).norm()) <= 2 ** -8 * float(b.float().norm()) + 1e-6


@pytest.mark.gpu
def test_no_rotation_and_positions():
    """Without freqs nothing is rotated; positions take the place of the packed rows'."""
    T, N, D, H, Hk, d = 40, 4, 128, 4, 4, 32
    args = _layer_inputs((T,), N, D, H, Hk, d, seed=5)
    freqs, _ = S.rotary_frequencies(32)
    cu = torch.tensor([0, 15, 40], dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(15), torch.arange(25)]).to(DEV)
    a = S.mhc_attention_layer_fn(*args, freqs, heads=H, cu_seqlens=cu)
    assert torch.equal(a, S.mhc_attention_layer_fn(*args, freqs, heads=H, cu_seqlens=cu, positions=pos))
    still = S.mhc_attention_layer_fn(*args, freqs, heads=H, cu_seqlens=cu, positions=torch.zeros_like(pos))
    assert torch.equal(still, S.mhc_attention_layer_fn(*args, heads=H, cu_seqlens=cu)) and not torch.equal(a, still)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,d", [(4, 2, 64), (32, 8, 128)])
def test_graph_replay(H, Hk, d):
    """A training step over packed sequences and a decoding step in captured
    graphs, replayed with eager work in between, other inputs, starts and lengths."""
    g = _gen(H)
    T, B, Lc = 700, 6, 3000
    r = lambda *s: torch.randn(*s, device=DEV, generator=g).to(torch.bfloat16)
    q, k, v, go = r(T, H, d), r(T, Hk, d), r(T, Hk, d), r(T, H, d)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    new, cache = r(B, 1, H, d), r(B, Lc, 2, Hk, d)
    used = torch.zeros(B, dtype=torch.int32, device=DEV)
    freqs, _ = S.rotary_frequencies(d)

    def step():
        qr, kr = S.rotary(q, k, freqs, cu_seqlens=cu)
        f = S.attention(qr, kr, v, cu, need_backward=True)
        gq, gk, gv = S.attention_backward(go, qr, kr, v, f["out"], f["lse"], cu)
        one, _ = S.rotary(new, None, freqs, used)
        return [f["out"], gv, *S.rotary_backward(gq, gk, freqs, cu_seqlens=cu),
                S.attention(one, cache[:, :, 0], cache[:, :, 1], lengths_k=used)["out"]]

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
    starts = ([0, 100, 100, 300, 301, 650, 700], [0, 0, 0, 0, 0, 0, 700], [0, 10, 20, 30, 40, 50, 60], [0, 699, 700, 700, 700, 700, 700])
    for rnd, at in enumerate(starts):
        cu.copy_(torch.tensor(at))
        used.copy_(torch.tensor([(997 * (rnd + 1) * (b + 1)) % (Lc + 1) for b in range(B)]))
        if rnd == 2:
            q.copy_(r(T, H, d))
            go.copy_(r(T, H, d))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, eager)):
            assert torch.equal(a, b), f"replay {rnd}: output {i} differs from eager"
