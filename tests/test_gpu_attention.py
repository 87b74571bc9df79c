"""Attention on the GPU against 64-bit formulas (bounds: tests/attention_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _cu(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _flat(t):
    return t.reshape(-1, *t.shape[-2:])


def _check(q, k, v, go, cu=None, cu_k=None, lengths=None, causal=True, scale=None, what=""):
    """Forward and backward of a call against the formulas."""
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    kw = dict(cu_seqlens_k=cu_k, lengths_k=lengths, causal=causal, scale=scale)
    f = S.attention(q, k, v, cu, need_backward=True, **kw)
    only = S.attention(q, k, v, cu, **kw)["out"]
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu, **kw)
    torch.cuda.synchronize()
    ck = cu if cu_k is None and cu is not None and k.dim() == 3 and lengths is None else cu_k
    batch = cu.numel() - 1 if cu is not None else (q.shape[0] if q.dim() == 4 else 1)
    want, lse = R.full(_flat(q), _flat(k), _flat(v), _flat(go), cu, ck, lengths, batch, causal, sc)
    for name, got, w in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
        assert got.dtype == q.dtype and got.is_contiguous()
        R.within(_flat(got), w, f"{what} {name}")
    R.within(_flat(only), want[0], f"{what} out alone")
    assert f["out"].shape == q.shape and [g.shape for g in grads] == [q.shape, k.shape, v.shape]
    assert torch.equal(f["lse"].isinf(), lse.isinf())
    fin = ~lse.isinf()
    d = q.shape[-1]
    # (rows past a cache's lengths are NaN here, and no part of it)
    size = float(_flat(q).double().norm(dim=-1).max() * _flat(k).double().norm(dim=-1).nan_to_num(0).max()) * sc if k.numel() else 0.0
    err = (f["lse"].double() - lse)[fin].abs()
    assert not err.numel() or float(err.max()) <= (2 * d * size + k.shape[0] + 16) * R.U + 8 * R.U * float(lse[fin].abs().max())
    return f, grads


PACKED = [
    # lengths, H, Hk, d
    ([1], 1, 1, 64), ([1, 1, 1], 2, 1, 64), ([5], 4, 2, 64), ([0, 7, 0], 2, 2, 128), ([33, 31, 64, 65], 4, 1, 64),
    ([127, 129], 6, 2, 128), ([200, 0, 57], 2, 2, 80), ([300], 7, 1, 128), ([96, 513], 2, 1, 96), ([130, 40], 2, 1, 256),
    ([70, 3], 4, 4, 192), ([65], 2, 2, 8), ([1030], 2, 1, 64), ([150, 20], 3, 3, 33),
]


def _packed(lengths, H, Hk, d, dtype, pad=0, seed=0):
    g = _gen(seed + sum(lengths) + d)
    T = sum(lengths) + pad
    return (*(_randn(g, T, n, d, dtype=DT[dtype]) for n in (H, Hk, Hk, H)), _cu(lengths))


@pytest.mark.parametrize("lengths,H,Hk,d", PACKED)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(lengths, H, Hk, d, dtype, causal):
    print(f"[attention] {lengths} H={H} Hk={Hk} d={d} {dtype} causal={causal}", flush=True)
    pad = 3 if len(lengths) > 1 else 0
    q, k, v, go, cu = _packed(lengths, H, Hk, d, dtype, pad)
    if dtype == "f32" and d > 128:
        with pytest.raises(NotImplementedError, match="width"):
            S.attention(q, k, v, cu)
        pytest.skip("fp32 heads wider than 128 are refused: a first kernel for them faulted, its cause is not known")
    f, grads = _check(q, k, v, go, cu, causal=causal, what=f"{lengths} {dtype}")
    if pad:  # rows behind the last sequence
        assert not any(t[-pad:].any() for t in (f["out"], *grads)) and bool((f["lse"][:, -pad:] == -math.inf).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 700), (4, 130), (70, 300), (130, 64), (33, 0)])
def test_queries_are_the_last_positions(dtype, Sq, Sk):
    """Batches with fewer or more queries than keys; more: the first see nothing."""
    print(f"[attention] Sq={Sq} Sk={Sk} {dtype}", flush=True)
    g = _gen(Sq * 7 + Sk)
    B, H, Hk, d = 3, 4, 2, 64
    q, k, v, go = (_randn(g, B, s, n, d, dtype=DT[dtype]) for s, n in ((Sq, H), (Sk, Hk), (Sk, Hk), (Sq, H)))
    f, _ = _check(q, k, v, go, what="batched")
    if Sq > Sk:
        assert not f["out"][:, :Sq - Sk].any() and bool((f["lse"].view(H, B, Sq)[:, :, :Sq - Sk] == -math.inf).all())
    _check(q, k, v, go, causal=False, what="batched, all")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cache_lengths(dtype):
    """Rows of a cache past the lengths are not read: they hold NaN."""
    g = _gen(3)
    B, S_, L, H, Hk, d = 5, 2, 333, 8, 2, 128
    q, go = (_randn(g, B, S_, H, d, dtype=DT[dtype]) for _ in range(2))
    cache = _randn(g, B, L + 7, 2, Hk, d, dtype=DT[dtype])
    lengths = torch.tensor([333, 0, 1, 65, 128], dtype=torch.int32, device=DEV)
    for b, n in enumerate(lengths.tolist()):
        cache[b, n:] = float("nan")
    k, v = cache[:, :L, 0], cache[:, :L, 1]
    _check(q, k, v, go, lengths=lengths, what="cache")
    cu = _cu([3, 0, 1, 2, 4])  # as many new tokens as each sequence has, packed
    qp, gp = (_randn(g, 10, H, d, dtype=DT[dtype]) for _ in range(2))
    _check(qp, k, v, gp, cu, lengths=lengths, what="packed queries over a cache")
    _check(qp, k, v, gp, cu, lengths=lengths, causal=False, what="packed queries over a cache, all")


def test_packed_queries_and_keys_of_their_own():
    g = _gen(4)
    lq, lk = [40, 0, 5, 100], [64, 9, 0, 30]
    q, go = (_randn(g, sum(lq), 4, 64, dtype=torch.bfloat16) for _ in range(2))
    k, v = (_randn(g, sum(lk) + 2, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    for causal in (True, False):
        _, grads = _check(q, k, v, go, _cu(lq), _cu(lk), causal=causal, what="lq, lk")
        assert not grads[1][-2:].any() and not grads[2][-2:].any()


def test_views_of_one_projection():
    g = _gen(5)
    T, H, Hk, d = 150, 4, 2, 64
    qkv = _randn(g, T, H + 2 * Hk, d, dtype=torch.bfloat16)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    go = _randn(g, H, T, d, dtype=torch.bfloat16).transpose(0, 1)
    f, grads = _check(q, k, v, go, what="views")
    same = S.attention(q.contiguous(), k.contiguous(), v.contiguous())["out"]
    assert torch.equal(f["out"], same)
    odd = _randn(g, T * 3 * d + 1, dtype=torch.bfloat16)[1:].view(T, 3, d)  # no multiple of 16 bytes
    _check(odd[:, :1], odd[:, 1:2], odd[:, 2:], _randn(g, T, 1, d, dtype=torch.bfloat16), what="unaligned")
    one = _randn(g, 1, 1, d, dtype=torch.bfloat16).expand(T, 1, d)
    _check(q[:, :1], one, one, go[:, :1], what="one key for all")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores_and_scale(dtype):
    """Scores of hundreds, rising and falling along the keys: the reference point moves."""
    g = _gen(6)
    q, k, v, go = (_randn(g, 400, 2, 64, dtype=DT[dtype]) for _ in range(4))
    ramp = torch.linspace(0.1, 6, 400, device=DEV)[:, None, None]
    _check((q * 3).to(DT[dtype]), (k * ramp).to(DT[dtype]), v, go, what="rising")
    _check((q * 3).to(DT[dtype]), (k * ramp.flip(0)).to(DT[dtype]), v, go, scale=0.7, what="falling")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_hidden_infinities_and_nans(dtype):
    """What a token holds reaches no query before it, and no key behind it (those
    keep their values; a tile with such a token is summed in another order)."""
    q, k, v, go, cu = _packed([100, 60], 2, 1, 64, dtype)
    want, _ = R.full(q, k, v, go, cu, cu, None, 2, True, 64 ** -0.5)

    def same(i, got, *rows):
        for r in rows:
            R.within(got[r], tuple(w[r] for w in want[i]), f"{i} {r}")

    before, behind, other = slice(0, 70), slice(71, 100), slice(100, 160)
    for t, val in ((k, float("nan")), (v, float("nan")), (v, float("inf")), (k, -float("inf"))):
        old = t[70].clone()
        t[70, 0, 5] = val
        f = S.attention(q, k, v, cu, need_backward=True)
        same(0, f["out"], before, other)
        assert t is k or not bool(f["out"][70:100, :, 5].isfinite().any())
        gq, _, _ = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
        same(1, gq, before, other)
        t[70] = old
    for t in (q, go):  # a query that is broken: keys behind it do not see it
        old = t[70].clone()
        t[70, 0, 5] = float("nan")
        f = S.attention(q, k, v, cu, need_backward=True)
        gq, gk, gv = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
        same(2, gk, behind, other)
        same(3, gv, behind, other)
        same(1, gq, before, behind, other)
        assert bool((gk if t is q else gv)[:71].isnan().any())
        t[70] = old


def test_repeats_bit_for_bit_and_streams():
    q, k, v, go, cu = _packed([700, 333], 8, 2, 128, "bf16")
    runs = []
    for _ in range(3):
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            f = S.attention(q, k, v, cu, need_backward=True)
            grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
        s.synchronize()
        runs.append((f["out"], f["lse"], *grads))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_autograd():
    q, k, v, go, cu = _packed([90, 41], 4, 2, 64, "bf16", pad=2)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    S.attention_fn(*leaves, cu).backward(go)
    f = S.attention(q, k, v, cu, need_backward=True)
    want = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))
    with torch.no_grad():
        assert torch.equal(S.attention_fn(*leaves, cu), f["out"])


def test_gradients_against_differences():
    q, k, v, go, cu = _packed([20, 13], 2, 1, 16, "f32")
    f = S.attention(q, k, v, cu, need_backward=True)
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
    g = _gen(9)
    for i, gr in enumerate(grads):
        u = _randn(g, *gr.shape)
        t = [q, k, v]
        step = 2.0 ** -6
        at = lambda s: float((S.attention(*[x + s * u if j == i else x for j, x in enumerate(t)], cu)["out"].double() * go).sum())
        # central differences of two steps, extrapolated: error of the order step^4
        d1, d2 = ((at(s) - at(-s)) / (2 * s) for s in (step, step / 2))
        num = (4 * d2 - d1) / 3
        assert abs(num - float((gr.double() * u).sum())) <= 1e-3 * float(gr.norm() * u.norm())
