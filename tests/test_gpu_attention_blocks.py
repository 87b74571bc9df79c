"""Every attention kernel on the GPU: blocks of 128 and of 256 queries (many
short sequences: many blocks, small references), parts of the keys and of the
queries, offsets past 32 bits, hidden infinities in each of them."""

from __future__ import annotations

import random

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_attention import DEV, DT, _check, _cu, _gen, _randn

pytestmark = pytest.mark.gpu


def _lengths(seed, B, longest):
    rng = random.Random(seed)
    n = [rng.choice([0, 1, rng.randint(2, 60), rng.randint(2, 200)]) for _ in range(B)]
    n[B // 2] = longest
    return n


def _inputs(lengths, H, Hk, d, dtype, pad=0, seed=0):
    g = _gen(seed + sum(lengths))
    T = sum(lengths) + pad
    return (*(_randn(g, T, n, d, dtype=DT[dtype]) for n in (H, Hk, Hk, H)), _cu(lengths))


# (heads, key heads) that choose a kernel for 70 sequences (tests/test_attention_plan.py checks that they do)
PAIRS, OF_128, OF_256 = (4, 2), (12, 4), (32, 8)


# 128 queries a block, with two waves for 32 of them or one
@pytest.mark.parametrize("heads", [PAIRS, OF_128])
@pytest.mark.parametrize("d", [64, 72, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
def test_blocks_of_128(heads, d, dtype, causal):
    if dtype == "f32" and d > 128:
        pytest.skip("fp32 heads wider than 128 are refused")
    print(f"[attention] 128: {heads} d={d} {dtype} causal={causal}", flush=True)
    q, k, v, go, cu = _inputs(_lengths(d, 70, 700), *heads, d, dtype, pad=5)
    _check(q, k, v, go, cu, causal=causal, what=f"{heads} {d} {dtype}")


# 256 queries, and keys, a block
@pytest.mark.parametrize("dtype,d,causal", [("bf16", 128, True), ("f16", 112, True), ("bf16", 128, False)])
def test_blocks_of_256(dtype, d, causal):
    print(f"[attention] 256: d={d} {dtype} causal={causal}", flush=True)
    q, k, v, go, cu = _inputs(_lengths(5, 70, 1200), *OF_256, d, dtype, pad=2)
    _check(q, k, v, go, cu, causal=causal, what=f"{d} {dtype}")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hk,d", [(8, 1, 64), (4, 4, 128), (6, 2, 96)])
def test_parts_of_the_keys(dtype, H, Hk, d):
    """Single tokens and short chunks over caches of different lengths."""
    g = _gen(H)
    for B, Sq, L in ((1, 1, 5000), (3, 1, 2100), (2, 5, 1537)):
        print(f"[attention] parts: B={B} Sq={Sq} L={L} {dtype}", flush=True)
        q, go = (_randn(g, B, Sq, H, d, dtype=DT[dtype]) for _ in range(2))
        k, v = (_randn(g, B, L, Hk, d, dtype=DT[dtype]) for _ in range(2))
        lengths = torch.tensor([L, 3, 0][:B], dtype=torch.int32, device=DEV)
        _check(q, k, v, go, lengths=lengths, what=f"{B} {Sq} {L}")


@pytest.mark.parametrize("B", [64, 65, 5000])
def test_many_sequences(B):
    """More sequences than one, and than 64, candidates a lane."""
    rng = random.Random(B)
    lengths = [rng.choice([0, 1, 1, 2]) for _ in range(B)]
    T = sum(lengths) + 3
    g = _gen(B)
    q, k, v, go = (_randn(g, T, n, 64, dtype=torch.bfloat16) for n in (4, 2, 2, 4))
    cu = _cu(lengths)
    f = S.attention(q, k, v, cu, need_backward=True)
    gq, gk, gv = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
    # in closed form: a first token copies its value, a second one weighs two
    first = torch.tensor([sum(lengths[:b]) for b in range(B) if lengths[b]], device=DEV)
    assert torch.equal(f["out"][first], v[first].repeat_interleave(2, 1))
    two = torch.tensor([sum(lengths[:b]) for b in range(B) if lengths[b] == 2], device=DEV)
    ks, vs, qd = (t.double() for t in (k, v, q))
    rep = lambda t: t.repeat_interleave(2, 1)
    s = torch.stack([(qd[two + 1] * rep(ks[two + i])).sum(-1) for i in (0, 1)], -1) / 8
    p = torch.softmax(s, -1)
    want = p[..., :1] * rep(vs[two]) + p[..., 1:] * rep(vs[two + 1])
    h = R.half_step(torch.bfloat16)
    size = p[..., :1] * rep(vs[two]).abs() + p[..., 1:] * rep(vs[two + 1]).abs()
    assert bool(((f["out"][two + 1].double() - want).abs() <= 2 * h * size + 1e-4 * size).all())
    assert not any(t[-3:].any() for t in (f["out"], gq, gk, gv))
    one = torch.tensor([sum(lengths[:b]) for b in range(B) if lengths[b] == 1], device=DEV)
    # a softmax of one key is constant: dP - D is the difference of two sums of 64 products, off by 64 U of their size each
    size = (go[one].double().abs() * rep(v[one].double().abs())).sum(-1, keepdim=True) * rep(k[one].double().abs()) / 8
    assert bool((gq[one].double().abs() <= 2 * 64 * R.U * size * (1 + 2 * h) + 1e-30).all())
    assert bool(((gv[one].double() - go[one].double().view(-1, 2, 2, 64).sum(2)).abs()
                 <= h * go[one].double().view(-1, 2, 2, 64).abs().sum(2) * 1.01).all())


def test_offsets_past_32_bits():
    """The last rows of a packed batch of 2.4 GB and the last sequence of a cache of 3.1 GB."""
    g = _gen(1)
    T, d, tail = 1_200_000, 256, 300
    k = torch.zeros(T, 4, d, dtype=torch.bfloat16, device=DEV)
    v, q = torch.zeros_like(k), torch.zeros(T, 4, d, dtype=torch.bfloat16, device=DEV)
    for t in (q, k, v):
        t[-tail:] = _randn(g, tail, 4, d, dtype=torch.bfloat16)
    assert (T - tail) * 4 * d * 2 > 1 << 31
    cu = torch.tensor([0] + [T - tail - 512 * i for i in range(2300, -1, -1)] + [T - 100, T], dtype=torch.int32, device=DEV)
    f = S.attention(q, k, v, cu, need_backward=True)
    want, _ = R.full(q[-tail:], k[-tail:], v[-tail:], q[-tail:], _cu([tail - 100, 100]), _cu([tail - 100, 100]), None, 2, True, d ** -0.5)
    R.within(f["out"][-tail:], want[0], "packed")
    go = q
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
    for i, gr in enumerate(grads):
        R.within(gr[-tail:], want[i + 1], f"packed gradient {i}")
    del f, grads, q, k, v
    B, L = 5, 300_000
    k = torch.zeros(B, L, 4, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    assert (B - 1) * L * 4 * d * 2 > 1 << 31
    for t in (k, v):
        t[-1, :70] = _randn(g, 70, 4, d, dtype=torch.bfloat16)
    q = _randn(g, B, 2, 8, d, dtype=torch.bfloat16)
    lengths = torch.tensor([L, 5, 0, L, 70], dtype=torch.int32, device=DEV)
    out = S.attention(q, k, v, lengths_k=lengths)["out"]
    want, _ = R.full(q[-1], k[-1, :70], v[-1, :70], None, None, None, None, 1, True, d ** -0.5)
    R.within(out[-1], want[0], "cache")
    assert not out[:4].any()


@pytest.mark.parametrize("d,H,Hk", [(64, *PAIRS), (128, *PAIRS), (64, *OF_128), (128, *OF_128), (128, *OF_256)])
def test_hidden_nans_in_blocks(d, H, Hk):
    """As for small calls: a token reaches no query before it and no key behind it."""
    lengths = _lengths(9, 70, 500)
    q, k, v, go, cu = _inputs(lengths, H, Hk, d, "bf16")
    at = sum(lengths[:35]) + 300  # within the long sequence
    lo, hi = sum(lengths[:35]), sum(lengths[:36])
    clean = S.attention(q, k, v, cu, need_backward=True)
    cg = S.attention_backward(go, q, k, v, clean["out"], clean["lse"], cu)
    before, other, behind = slice(lo, at), [slice(0, lo), slice(hi, None)], slice(at + 1, hi)

    def near(a, b, rows):
        # the tile with such a token is summed in another order: fp32 sums, then one rounding
        for r in rows:
            x, y = a[r].double(), b[r].double()
            assert bool(x.isfinite().all())
            assert float((x - y).norm()) <= 2 ** -8 * float(y.norm())

    for t in (k, v):
        old = t[at].clone()
        t[at, 0, 3] = float("nan")
        f = S.attention(q, k, v, cu, need_backward=True)
        gq, _, _ = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
        near(f["out"], clean["out"], [before, *other])
        near(gq, cg[0], [before, *other])
        assert bool(f["out"][at:hi, 0, 3].isnan().all())
        t[at] = old
    for t in (q, go):
        old = t[at].clone()
        t[at, 0, 3] = float("nan")
        f = S.attention(q, k, v, cu, need_backward=True)
        gq, gk, gv = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)
        near(gk, cg[1], [behind, *other])
        near(gv, cg[2], [behind, *other])
        near(gq, cg[0], [before, behind, *other])
        t[at] = old


def test_two_streams_at_once():
    """Calls on two streams, each with workspaces of its own, equal those alone."""
    works = []
    for i, (lengths, H, Hk, d) in enumerate((([900, 411], 8, 2, 128), ([1500], 4, 4, 64))):
        q, k, v, go, cu = _inputs(lengths, H, Hk, d, "bf16", seed=i)
        cache = _randn(_gen(i), 1, 6000, 2, Hk, d, dtype=torch.bfloat16)

        def step(q=q, k=k, v=v, go=go, cu=cu, cache=cache):
            f = S.attention(q, k, v, cu, need_backward=True)
            one = S.attention(q[None, :1], cache[:, :, 0], cache[:, :, 1])["out"]
            return [f["out"], one, *S.attention_backward(go, q, k, v, f["out"], f["lse"], cu)]

        works.append(step)
    want = [w() for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(5):
        got = []
        for s, w in zip(streams, works):
            with torch.cuda.stream(s):
                got.append(w())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
