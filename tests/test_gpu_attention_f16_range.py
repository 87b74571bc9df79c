"""fp16's narrow range in attention's backward: weights of rows over many keys, and
gradients of the scores far below 2^-14 or past 65504, in every kernel that
rounds them to fp16.

Norms of errors are held to twice that of rounding the exact result.  Two
roundings of independent values make a result: of the weights (out, dv) or of
dS (dq, dk), each to within the type's relative half step while they are normal
numbers, which adds as much again as the result's own rounding; together
sqrt(2) of it.  D from the rounded out is off by a relative step that is the
same for all of a query's keys and so adds 1 / sqrt(keys) of that.  fp32's part,
64 products and sums of 2^-24, is below 2^-17 of the result."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _exact(q, k, v, go, scale):
    """(out, dq, dk, dv) of one sequence, every key seen, in 64 bits."""
    H, Hk = q.shape[1], k.shape[1]
    res = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (q, q, k, v)]
    for h in range(H):
        c = h * Hk // H
        qh, kh, vh, gh = q[:, h].double(), k[:, c].double(), v[:, c].double(), go[:, h].double()
        p = torch.softmax(torch.mm(qh, kh.t().contiguous()) * scale, 1)
        o = torch.mm(p, vh)
        ds = torch.mm(gh, vh.t().contiguous())
        ds.sub_((gh * o).sum(1, keepdim=True)).mul_(p)
        res[0][:, h] = o
        res[1][:, h] = scale * torch.mm(ds, kh)
        res[2][:, c] += scale * torch.mm(ds.t().contiguous(), qh)
        res[3][:, c] += torch.mm(p.t().contiguous(), gh)
    return res


def _near(got, want, what):
    own = float((want.to(F16).double() - want).norm())
    err, size = float((got.double() - want).norm()), float(want.norm())
    assert err <= 2 * own + 2.0 ** -17 * size, f"{what}: error {err / size:.2e} of its size, rounding {own / size:.2e}"


# T, H, Hk, d: rows of a group in tiles of 32; waves that share keys; blocks of 128; of 256; wide heads
KERNELS = {"split": (8192, 2, 1, 64), "pairs": (8192, 8, 4, 64), "pairs_128": (4096, 16, 4, 128), "of_128": (8192, 16, 8, 96),
           "of_256": (8192, 64, 16, 128), "wide": (4096, 24, 8, 256)}


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, "dq", "dk"])
def test_small_gradients(kernel, size):
    """grad_out of 1e-4, over thousands of keys; and of 2^-16 where dq ("dq": small
    queries, large keys) or dk are nevertheless normal numbers."""
    print(f"[attention f16] {kernel} {size}", flush=True)
    T, H, Hk, d = KERNELS[kernel]
    g = _gen(T + H + d)
    r = lambda n, s=1.0: (torch.randn(T, n, d, device=DEV, generator=g) * s).to(F16)
    up = {"dq": 2.0 ** -10, "dk": 2.0 ** 10}.get(size, 1.0)
    q, k, v = r(H, up), r(Hk, 1 / up), r(Hk)
    go = r(H, size if isinstance(size, float) else 2.0 ** -16)
    f = S.attention(q, k, v, causal=False, need_backward=True)
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], causal=False)
    want = _exact(q, k, v, go, d ** -0.5)
    for name, a, b in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
        if size in ("dq", "dk") and name in ("grad_q", "grad_k") and name[-1] != size[-1]:
            continue  # the other one is below the type's numbers
        _near(a, b, f"{kernel} {size} {name}")


@pytest.mark.parametrize("H,Hk", [(2, 1), (4, 2), (12, 4), (64, 16)])
@pytest.mark.parametrize("d", [64, 128, 192])
def test_large_gradients(H, Hk, d):
    """dS past 65504 where dq and dk are far within: two to four keys, gradients of 1.2e4."""
    print(f"[attention f16] large {H} {Hk} {d}", flush=True)
    lengths = [2, 3, 4, 2] * 70
    T, g = sum(lengths), _gen(H + d)
    r = lambda n, s=1.0: (torch.randn(T, n, d, device=DEV, generator=g) * s).to(F16)
    q, k, v, go = r(H), r(Hk), r(Hk), r(H, 1.2e4)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    scale = 2.0 ** -7
    f = S.attention(q, k, v, cu, causal=False, scale=scale, need_backward=True)
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu, causal=False, scale=scale)
    parts = [_exact(*(x[a:b] for x in (q, k, v, go)), scale) for a, b in zip(cu.tolist(), cu.tolist()[1:])]
    want = [torch.cat(w) for w in zip(*parts)]
    for name, a, b in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
        # (a draw in 2e7 is beyond 5.46 of its deviation and infinite in fp16 itself, and dv, sums of
        # up to 16 of them, passes 65504 now and then: the exact result tells)
        fits = b.abs() < 65504 * (1 - 2.0 ** -9)
        assert float(fits.double().mean()) > 0.999
        assert bool(a[fits].isfinite().all()), name
        _near(a[fits], b[fits], f"{H} {d} {name}")


@pytest.mark.parametrize("kernel", ["split", "pairs", "of_128", "of_256"])
@pytest.mark.parametrize("rising", [True, False])
def test_gradients_of_different_sizes(kernel, rising):
    """Queries whose gradients rise (fall) by 2^24 along the sequence: each query's dq has
    the precision of its own size, whatever its neighbours'; dk is that of the largest."""
    T, H, Hk, d = KERNELS[kernel]
    T //= 4
    print(f"[attention f16] {kernel} {rising}", flush=True)
    g = _gen(T + d)
    r = lambda n, s=1.0: (torch.randn(T, n, d, device=DEV, generator=g) * s).to(F16)
    q, k, v = r(H, 2.0 ** -9), r(Hk, 2.0 ** 9), r(Hk)
    sizes = torch.exp2(torch.linspace(-16, 8, T, device=DEV))
    go = (torch.randn(T, H, d, device=DEV, generator=g) * (sizes if rising else sizes.flip(0))[:, None, None]).to(F16)
    f = S.attention(q, k, v, causal=False, need_backward=True)
    gq, gk, gv = S.attention_backward(go, q, k, v, f["out"], f["lse"], causal=False)
    _, wq, wk, wv = _exact(q, k, v, go, d ** -0.5)
    _near(gv, wv, "grad_v")
    for lo in range(0, T, T // 16):  # of runs of neighbours
        _near(gq[lo:lo + T // 16], wq[lo:lo + T // 16], f"grad_q from {lo}")
    # the same sizes along the keys
    q2, k2 = k[:, :1].expand(T, H, d).contiguous(), q[:, :Hk].contiguous()
    f = S.attention(q2, k2, v, causal=False, need_backward=True)
    _, gk, _ = S.attention_backward(go, q2, k2, v, f["out"], f["lse"], causal=False)
    _near(gk, _exact(q2, k2, v, go, d ** -0.5)[2], "grad_k")
