"""The check of norms tells the operators' roundings from mistakes (on the CPU)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_norms as N
import attention_ref as R


def _kernels(q, k, v, go, scale, causal, dtype, half_D=False, drop=None):
    """out, dq, dk, dv as the kernels round them, and with a mistake: D halved, or a tile of keys
    left out of the second product."""
    r = lambda t: t.to(dtype).double()
    n, m = q.shape[0], k.shape[0]
    s = (q.double() @ k.double().t()) * scale
    hidden = torch.arange(m)[None] > torch.arange(n)[:, None] + (m - n) if causal else torch.zeros(n, m, dtype=torch.bool)
    s = s.masked_fill(hidden, -math.inf)
    e = torch.exp(s - s.amax(1, keepdim=True))
    p, keep = torch.softmax(s, 1), torch.ones(m, dtype=torch.float64)
    if drop is not None:
        keep[drop:drop + 32] = 0
    out = r((r(e) * keep) @ v.double() / e.sum(1, keepdim=True))
    D = (go.double() * out).sum(1, keepdim=True) * (0.5 if half_D else 1)
    ds = r(p * (go.double() @ v.double().t() - D)) * keep
    return out, r(scale * ds @ k.double()), r(scale * ds.t() @ q.double()), r(r(p).t() @ go.double())


@pytest.mark.parametrize("n,d", [(300, 64), (700, 256), (1200, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_roundings_pass_and_mistakes_do_not(n, d, dtype, causal):
    g = torch.Generator().manual_seed(n + d)
    q, k, v, go = (torch.randn(n, d, generator=g).to(dtype) for _ in range(4))
    scale = d ** -0.5
    (out, _), _, grads = R.head(q, k, v, go, scale, causal, dtype)
    want, part = [out, *(g_[0] for g_ in grads)], N.fp32_part(q, k, scale, n)
    passes = lambda got: [_passes(a, b, part, dtype) for a, b in zip(got, want)]
    first = 256 if causal else 0  # (queries of few keys have D from the weights themselves)
    good = _kernels(q, k, v, go, scale, causal, dtype)
    assert all(passes(good)[i] for i in (0, 2, 3)) and _passes(good[1][first:], want[1][first:], part, dtype)
    assert not any(passes(_kernels(q, k, v, go, scale, causal, dtype, half_D=True))[1:3])
    assert not any(passes(_kernels(q, k, v, go, scale, causal, dtype, drop=n // 2))[:3])


def _passes(got, want, part, dtype):
    try:
        N.near(got.to(dtype), want, "", part)
        return True
    except AssertionError:
        return False
