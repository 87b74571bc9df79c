"""64-bit formulas of attention and rotary positions, and the bounds their
outputs are held to (test infrastructure).

H is half a step of the operands' type, U of fp32.  Bounds hold element by
element, from the roundings the operators document:
  score    d products added in fp32 (any order): d U sum |q k|, the factor and
           exp2's argument: 4 U |score|; its error is e^p's relative one, as is
           that of lse, and exp2's own 2 U
  weight   rounded to the type: H (fp32: none), in fp16 at least 2^-25 of the
           row's largest
  out      sum of weights times v: the weights' errors times |v|, n U for the sum
  D        go . out with out rounded: H sum |go out|, d U sum |go out|
  dS       P (dP - D): errors of P, dP (d U sum |go v|) and D, rounded: H
  dq, dk   sums of dS times k, q; dv of P times go; each rounded at the end: H
A result is rounded by H of its size, and in fp16 by at least 2^-25: its
numbers below 2^-14 are 2^-24 apart, so half a step there is 2^-25 (an element
of 2^-16.7 was off by 2.63e-8 = 0.88 * 2^-25, more than H of it, 2.35e-8 with
every other term).  fp32 and bf16 numbers below 2^-126 are zero to exp2 and the
matrix instructions: a weight, and a dS, may be off by that (scores that are
hundreds below their row's largest; an element of dk came as 5e-37, from
weights of 1e-38 times dP - D of 60 over a hundred queries)."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def head(q, k, v, go, scale, causal, dtype):
    """((out, bound), lse, [(dq, bound), (dk, bound), (dv, bound)]) of one head in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    h = half_step(dtype)
    hp = 0.0 if dtype == torch.float32 else h
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    s = (q @ k.t().contiguous()) * scale
    hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.arange(m, device=q.device)[None] > torch.arange(n, device=q.device)[:, None] + (m - n)
    s = s.masked_fill(hidden, -math.inf)
    if m == 0:
        z = torch.zeros_like(q)
        return (z, z), torch.full((n,), -math.inf, dtype=torch.float64, device=q.device), [(z, z), (k, k), (v, v)]
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[:, None])
    fin = torch.where(hidden, 0.0, s)
    # relative error of exp(score - reference): arguments are rounded relative to their size
    es = (d * U) * ((q.abs() @ k.abs().t().contiguous()) * scale) + 4 * U * fin.abs()
    es = es.masked_fill(hidden, 0.0)
    top = fin.abs().amax(1, keepdim=True)
    es = es + es.amax(1, keepdim=True) + 4 * U * top + (m + 8) * U
    out = p @ v
    pmax = p.amax(1, keepdim=True)
    av = v.abs()
    bo = (p * (es + hp)) @ av + tiny * pmax * 256 * av.sum(0) + (h + 4 * U) * out.abs() + tiny
    grads = []
    if go is not None:
        go = go.double()
        dp = go @ v.t().contiguous()
        D = (go * out).sum(1, keepdim=True)
        ds = p * (dp - D)
        eD = (go.abs() * bo).sum(1, keepdim=True) + d * U * (go * out).abs().sum(1, keepdim=True)
        e = p * (eD + d * U * (go.abs() @ av.t().contiguous())) + ds.abs() * (2 * es + hp) + tiny * (1 + (dp - D).abs())
        e = e.masked_fill(hidden, 0.0)
        dq, dk, dv = scale * (ds @ k), scale * (ds.t().contiguous() @ q), p.t().contiguous() @ go
        bq = scale * ((e + m * U * ds.abs()) @ k.abs()) + (h + 4 * U) * dq.abs() + tiny
        bk = scale * ((e + n * U * ds.abs()).t().contiguous() @ q.abs()) + (h + 4 * U) * dk.abs() + tiny
        ep = (p * (2 * es + hp + n * U) + tiny).masked_fill(hidden, 0.0)
        bv = ep.t().contiguous() @ go.abs() + (h + 4 * U) * dv.abs() + tiny
        grads = [(dq, bq), (dk, bk), (dv, bv)]
    return (out, bo), lse, grads


def sequences(rows, batch, cu):
    """[(first row, row past the last)] of packed or equally long sequences."""
    if cu is not None:
        at = [0] + [int(c) for c in cu[1:]]
        return list(zip(at, at[1:]))
    n = rows // max(1, batch)
    return [(b * n, (b + 1) * n) for b in range(batch)]


def full(q, k, v, go, cu_q, cu_k, lengths, batch, causal, scale):
    """Every head of packed rows (T, H, d): [(value, bound)] of out and the gradients, and lse; rows of no
    sequence are 0 with bound 0."""
    H, Hk = q.shape[1], k.shape[1]
    res = [(torch.zeros(t.shape, dtype=torch.float64, device=q.device), torch.zeros(t.shape, dtype=torch.float64, device=q.device))
           for t in (q, q, k, v)]
    lses = torch.full((H, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    ks = sequences(k.shape[0], batch, cu_k)
    for b, (lo, hi) in enumerate(sequences(q.shape[0], batch, cu_q)):
        klo, khi = ks[b]
        if lengths is not None:
            khi = klo + int(lengths[b])
        for h in range(H):
            c = h * Hk // H
            o, lse, g = head(q[lo:hi, h], k[klo:khi, c], v[klo:khi, c], None if go is None else go[lo:hi, h], scale, causal, q.dtype)
            lses[h, lo:hi] = lse
            for j, (val, bound) in enumerate([o, *g]):
                a, z = (lo, hi) if j < 2 else (klo, khi)
                col = h if j < 2 else c
                res[j][0][a:z, col] += val
                res[j][1][a:z, col] += bound
    return res, lses


def within(got, want, what):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    over = (got.double() - value).abs() - bound
    assert not bool(got.isnan().any()), f"{what}: NaN"
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0.0, f"{what}: an element is {worst:.3e} beyond its bound {float(bound.flatten()[over.argmax()]):.3e}"
