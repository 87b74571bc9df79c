"""Norms of the errors of every attention kernel, tensor by tensor and sequence by
sequence (bounds: tests/attention_norms.py)."""

from __future__ import annotations

import pytest
import torch

import attention_norms as N
import attention_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_attention import DEV, DT, _cu, _gen, _randn

pytestmark = pytest.mark.gpu

# lengths, H, Hk, widths: rows of a group in tiles of 32, waves that share rows, blocks of 128, of 256
KERNELS = {"split": ([900, 40, 333], 4, 2, (64, 128, 192, 256)), "pairs": ([700, 500, 3, 200], 32, 4, (64, 96, 128, 192)),
           "of_128": ([700, 500, 3, 200], 64, 16, (64, 128, 256)), "of_256": ([2100, 1900], 128, 32, (128,))}
CALLS = [(n, d, t, c) for n, (_, _, _, widths) in KERNELS.items() for d in widths for t in ("bf16", "f16", "f32")
         for c in (True, False) if not (t == "f32" and (d > 128 or n == "of_256"))]


def _sequences(lengths, T):
    at = [0, *torch.tensor(lengths).cumsum(0).tolist()]
    return [("all", slice(0, T)), *((f"sequence {i}", slice(a, b)) for i, (a, b) in enumerate(zip(at, at[1:])) if b - a > 32)]


@pytest.mark.parametrize("kernel,d,dtype,causal", CALLS)
def test_norms(kernel, d, dtype, causal):
    lengths, H, Hk, _ = KERNELS[kernel]
    print(f"[attention norms] {kernel} d={d} {dtype} causal={causal}", flush=True)
    g, T = _gen(d + H), sum(lengths)
    q, k, v, go = (_randn(g, T, n, d, dtype=DT[dtype]) for n in (H, Hk, Hk, H))
    cu, scale = _cu(lengths), d ** -0.5
    f = S.attention(q, k, v, cu, causal=causal, need_backward=True)
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], cu, causal=causal)
    want, _ = R.full(q, k, v, go, cu, cu, None, len(lengths), causal, scale)
    part = N.fp32_part(q, k, scale, max(lengths) * (H // Hk))
    for name, got, (w, _) in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
        for what, rows in _sequences(lengths, T):
            N.near(got[rows], w[rows], f"{kernel} {d} {dtype} {name}, {what}", part)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,Sq,L,H,Hk,d", [(1, 1, 5000, 8, 1, 64), (3, 1, 2100, 4, 4, 128), (2, 5, 1537, 6, 2, 96), (70, 1, 2100, 8, 2, 128)])
def test_norms_over_caches(B, Sq, L, H, Hk, d, dtype):
    """Single tokens and short chunks, in parts of the keys; their gradients."""
    g = _gen(B + L)
    q, go = (_randn(g, B, Sq, H, d, dtype=DT[dtype]) for _ in range(2))
    k, v = (_randn(g, B, L, Hk, d, dtype=DT[dtype]) for _ in range(2))
    lengths = torch.tensor([L - 37 * b % (L // 2) for b in range(B)], dtype=torch.int32, device=DEV)
    f = S.attention(q, k, v, lengths_k=lengths, need_backward=True)
    grads = S.attention_backward(go, q, k, v, f["out"], f["lse"], lengths_k=lengths)
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, _ = R.full(flat(q), flat(k), flat(v), flat(go), None, None, lengths, B, True, d ** -0.5)
    part = N.fp32_part(q, k, d ** -0.5, L)
    for name, got, (w, _) in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
        N.near(flat(got), w, f"{B} {Sq} {L} {dtype} {name}", part)
