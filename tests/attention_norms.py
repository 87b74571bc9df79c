"""Norms of attention's errors, tensor by tensor (test infrastructure).  Bounds
element by element (attention_ref.py) add worst cases, which over hundreds of
keys leave room for a tenth of a gradient; norms do not.

bf16, fp16: twice the norm of rounding the exact result.  Two roundings of
independent values make a result: of the weights (out, dv) or of dS (dq, dk),
each by the type's relative step, which adds as much again as the result's own
rounding: sqrt(2) of it.  D from the rounded out is off by a relative step that
is the same for all of a query's keys: 1 / sqrt(keys) of that (it is taken so
beyond 256 keys).  fp32, and what of it the others hold: scores are off by
sqrt(d) U |q| |k| scale (d roundings of sums no larger, of independent sign), by
4 U of themselves as arguments of exp2, their row's lse by as much, sums over n
keys by sqrt(n) U, the rest by a few U."""

from __future__ import annotations

import math

from attention_ref import U


def fp32_part(q, k, scale, keys):
    """The relative error that fp32 leaves a result of these queries and keys."""
    size = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * scale
    return U * (2 * (math.sqrt(q.shape[-1]) + 4) * size + math.sqrt(keys) + 16)


def near(got, want, what, part):
    """got, in its type, is want (64 bits) but for the roundings above."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    own = float((want.to(got.dtype).double() - want).norm())
    err, size = float((got.double() - want).norm()), float(want.norm())
    assert err <= 2 * own + part * size, (f"{what}: error {err:.3e} of {size:.3e} ({err / size if size else 0:.2e}), "
                                          f"rounding {own:.3e}, fp32 {part * size:.3e}")
