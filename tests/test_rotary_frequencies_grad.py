"""Frequencies that are trained: their gradient is not computed, and a call that
would leave it out without a word is refused."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from FlagOS_mhc import library as L, sublayer as S
from test_attention_library import F, K, Q, no_kernels  # noqa: F401 (no_kernels is a fixture)

OPS = torch.ops.flagos_mhc
CALLS = {"fn": lambda q, f: S.rotary_fn(q, K, f), "fn of q alone": lambda q, f: S.rotary_fn(q, None, f),
         "op": lambda q, f: L.rotary_op(q, K, f), "registered": lambda q, f: OPS.rotary(q, K, f)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("trained", [True, False])
def test_trained_frequencies_are_refused(no_kernels, name, trained):  # noqa: F811
    q, f = Q.clone().requires_grad_(trained), F.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="freqs"):
        CALLS[name](q, f)
    with torch.no_grad():
        assert CALLS[name](q, f)[0].shape == Q.shape
    assert CALLS[name](q, f.detach())[0].requires_grad == trained


@pytest.mark.parametrize("name", [n for n in CALLS if n != "registered"])
def test_tangents_of_frequencies_are_refused(no_kernels, name):  # noqa: F811
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            CALLS[name](Q, fwAD.make_dual(F, torch.ones_like(F)))
