"""The feed-forward layer hands every dropout_p but zero to dropout, whose check
refuses what is no probability.  No GPU: what comes before is replaced."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import _lib, library as L, sublayer as S

X, Y = torch.ones(3, 2, 4), torch.ones(3, 4)


@pytest.fixture(autouse=True)
def no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    for module, suffix in ((S, "_fn"), (L, "_op")):
        monkeypatch.setattr(module, "mhc_pre_clamp_sinkhorn" + suffix, lambda *a, **k: (Y, None, None))
        monkeypatch.setattr(module, "layer_norm" + suffix, lambda h, *a: h)
        monkeypatch.setattr(module, "gated_ffn" + suffix, lambda h, *a: h)
        monkeypatch.setattr(module, "mhc_post" + suffix, lambda x, comb, h, post: x * h.sum())


@pytest.mark.parametrize("layer", [S.mhc_ffn_layer_fn, L.mhc_ffn_layer_op])
@pytest.mark.parametrize("p", [-0.1, -1e-9, float("nan"), 1.5, float("-inf")])
def test_no_probability_is_refused(layer, p):
    with pytest.raises(ValueError, match="no probability"):
        layer(X, *(None,) * 8, dropout_p=p)


@pytest.mark.parametrize("layer", [S.mhc_ffn_layer_fn, L.mhc_ffn_layer_op])
@pytest.mark.parametrize("p", [0, 0.0, -0.0])
def test_zero_leaves_dropout_out(layer, p):
    assert torch.equal(layer(X, *(None,) * 8, dropout_p=p), X * 12)
