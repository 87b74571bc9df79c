"""Operands on two devices are refused before a kernel gets an address.  One
GPU, or none, is enough: stand-ins say where they are, and nothing else of
them is looked at before that."""

from __future__ import annotations

import types

import pytest
import torch

import FlagOS_mhc as m
from FlagOS_mhc import _lib, sublayer as S


def _on(index):
    return types.SimpleNamespace(is_cuda=True, device=torch.device("cuda", index), get_device=lambda: index)


CALLS = {
    "layer_norm": (S.layer_norm, 3),
    "layer_norm_backward": (S.layer_norm_backward, 5),
    "gated_ffn": (S.gated_ffn, 4),
    "gated_ffn_backward": (S.gated_ffn_backward, 8),
    "dropout": (lambda x, state: S.dropout(x, 0.5, state=state), 2),
    "mhc_post": (m.mhc_post, 4),
    "mhc_post_backward": (m.mhc_post_backward, 5),
    "mhc_pre_clamp_sinkhorn": (m.mhc_pre_clamp_sinkhorn, 4),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, count) in CALLS.items() for i in range(count)])
def test_another_device_is_refused(name, at):
    fn, count = CALLS[name]
    with pytest.raises(ValueError, match="expected one device"):
        fn(*[_on(1 if i == at else 0) for i in range(count)])


def test_one_device_and_absent_tensors_pass():
    _lib.require_device("op", None, _on(1), None, _on(1))
    with pytest.raises(RuntimeError, match="HIP"):
        _lib.require_device("op", _on(0), torch.zeros(1))
