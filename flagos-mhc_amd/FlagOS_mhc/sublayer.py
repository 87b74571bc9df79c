"""The operators between mhc_pre_clamp_sinkhorn and mhc_post, and the mHC
feed-forward layer they make.

    from FlagOS_mhc.sublayer import layer_norm_fn, gated_ffn_fn, dropout_fn, mhc_ffn_layer_fn

``layer_norm``, ``gated_ffn`` and ``dropout`` run the HIP kernels of
``libmhc_amd.so`` on the current stream; each has its backward, an
autograd-aware ``*_fn`` and a PyTorch ``*_ref``.  The same operators are
registered as torch.ops.flagos_mhc.* (``FlagOS_mhc.library``).
"""

from __future__ import annotations

from .autograd import mhc_post_fn, mhc_pre_clamp_sinkhorn_fn
from .dropout import DropoutFn, dropout, dropout_backward, dropout_fn, dropout_ref
from .gated_ffn import GatedFfnFn, gated_ffn, gated_ffn_backward, gated_ffn_fn, gated_ffn_ref
from .layer_norm import LayerNormFn, layer_norm, layer_norm_backward, layer_norm_fn, layer_norm_ref

__all__ = [
    "layer_norm", "layer_norm_backward", "layer_norm_ref", "LayerNormFn", "layer_norm_fn",
    "gated_ffn", "gated_ffn_backward", "gated_ffn_ref", "GatedFfnFn", "gated_ffn_fn",
    "dropout", "dropout_backward", "dropout_ref", "DropoutFn", "dropout_fn",
    "mhc_ffn_layer_fn",
]


def mhc_ffn_layer_fn(x, phi, alpha, base, norm_weight, norm_bias, w_gate, w_up, w_down, *,
                     activation="silu", dropout_p=0.0, seed=0, offset=0, state=None, ln_eps=1e-5, **mhc):
    """One mHC feed-forward layer, autograd-aware: the residual streams x
    (..., N, D) are mixed into the sublayer's input, which is normalised, goes
    through the gated feed-forward block and dropout, and is written back into
    the streams.  ``mhc``: norm_eps, hc_eps, clamp_min, clamp_max, iter_times
    and compensated of ``mhc_pre_clamp_sinkhorn_fn``; seed, offset and state
    as in ``dropout``.  Returns the streams after the layer."""
    y, post, comb = mhc_pre_clamp_sinkhorn_fn(x, phi, alpha, base, **mhc)
    h = layer_norm_fn(y, norm_weight, norm_bias, ln_eps)
    h = gated_ffn_fn(h, w_gate, w_up, w_down, activation)
    if dropout_p != 0.0:
        h = dropout_fn(h, dropout_p, seed, offset, state)
    return mhc_post_fn(x, comb, h, post)
