"""The operators between mhc_pre_clamp_sinkhorn and mhc_post, and the mHC
feed-forward and attention layers they make.

    from FlagOS_mhc.sublayer import layer_norm_fn, gated_ffn_fn, dropout_fn, mhc_ffn_layer_fn
    from FlagOS_mhc.sublayer import rotary_frequencies, rotary_fn, attention_fn, mhc_attention_layer_fn

``layer_norm``, ``gated_ffn``, ``dropout``, ``rotary`` and ``attention`` run the HIP kernels of
``libmhc_amd.so`` on the current stream; each has its backward, an
autograd-aware ``*_fn`` and a PyTorch ``*_ref``.  The same operators are
registered as torch.ops.flagos_mhc.* (``FlagOS_mhc.library``).
"""

from __future__ import annotations

from torch.nn.functional import linear

from .attention import AttentionFn, attention, attention_backward, attention_fn, attention_ref, projected_width
from .autograd import mhc_post_fn, mhc_pre_clamp_sinkhorn_fn
from .dropout import DropoutFn, dropout, dropout_backward, dropout_fn, dropout_ref
from .gated_ffn import GatedFfnFn, gated_ffn, gated_ffn_backward, gated_ffn_fn, gated_ffn_ref
from .layer_norm import LayerNormFn, layer_norm, layer_norm_backward, layer_norm_fn, layer_norm_ref
from .rotary import RotaryFn, rotary, rotary_backward, rotary_fn, rotary_frequencies, rotary_ref

__all__ = [
    "layer_norm", "layer_norm_backward", "layer_norm_ref", "LayerNormFn", "layer_norm_fn",
    "gated_ffn", "gated_ffn_backward", "gated_ffn_ref", "GatedFfnFn", "gated_ffn_fn",
    "dropout", "dropout_backward", "dropout_ref", "DropoutFn", "dropout_fn",
    "rotary", "rotary_backward", "rotary_frequencies", "rotary_ref", "RotaryFn", "rotary_fn",
    "attention", "attention_backward", "attention_ref", "AttentionFn", "attention_fn",
    "mhc_ffn_layer_fn", "mhc_attention_layer_fn",
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


def mhc_attention_layer_fn(x, phi, alpha, base, norm_weight, norm_bias, w_q, w_k, w_v, w_out, freqs=None, *, heads,
                           cu_seqlens=None, positions=None, layout="half", amplitude=1.0, causal=True, scale=None,
                           dropout_p=0.0, seed=0, offset=0, state=None, ln_eps=1e-5, **mhc):
    """One mHC attention layer, autograd-aware: the residual streams x are
    mixed into the sublayer's input, which is normalised and projected to
    queries (w_q (heads * d, D)), keys and values (w_k, w_v (heads_k * d, D));
    those get their rotary positions (freqs and amplitude of
    ``rotary_frequencies``; None: none), the attention's result goes through
    w_out (D, heads * d) and dropout and is written back into the streams.
    x is (T, N, D) of packed sequences with cu_seqlens (or of one), or
    (B, S, N, D).  positions as in ``rotary``; ``mhc``: norm_eps, hc_eps,
    clamp_min, clamp_max, iter_times and compensated of
    ``mhc_pre_clamp_sinkhorn_fn``; seed, offset and state as in ``dropout``.
    The projections are torch's linear.  Returns the streams after the layer."""
    d = projected_width("mhc_attention_layer", heads, w_q, w_k, w_v)
    y, post, comb = mhc_pre_clamp_sinkhorn_fn(x, phi, alpha, base, **mhc)
    h = layer_norm_fn(y, norm_weight, norm_bias, ln_eps)
    q, k, v = (linear(h, w).unflatten(-1, (w.shape[0] // d, d)) for w in (w_q, w_k, w_v))
    if freqs is not None:
        at = None if positions is not None else cu_seqlens
        q, k = rotary_fn(q, k, freqs, positions, cu_seqlens=at, layout=layout, amplitude=amplitude)
    h = linear(attention_fn(q, k, v, cu_seqlens, causal=causal, scale=scale).flatten(-2), w_out)
    if dropout_p != 0.0:
        h = dropout_fn(h, dropout_p, seed, offset, state)
    return mhc_post_fn(x, comb, h, post)
