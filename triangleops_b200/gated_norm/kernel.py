"""The norms around a block fused with its gate and residual scale: the launchers.

    u = post(y)                      the norm after the block (``post_norm=False``: u = y)
    r = u * sigmoid(gate)            (no ``gate``: r = u)
    h = x + res_scale * r            the residual stream
    n = pre(h)                       the norm before the next block (``pre_norm=False``: none)

``kind`` "layer": norm(t) = (t - mean) / sqrt(var + eps) * weight + bias;
"rms": t / sqrt(mean(t^2) + eps) * weight (+ bias). A weight of None is 1, a bias 0.
x and y are (..., C) of one shape. The gate has x's shape, or 1 in the last places before C
(one row for all tokens of a sample: ``(B, 1, C)``). C <= 8192. Weights in x's dtype or fp32.

One launch reads each tensor once and writes each once; statistics and sums are fp32. No
counterpart in the reference, which folds its norms into the projections.
"""

from __future__ import annotations

from .. import _lib

_GRADS = ("dx", "dy", "dgate", "dpost_weight", "dpost_bias", "dres_scale", "dpre_weight", "dpre_bias")


def forward(x, y, gate=None, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None, pre_bias=None,
            kind="layer", post_norm=True, pre_norm=True, eps=1e-5):
    """-> (h, n, stats): h and n like x (n None without ``pre_norm``), stats (..., 4) fp32 for
    :func:`backward` (mean and 1/std of y, of h)."""
    return _lib.bind().gated_norm_forward(x, y, gate, post_weight, post_bias, res_scale, pre_weight, pre_bias, kind,
                                          post_norm, pre_norm, eps)


def backward(dh, dn, x, y, gate, stats, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None,
             pre_bias=None, kind="layer", post_norm=True, pre_norm=True):
    """Gradients from those of h and n (either may be None: zero), as a dict: ``dx``, ``dy``,
    ``dgate`` (with a gate, in its shape) and ``d<name>`` for each weight given, in its dtype
    (summed over the tokens in fp32, in a fixed order)."""
    got = _lib.bind().gated_norm_backward(dh, dn, x, y, gate, stats, post_weight, post_bias, res_scale, pre_weight,
                                          pre_bias, kind, post_norm, pre_norm)
    return {k: t for k, t in zip(_GRADS, got) if t is not None}
