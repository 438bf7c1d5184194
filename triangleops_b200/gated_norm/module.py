"""Public API of the fused norms around a block: the differentiable one-shot."""

from __future__ import annotations

import torch

from .. import _autograd
from . import kernel

_WEIGHTS = ("post_weight", "post_bias", "res_scale", "pre_weight", "pre_bias")


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, opts, eps, *weights):
        h, n, stats = kernel.forward(x, y, gate, eps=eps, **dict(zip(_WEIGHTS, weights)), **opts)
        ctx.save_for_backward(x, y, gate, stats, *weights)
        ctx.opts = opts
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    def backward(ctx, dh, dn):
        x, y, gate, stats, *weights = ctx.saved_tensors

        def call():
            g = kernel.backward(dh, dn, x, y, gate, stats, **dict(zip(_WEIGHTS, weights)), **ctx.opts)
            return (g["dx"], g["dy"], g.get("dgate"), *(g.get("d" + w) for w in _WEIGHTS))

        dx, dy, dgate, *dw = _autograd.first_order("gated_norm", call, dh, dn, x, y, gate, *weights)
        return (dx, dy, dgate, None, None, *dw)


def gated_norm(x, y, gate=None, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None, pre_bias=None,
               kind="layer", post_norm=True, pre_norm=True, eps=1e-5):
    """(h, n): the residual stream after a block's output y was normed, gated, scaled and added
    to x, and its norm for the next block (:mod:`triangleops_b200.gated_norm.kernel` has the
    definition); differentiable (once) in x, y, the gate and the weights."""
    opts = dict(kind=kind, post_norm=post_norm, pre_norm=pre_norm)
    return _GatedNorm.apply(x, y, gate, opts, eps, post_weight, post_bias, res_scale, pre_weight, pre_bias)
