"""Public API of windowed attention with sinks: the differentiable one-shot."""

from __future__ import annotations

import torch

from .. import _autograd
from . import kernel


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, mask):
        out, lse = kernel.forward(q, k, v, window=window, sinks=sinks, scale=scale, mask=mask)
        ctx.save_for_backward(q, k, v, out, lse, mask)
        ctx.opts = dict(window=window, sinks=sinks, scale=scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, mask = ctx.saved_tensors
        grads = _autograd.first_order(
            "window_attention", lambda: kernel.backward(dout, q, k, v, out, lse, mask=mask, **ctx.opts), dout, q, k, v)
        return (*grads, None, None, None, None)


def window_attention(q, k, v, *, window, sinks=0, scale=None, mask=None):
    """softmax(scale q k^T) v over each query's window and the first ``sinks`` keys
    (:mod:`triangleops_b200.window_attn.kernel` has the definition); differentiable (once) in q, k
    and v. q (B, Nq, Hq, D), k and v (B, Nk, Hkv, D) -> (B, Nq, Hq, D)."""
    return _WindowAttention.apply(q, k, v, window, sinks, scale, mask)
