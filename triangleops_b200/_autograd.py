"""What the differentiable one-shots share: gradients that are constants to autograd say so."""

from __future__ import annotations

import torch


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, call, *inputs):
        ctx.what = what
        return call()

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no second derivatives: its gradients were computed by a kernel")


def first_order(what, call, *inputs):
    """``call()``, the gradients that a backward pass made of ``inputs``. Where that pass is itself
    recorded (``create_graph=True``) they carry a node that refuses to be differentiated:
    without one, autograd would take them for constants and leave terms out."""
    return _Once.apply(what, call, *inputs) if torch.is_grad_enabled() else call()
