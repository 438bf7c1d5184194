"""Public API of rotary positions: the tables of frequencies and the differentiable one-shot."""

from __future__ import annotations

import torch

from .. import _autograd
from . import kernel


def frequencies(D, sections, *, base=10000.0, per_axis=False, device=None):
    """(inv_freq, axis) for heads of D channels and ``sections[a]`` frequencies on axis a.

    One ladder ``base ** (-2f / D)`` runs over all sections, or, with ``per_axis``, each
    section has its own, ``base ** (-j / sections[a])``."""
    if any(s < 0 for s in sections):
        raise ValueError(f"sections must not be negative, got {list(sections)}")
    P = sum(sections)
    assert 0 < 2 * P <= D, "the sections must hold between 1 and D/2 frequencies"
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(list(sections)))
    if per_axis:
        e = torch.cat([torch.arange(s, dtype=torch.float64) / max(s, 1) for s in sections])
    else:
        e = torch.arange(P, dtype=torch.float64) * 2 / D
    return (float(base) ** -e).float().to(device), axis.int().to(device)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axis, interleaved):
        ctx.save_for_backward(positions, inv_freq, axis)
        ctx.interleaved = interleaved
        return kernel.forward(q, k, positions, inv_freq=inv_freq, axis=axis, interleaved=interleaved)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq, axis = ctx.saved_tensors
        grads = _autograd.first_order(
            "rotary", lambda: kernel.backward(dq, dk, positions, inv_freq=inv_freq, axis=axis,
                                              interleaved=ctx.interleaved), dq, dk)
        return (*grads, None, None, None, None)


def rotary(q, k, positions, *, inv_freq, axis, interleaved=False):
    """q and k (or None) turned by their tokens' positions
    (:mod:`triangleops_b200.rotary.kernel` has the definition); differentiable (once) in q and k."""
    return _Rotary.apply(q, k, positions, inv_freq, axis, interleaved)
