"""Rotary positions with several axes: the launcher.

Frequency f belongs to one axis of the positions; its pair of channels turns by
``positions[axis[f], b, n] * inv_freq[f]``:

    (a, b) -> (a cos - b sin, a sin + b cos)

Pairs are channels (f, D/2 + f), or (2f, 2f + 1) with ``interleaved``. There are
P <= D/2 frequencies; channels of no pair are copied. (A partial turn that pairs f with P + f within
the first 2P channels is another form: turn ``q[..., :2 * P]``, a strided view, as heads of 2P.) Queries and keys go in one launch, an
angle is formed in 64 bits. No counterpart in the reference.
"""

from __future__ import annotations

from .. import _lib


def forward(q, k, positions, *, inv_freq, axis, interleaved=False):
    """q (B, N, Hq, D) and k (B, N, Hk, D) or None, any strides; positions (axes, B, N) int32
    or int64, any strides; inv_freq (P,) fp32 and axis (P,) int32
    (:func:`~triangleops_b200.rotary.frequencies` makes them) -> (q, k) turned, contiguous."""
    return _lib.bind().rotary(q, k, positions, inv_freq, axis, interleaved, False)


def backward(dq, dk, positions, *, inv_freq, axis, interleaved=False):
    """Gradients of q and k from those of the turned ones: the turn by the negated angles."""
    return _lib.bind().rotary(dq, dk, positions, inv_freq, axis, interleaved, True)
