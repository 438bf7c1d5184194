"""Windowed attention with sinks: the launchers.

Query i of Nq stands at key position p = i + Nk - Nq (the queries are the last tokens of
the keys) and sees key j where

    j <= p + right  and  (j >= p - left or j < sinks)  and  mask[b, j]

    S = scale q k^T,   P = softmax over the seen keys,   out = P v

``window`` is ``(left, right)``, or an int W for the causal window of the W newest keys,
``(W - 1, 0)``. The first ``sinks`` keys stay visible from any distance to their right.
Several query heads may share a key head (Hq a multiple of Hkv). A query that sees no key
gets zeros, log-sum-exp -inf, and passes no gradient; what masked keys hold (NaN and
infinity too) reaches nothing, nor does what such a query and its gradient hold. A key that is
not masked must be finite, seen or not: in :func:`forward` and :func:`backward` a tile's other
queries multiply it by a probability of zero. (:func:`decode` reads only the keys that are
seen.)

In 16 bits P enters its products rounded once to the IO dtype and dS as two parts of it; in f16
both are held at powers of two of their size there, so that small probabilities and gradients of any
size keep their digits. Sums, maxima and statistics are fp32.

No counterpart in the reference, whose attentions are dense.
"""

from __future__ import annotations

from .. import _lib


def _window(window):
    """(left, right) of a window argument."""
    if isinstance(window, int):
        if window < 1:
            raise ValueError(f"window must be at least 1 key, got {window}")
        return window - 1, 0
    left, right = window
    if left < 0 or right < 0:
        raise ValueError(f"window must be (left, right) with neither negative, got {window}")
    return int(left), int(right)


def forward(q, k, v, *, window, sinks=0, scale=None, mask=None, out=None):
    """q (B, Nq, Hq, D), k and v (B, Nk, Hkv, D), any strides -> (out (B, Nq, Hq, D),
    lse (B, Hq, Nq) fp32, the natural log of each row's sum). ``scale`` defaults to
    1/sqrt(D); ``mask`` (B, Nk) keeps a key where it is nonzero; ``out`` (contiguous)
    receives the result."""
    left, right = _window(window)
    return _lib.bind().window_attn_forward(q, k, v, mask, left, right, sinks, scale, out)


def backward(dout, q, k, v, out, lse, *, window, sinks=0, scale=None, mask=None):
    """Gradients (dq, dk, dv) from that of ``out``; ``out`` and ``lse`` as :func:`forward`
    gave them, the other arguments as it got them. Sums run in a fixed order: the same
    inputs give the same bits."""
    left, right = _window(window)
    return _lib.bind().window_attn_backward(dout, q, k, v, out, lse, mask, left, right, sinks, scale)


def decode(q, k_cache, v_cache, lengths, *, window, sinks=0, scale=None):
    """One token for each sequence: q (B, Hq, D) stands at the last of the ``lengths[b]``
    keys that sequence has in the caches (B, N, Hkv, D), any strides, and sees the
    ``window`` newest of them and the first ``sinks``. ``lengths`` (B,) int32 (or int64, at the cost of two more
    launches) on the device; a length of 0 gives zeros, one beyond N counts as N. Returns (B, Hq, D)."""
    if not isinstance(window, int):
        raise ValueError(f"window must be a number of keys, at least 1, got {window}")
    return _lib.bind().window_attn_decode(q, k_cache, v_cache, lengths, window, sinks, scale)


def store(k, v, k_cache, v_cache, lengths):
    """The keys and values (B, Hkv, D) of one token for each sequence to place ``lengths[b]`` of the
    caches. A sequence whose place the caches do not have (below 0, or N and beyond) writes nothing."""
    _lib.bind().window_attn_store(k, v, k_cache, v_cache, lengths)
