"""Rotary positions with several axes: the launcher over the C-ABI.

Frequency f belongs to one axis of the positions; its pair of channels turns by
``positions[axis[f], b, n] * inv_freq[f]``:

    (a, b) -> (a cos - b sin, a sin + b cos)

Pairs are channels (f, D/2 + f), or (2f, 2f + 1) with ``interleaved``. There are
P <= D/2 frequencies; channels of no pair are copied. Queries and keys go in one launch, an
angle is formed in 64 bits. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib

_P, _I, _I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_lib.register("tops_rotary",
              [_I, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _P])

_I3, _I6 = ctypes.c_int64 * 3, ctypes.c_int64 * 6


def _turn(q, k, positions, inv_freq, axis, interleaved, negate):
    dt = _lib.dtype_code(q.dtype)
    assert q.dim() == 4, "q must be (B, N, H, D)"
    B, N, Hq, D = q.shape
    assert inv_freq.dim() == 1 and positions.dim() == 3, "inv_freq must be (P,) and positions (axes, B, N)"
    P = inv_freq.shape[0]
    A, Bp, Np = positions.shape
    assert 0 < 2 * P <= D, "inv_freq must be (P,) with 0 < 2P <= D"
    assert axis.shape == inv_freq.shape, "axis must be (P,) like inv_freq"
    assert Bp == B and Np == N and A > 0, "positions must be (axes, B, N)"
    if inv_freq.dtype != torch.float32 or axis.dtype != torch.int32:
        raise ValueError(f"inv_freq must be fp32 and axis int32, got {inv_freq.dtype} and {axis.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    Hk = 0
    if k is not None:
        assert k.dim() == 4, "k must be (B, N, Hk, D) like q"
        Bk, Nk, Hk, Dk = k.shape
        assert Bk == B and Nk == N and Dk == D, "k must be (B, N, Hk, D) like q"
        if k.dtype != q.dtype:
            raise ValueError(f"q and k must have one dtype, got {q.dtype} and {k.dtype}")
    dev = q.device
    assert positions.device == inv_freq.device == axis.device == dev and (k is None or k.device == dev), \
        "q, k, positions, inv_freq and axis must be on one device"
    _lib.require_cuda(q)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    if q.stride(3) != 1:
        q = q.contiguous()
    if k is not None and k.stride(3) != 1:
        k = k.contiguous()
    st = _I6(*q.stride()[:3], *(k.stride()[:3] if k is not None else (0, 0, 0)))
    if not (inv_freq.is_contiguous() and axis.is_contiguous()):
        inv_freq, axis = inv_freq.contiguous(), axis.contiguous()
    _lib.launch("tops_rotary", dev, dt, B, N, Hq, Hk, D, P, A, bool(interleaved), negate,
                q.data_ptr(), _lib.ptr(k), st, positions.data_ptr(), positions.dtype == torch.int64,
                _I3(*positions.stride()), inv_freq.data_ptr(), axis.data_ptr(), qo.data_ptr(), _lib.ptr(ko))
    return qo, ko


def forward(q, k, positions, *, inv_freq, axis, interleaved=False):
    """q (B, N, Hq, D) and k (B, N, Hk, D) or None, any strides; positions (axes, B, N) int32
    or int64, any strides; inv_freq (P,) fp32 and axis (P,) int32
    (:func:`~triangleops_b200.rotary.frequencies` makes them) -> (q, k) turned, contiguous."""
    return _turn(q, k, positions, inv_freq, axis, interleaved, False)


def backward(dq, dk, positions, *, inv_freq, axis, interleaved=False):
    """Gradients of q and k from those of the turned ones: the turn by the negated angles."""
    return _turn(dq, dk, positions, inv_freq, axis, interleaved, True)
