"""Windowed attention with sinks: the launchers over the C-ABI.

Query i of Nq stands at key position p = i + Nk - Nq (the queries are the last tokens of
the keys) and sees key j where

    j <= p + right  and  (j >= p - left or j < sinks)  and  mask[b, j]

    S = scale q k^T,   P = softmax over the seen keys,   out = P v

``window`` is ``(left, right)``, or an int W for the causal window of the W newest keys,
``(W - 1, 0)``. The first ``sinks`` keys stay visible from any distance to their right.
Several query heads may share a key head (Hq a multiple of Hkv). A query that sees no key
gets zeros, log-sum-exp -inf, and passes no gradient; what masked keys hold (NaN and
infinity too) reaches nothing.

No counterpart in the reference, whose attentions are dense.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib

_P, _I, _I64, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_lib.register("tops_window_attn_forward",
              [_I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64, _I64, _I64, _F, _P, _P, _P])
_lib.register("tops_window_attn_backward",
              [_I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64, _I64, _I64, _F, _P, _P, _P, _P, _P,
               _P, _P, _P, _P])
_lib.register("tops_window_attn_backward_workspace_bytes",
              [_I, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _P])
_lib.register("tops_window_attn_decode",
              [_I, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64, _I64, _F, _P, _P, _P])
_lib.register("tops_window_attn_decode_workspace_bytes", [_I64, _I64, _I64, _I64, _I64, _I64, _I64, _P])


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


def _rows(t):
    """The tensor with contiguous channels (a copy where it has none)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tiles(t):
    """As :func:`_rows`, and where the tensor cores take the type and head size, with rows that
    their loads can follow: 16-byte aligned, none repeated by a stride of zero (one copy costs
    far less than the CUDA-core path that takes such rows as they are)."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    t = _rows(t)
    if t.dtype == torch.float32 or t.shape[-1] % 8 or t.shape[-1] > 128:
        return t
    if t.data_ptr() % 16 or any(n > 1 and (s % 8 or s == 0) for n, s in zip(t.shape[:-1], t.stride())):
        return t.clone(memory_format=torch.contiguous_format)
    return t


_I3, _I8, _I9 = ctypes.c_int64 * 3, ctypes.c_int64 * 8, ctypes.c_int64 * 9


def _strides(q, k, v):
    return _I9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])


def _check(q, k, v):
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k and v must be (B, N, H, D)"
    B, Nq, Hq, D = q.shape
    Bk, Nk, Hkv, Dk = k.shape
    assert k.shape == v.shape and Bk == B and Dk == D, "k and v must be (B, Nk, Hkv, D) like q"
    assert Hkv > 0 and Hq % Hkv == 0, "the query heads must be a multiple of the key heads"
    assert Nk >= Nq, "the queries are the last Nq of the Nk tokens"
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    assert q.device == k.device == v.device, "q, k and v must be on one device"
    return B, Nq, Nk, Hq, Hkv, D


def _mask(mask, B, Nk, device):
    if mask is None:
        return None
    assert mask.shape == (B, Nk), "mask must be (B, Nk)"
    assert mask.device == device, "mask must be on the device of q"
    if mask.dtype != torch.bool:
        mask = mask != 0
    return mask.contiguous()


def forward(q, k, v, *, window, sinks=0, scale=None, mask=None, out=None):
    """q (B, Nq, Hq, D), k and v (B, Nk, Hkv, D), any strides -> (out (B, Nq, Hq, D),
    lse (B, Hq, Nq) fp32, the natural log of each row's sum). ``scale`` defaults to
    1/sqrt(D); ``mask`` (B, Nk) keeps a key where it is nonzero; ``out`` (contiguous)
    receives the result."""
    dt = _lib.dtype_code(q.dtype)
    B, Nq, Nk, Hq, Hkv, D = _check(q, k, v)
    left, right = _window(window)
    dev = q.device
    _lib.require_cuda(q)
    m = _mask(mask, B, Nk, dev)
    q, k, v = _tiles(q), _tiles(k), _tiles(v)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        assert out.shape == (B, Nq, Hq, D) and out.dtype == q.dtype and out.is_contiguous() and out.device == dev, \
            "out must be like q, contiguous"
    lse = q.new_empty((B, Hq, Nq), dtype=torch.float32)
    _lib.launch("tops_window_attn_forward", dev, dt, B, Nq, Nk, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                _strides(q, k, v), None if m is None else m.data_ptr(), left, right, int(sinks),
                D ** -0.5 if scale is None else float(scale), out.data_ptr(), lse.data_ptr())
    return out, lse


def backward(dout, q, k, v, out, lse, *, window, sinks=0, scale=None, mask=None):
    """Gradients (dq, dk, dv) from that of ``out``; ``out`` and ``lse`` as :func:`forward`
    gave them, the other arguments as it got them. Sums run in a fixed order: the same
    inputs give the same bits."""
    dt = _lib.dtype_code(q.dtype)
    B, Nq, Nk, Hq, Hkv, D = _check(q, k, v)
    left, right = _window(window)
    assert dout.shape == q.shape and out.shape == q.shape, "dout and out must be like q"
    assert lse.shape == (B, Hq, Nq) and lse.dtype == torch.float32, "lse must be (B, Hq, Nq) fp32"
    if dout.dtype != q.dtype or out.dtype != q.dtype:
        raise ValueError(f"dout and out must be {q.dtype}")
    dev = q.device
    assert dout.device == out.device == lse.device == dev, "dout, out and lse must be on the device of q"
    _lib.require_cuda(q)
    m = _mask(mask, B, Nk, dev)
    q, k, v, dout = _tiles(q), _tiles(k), _tiles(v), _tiles(dout)
    out, lse = out.contiguous(), lse.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dv = torch.empty_like(dk)
    need = ctypes.c_int64(0)
    _lib.call("tops_window_attn_backward_workspace_bytes", dt, B, Nq, Nk, Hq, Hkv, D, left, right, int(sinks),
              ctypes.byref(need))
    ws = q.new_empty(max(16, need.value), dtype=torch.uint8)
    _lib.launch("tops_window_attn_backward", dev, dt, B, Nq, Nk, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                _strides(q, k, v), None if m is None else m.data_ptr(), left, right, int(sinks),
                D ** -0.5 if scale is None else float(scale), dout.data_ptr(), _I3(*dout.stride()[:3]),
                out.data_ptr(), lse.data_ptr(), ws.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    return dq, dk, dv


def decode(q, k_cache, v_cache, lengths, *, window, sinks=0, scale=None):
    """One token for each sequence: q (B, Hq, D) stands at the last of the ``lengths[b]``
    keys that sequence has in the caches (B, N, Hkv, D), any strides, and sees the
    ``window`` newest of them and the first ``sinks``. ``lengths`` (B,) int32 on the
    device; a length of 0 gives zeros, one beyond N counts as N. Returns (B, Hq, D)."""
    dt = _lib.dtype_code(q.dtype)
    assert q.dim() == 3, "q must be (B, Hq, D)"
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "the caches must be (B, N, Hkv, D)"
    B, Hq, D = q.shape
    Bk, N, Hkv, Dk = k_cache.shape
    assert Bk == B and Dk == D, "the caches must be (B, N, Hkv, D) like q"
    assert Hkv > 0 and Hq % Hkv == 0, "the query heads must be a multiple of the key heads"
    if not (q.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError(f"q and the caches must have one dtype, got {q.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    dev = q.device
    assert k_cache.device == v_cache.device == lengths.device == dev, "q, the caches and lengths must be on one device"
    assert lengths.shape == (B,), "lengths must be (B,)"
    if not isinstance(window, int) or window < 1:
        raise ValueError(f"window must be a number of keys, at least 1, got {window}")
    _lib.require_cuda(q)
    sinks = int(sinks)
    q, k, v = _rows(q), _rows(k_cache), _rows(v_cache)
    if lengths.dtype != torch.int32 or not lengths.is_contiguous():
        lengths = lengths.to(torch.int32).contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    need = ctypes.c_int64(0)
    _lib.call("tops_window_attn_decode_workspace_bytes", B, N, Hq, Hkv, D, window, sinks, ctypes.byref(need))
    ws = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _lib.launch("tops_window_attn_decode", dev, dt, B, N, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                _I8(*q.stride()[:2], *k.stride()[:3], *v.stride()[:3]), lengths.data_ptr(), window, sinks,
                D ** -0.5 if scale is None else float(scale), None if ws is None else ws.data_ptr(), out.data_ptr())
    return out
