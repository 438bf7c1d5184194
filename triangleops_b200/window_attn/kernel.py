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
    t = _rows(t)
    if t.dtype == torch.float32 or t.shape[-1] % 8 or t.shape[-1] > 128:
        return t
    if t.data_ptr() % 16 or any(n > 1 and (s % 8 or s == 0) for n, s in zip(t.shape[:-1], t.stride())):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(*tensors):
    st = [s for t in tensors for s in t.stride()[:-1]]
    return (ctypes.c_int64 * len(st))(*st)


def _check(q, k, v):
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k and v must be (B, N, H, D)"
    B, Nq, Hq, D = q.shape
    assert k.shape == v.shape and k.shape[0] == B and k.shape[3] == D, "k and v must be (B, Nk, Hkv, D) like q"
    Nk, Hkv = k.shape[1], k.shape[2]
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
    return mask.contiguous().view(torch.uint8)


def forward(q, k, v, *, window, sinks=0, scale=None, mask=None, out=None):
    """q (B, Nq, Hq, D), k and v (B, Nk, Hkv, D), any strides -> (out (B, Nq, Hq, D),
    lse (B, Hq, Nq) fp32, the natural log of each row's sum). ``scale`` defaults to
    1/sqrt(D); ``mask`` (B, Nk) keeps a key where it is nonzero; ``out`` (contiguous)
    receives the result."""
    dt = _lib.dtype_code(q.dtype)
    B, Nq, Nk, Hq, Hkv, D = _check(q, k, v)
    left, right = _window(window)
    _lib.require_cuda(q, k, v)
    m = _mask(mask, B, Nk, q.device)
    q, k, v = _tiles(q), _tiles(k), _tiles(v)
    if out is None:
        out = torch.empty(B, Nq, Hq, D, dtype=q.dtype, device=q.device)
    assert out.shape == (B, Nq, Hq, D) and out.dtype == q.dtype and out.is_contiguous(), "out must be like q, contiguous"
    lse = torch.empty(B, Hq, Nq, dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("tops_window_attn_forward", dt, B, Nq, Nk, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  _strides(q, k, v), _lib.ptr(m), left, right, int(sinks), D ** -0.5 if scale is None else float(scale),
                  out.data_ptr(), lse.data_ptr(), _lib.stream_ptr(q.device))
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
    _lib.require_cuda(q, k, v, dout, out, lse)
    m = _mask(mask, B, Nk, q.device)
    q, k, v, dout = _tiles(q), _tiles(k), _tiles(v), _tiles(dout)
    out, lse = out.contiguous(), lse.contiguous()
    dq = torch.empty(B, Nq, Hq, D, dtype=q.dtype, device=q.device)
    dk = torch.empty(B, Nk, Hkv, D, dtype=q.dtype, device=q.device)
    dv = torch.empty_like(dk)
    need = ctypes.c_int64(0)
    _lib.call("tops_window_attn_backward_workspace_bytes", dt, B, Nq, Nk, Hq, Hkv, D, left, right, int(sinks),
              ctypes.byref(need))
    ws = torch.empty(max(16, need.value), dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("tops_window_attn_backward", dt, B, Nq, Nk, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  _strides(q, k, v), _lib.ptr(m), left, right, int(sinks), D ** -0.5 if scale is None else float(scale),
                  dout.data_ptr(), _strides(dout), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), dq.data_ptr(),
                  dk.data_ptr(), dv.data_ptr(), _lib.stream_ptr(q.device))
    return dq, dk, dv


def decode(q, k_cache, v_cache, lengths, *, window, sinks=0, scale=None):
    """One token for each sequence: q (B, Hq, D) stands at the last of the ``lengths[b]``
    keys that sequence has in the caches (B, N, Hkv, D), any strides, and sees the
    ``window`` newest of them and the first ``sinks``. ``lengths`` (B,) int32 on the
    device; a length of 0 gives zeros, one beyond N counts as N. Returns (B, Hq, D)."""
    dt = _lib.dtype_code(q.dtype)
    assert q.dim() == 3, "q must be (B, Hq, D)"
    B, Hq, D = q.shape
    _check(q.unsqueeze(1), k_cache, v_cache)
    N, Hkv = k_cache.shape[1], k_cache.shape[2]
    assert lengths.shape == (B,) and lengths.device == q.device, "lengths must be (B,) on the device of q"
    if not isinstance(window, int) or window < 1:
        raise ValueError(f"window must be a number of keys, at least 1, got {window}")
    _lib.require_cuda(q, k_cache, v_cache, lengths)
    q, k, v = _rows(q), _rows(k_cache), _rows(v_cache)
    lengths = lengths.to(torch.int32).contiguous()
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    need = ctypes.c_int64(0)
    _lib.call("tops_window_attn_decode_workspace_bytes", B, N, Hq, Hkv, D, window, int(sinks), ctypes.byref(need))
    ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    with torch.cuda.device(q.device):
        _lib.call("tops_window_attn_decode", dt, B, N, Hq, Hkv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  _strides(q, k, v), lengths.data_ptr(), window, int(sinks),
                  D ** -0.5 if scale is None else float(scale), _lib.ptr(ws), out.data_ptr(),
                  _lib.stream_ptr(q.device))
    return out
