"""The norms around a block fused with its gate and residual scale: the launchers over the C-ABI.

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

import ctypes

import torch

from .. import _lib

_P, _I, _I64, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_lib.register("tops_gated_norm_forward",
              [_I, _I, _I64, _I64, _I64, _I, _I, _I, _F, _P, _I64, _P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _P, _P,
               _P])
_lib.register("tops_gated_norm_backward",
              [_I, _I, _I64, _I64, _I64, _I, _I, _I, _P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _P, _P, _P,
               _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P])
_lib.register("tops_gated_norm_backward_workspace_bytes", [_I64, _I64, _I64, _P])

MAX_C = 8192


def _rows(t, C):
    """(tensor, row stride) of (..., C) as rows with contiguous channels and one stride (a copy
    where the tensor has no such view); (None, 0) of None."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, C
    if t.stride(-1) == 1 or C == 1:
        if t.dim() == 2:
            return t, t.stride(0)
        try:
            t = t.view(-1, C)
            return t, t.stride(0)
        except RuntimeError:
            pass
    return t.contiguous(), C


def _check(x, y, gate, weights, kind):
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    dtype, shape, dev = x.dtype, x.shape, x.device
    dt = _lib.dtype_code(dtype)
    assert shape and shape == y.shape, "x and y must have one shape (..., C)"
    C = shape[-1]
    assert 0 < C <= MAX_C, f"C must be in 1..{MAX_C}"
    if y.dtype != dtype or (gate is not None and gate.dtype != dtype):
        raise ValueError(f"x, y and gate must have one dtype, got {dtype}, {y.dtype}"
                         + ("" if gate is None else f", {gate.dtype}"))
    rows = groups = x.numel() // C
    if gate is not None:
        gs = gate.shape
        if gs != shape:
            lead = len(shape) - 1
            assert len(gs) == lead + 1 and gs[lead] == C, "gate must be like x, or with 1 in its last places before C"
            while lead and gs[lead - 1] == 1:
                lead -= 1
            assert gs[:lead] == shape[:lead], "gate must be like x, or with 1 in its last places before C"
            groups = gate.numel() // C
        assert gate.device == dev, "x, y and gate must be on one device"
    assert y.device == dev, "x, y and gate must be on one device"
    w_dt = None
    for w in weights:
        if w is not None:
            assert w.dim() == 1 and w.shape[0] == C and w.device == dev, "a weight must be (C,) on the device of x"
            if w_dt is None:
                w_dt = w.dtype
            if w.dtype != w_dt or (w_dt != dtype and w_dt != torch.float32):
                raise ValueError(f"the weights must all be {dtype} or all fp32, got {w_dt} and {w.dtype}")
    return dt, dt if w_dt is None or w_dt == dtype else _lib.F32, C, rows, groups


def _w(t):
    """Address of a weight; a strided one is replaced by a copy that the caller holds."""
    return None if t is None else t.data_ptr()


def _dense(weights):
    return [w if w is None or w.is_contiguous() else w.contiguous() for w in weights]


def forward(x, y, gate=None, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None, pre_bias=None,
            kind="layer", post_norm=True, pre_norm=True, eps=1e-5):
    """-> (h, n, stats): h and n like x (n None without ``pre_norm``), stats (..., 4) fp32 for
    :func:`backward` (mean and 1/std of y, of h)."""
    w = _dense((post_weight, post_bias, res_scale, pre_weight, pre_bias))
    dt, w_dt, C, rows, groups = _check(x, y, gate, w, kind)
    _lib.require_cuda(x)
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    n = torch.empty_like(h) if pre_norm else None
    stats = x.new_empty((*x.shape[:-1], 4), dtype=torch.float32)
    if rows == 0:
        return h, n, stats
    (x, xs), (y, ys), (gate, gs) = _rows(x, C), _rows(y, C), _rows(gate, C)
    _lib.launch("tops_gated_norm_forward", h.device, dt, w_dt, rows, groups, C, kind == "layer", bool(post_norm),
                bool(pre_norm), eps, x.data_ptr(), xs, y.data_ptr(), ys, _w(gate), gs, _w(w[0]), _w(w[1]), _w(w[2]),
                _w(w[3]), _w(w[4]), h.data_ptr(), _w(n), stats.data_ptr())
    return h, n, stats


def backward(dh, dn, x, y, gate, stats, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None,
             pre_bias=None, kind="layer", post_norm=True, pre_norm=True):
    """Gradients from those of h and n (either may be None: zero), as a dict: ``dx``, ``dy``,
    ``dgate`` (with a gate, in its shape) and ``d<name>`` for each weight given, in its dtype
    (summed over the tokens in fp32, in a fixed order)."""
    w = _dense((post_weight, post_bias, res_scale, pre_weight, pre_bias))
    dt, w_dt, C, rows, groups = _check(x, y, gate, w, kind)
    dev = x.device
    for d in (dh, dn):
        if d is not None:
            assert d.shape == x.shape and d.device == dev, "dh and dn must be like x"
            if d.dtype != x.dtype:
                raise ValueError(f"dh and dn must be {x.dtype}")
    assert stats.shape == (*x.shape[:-1], 4) and stats.dtype == torch.float32 and stats.is_contiguous() \
        and stats.device == dev, "stats must be what forward returned"
    _lib.require_cuda(x)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dy = torch.empty_like(dx)
    dgate = None if gate is None else torch.empty_like(gate, memory_format=torch.contiguous_format)
    dw = [None if t is None else torch.empty_like(t) for t in w]
    if rows == 0:
        for t in (dgate, *dw):
            if t is not None:
                t.zero_()
    else:
        need = ctypes.c_int64(0)
        _lib.call("tops_gated_norm_backward_workspace_bytes", rows, groups, C, ctypes.byref(need))
        ws = x.new_empty(need.value, dtype=torch.uint8)
        (x, xs), (y, ys), (gate, gs), (dh, dhs), (dn, dns) = (_rows(t, C) for t in (x, y, gate, dh, dn))
        _lib.launch("tops_gated_norm_backward", dev, dt, w_dt, rows, groups, C, kind == "layer", bool(post_norm),
                    bool(pre_norm), _w(dh), dhs, _w(dn), dns, x.data_ptr(), xs, y.data_ptr(), ys, _w(gate), gs,
                    stats.data_ptr(), _w(w[0]), _w(w[1]), _w(w[2]), _w(w[3]), dx.data_ptr(), dy.data_ptr(), _w(dgate),
                    *map(_w, dw), ws.data_ptr())
    res = {"dx": dx, "dy": dy}
    if dgate is not None:
        res["dgate"] = dgate
    for name, t in zip(("dpost_weight", "dpost_bias", "dres_scale", "dpre_weight", "dpre_bias"), dw):
        if t is not None:
            res[name] = t
    return res
