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
    """(rows, C) view of (..., C) with contiguous channels and one row stride (a copy where
    the tensor has no such view)."""
    if t is None:
        return None
    if t.is_contiguous():
        return t
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    if t.shape[-1] == 1 or t.stride(-1) == 1:
        try:
            return t.view(-1, C)
        except RuntimeError:
            pass
    return t.contiguous()


def _pitch(t, C):
    """Row stride of what :func:`_rows` gave."""
    return 0 if t is None else C if t.is_contiguous() else t.stride(0)


def _check(x, y, gate, weights, kind):
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    dt = _lib.dtype_code(x.dtype)
    assert x.dim() >= 1 and x.shape == y.shape, "x and y must have one shape (..., C)"
    C = x.shape[-1]
    assert 0 < C <= MAX_C, f"C must be in 1..{MAX_C}"
    if y.dtype != x.dtype or (gate is not None and gate.dtype != x.dtype):
        raise ValueError(f"x, y and gate must have one dtype, got {x.dtype}, {y.dtype}"
                         + ("" if gate is None else f", {gate.dtype}"))
    rows = x.numel() // C
    groups = rows
    if gate is not None:
        assert gate.dim() == x.dim() and gate.shape[-1] == C, "gate must be like x, or with 1 in its last places before C"
        lead = x.dim() - 1
        while lead and gate.shape[lead - 1] == 1:
            lead -= 1
        assert gate.shape[:lead] == x.shape[:lead], "gate must be like x, or with 1 in its last places before C"
        groups = gate.numel() // C
    wt = {w.dtype for w in weights if w is not None}
    if len(wt) > 1 or not wt <= {x.dtype, torch.float32}:
        raise ValueError(f"the weights must all be {x.dtype} or all fp32, got {sorted(map(str, wt))}")
    dev = x.device
    for w in weights:
        assert w is None or (w.shape == (C,) and w.device == dev), "a weight must be (C,) on the device of x"
    assert y.device == dev and (gate is None or gate.device == dev), "x, y and gate must be on one device"
    w_dt = _lib.dtype_code(wt.pop()) if wt else dt
    return dt, w_dt, C, rows, groups


def _w(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def forward(x, y, gate=None, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None, pre_bias=None,
            kind="layer", post_norm=True, pre_norm=True, eps=1e-5):
    """-> (h, n, stats): h and n like x (n None without ``pre_norm``), stats (..., 4) fp32 for
    :func:`backward` (mean and 1/std of y, of h)."""
    weights = [_w(w) for w in (post_weight, post_bias, res_scale, pre_weight, pre_bias)]
    dt, w_dt, C, rows, groups = _check(x, y, gate, weights, kind)
    _lib.require_cuda(x)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = torch.empty_like(h) if pre_norm else None
    stats = torch.empty((*x.shape[:-1], 4), dtype=torch.float32, device=x.device)
    if rows == 0:
        return h, n, stats
    x2, y2, g2 = _rows(x, C), _rows(y, C), _rows(gate, C)
    ptr = _lib.ptr
    _lib.launch("tops_gated_norm_forward", x.device, dt, w_dt, rows, groups, C, kind == "layer", bool(post_norm),
                bool(pre_norm), float(eps), x2.data_ptr(), _pitch(x2, C), y2.data_ptr(), _pitch(y2, C), ptr(g2),
                _pitch(g2, C), *map(ptr, weights), h.data_ptr(), ptr(n), stats.data_ptr())
    return h, n, stats


def backward(dh, dn, x, y, gate, stats, *, post_weight=None, post_bias=None, res_scale=None, pre_weight=None,
             pre_bias=None, kind="layer", post_norm=True, pre_norm=True):
    """Gradients from those of h and n (either may be None: zero), as a dict: ``dx``, ``dy``,
    ``dgate`` (with a gate, in its shape) and ``d<name>`` for each weight given, in its dtype
    (summed over the tokens in fp32, in a fixed order)."""
    named = dict(post_weight=post_weight, post_bias=post_bias, res_scale=res_scale, pre_weight=pre_weight,
                 pre_bias=pre_bias)
    weights = [_w(w) for w in named.values()]
    dt, w_dt, C, rows, groups = _check(x, y, gate, weights, kind)
    for d in (dh, dn):
        assert d is None or d.shape == x.shape, "dh and dn must be like x"
        assert d is None or d.device == x.device, "dh and dn must be on the device of x"
        if d is not None and d.dtype != x.dtype:
            raise ValueError(f"dh and dn must be {x.dtype}")
    assert stats.shape == (*x.shape[:-1], 4) and stats.dtype == torch.float32 and stats.is_contiguous(), \
        "stats must be what forward returned"
    assert stats.device == x.device, "stats must be on the device of x"
    _lib.require_cuda(x)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    res = {"dx": dx, "dy": torch.empty_like(dx)}
    if gate is not None:
        res["dgate"] = torch.empty(gate.shape, dtype=x.dtype, device=x.device)
    dw = [None if w is None else torch.empty_like(w) for w in weights]
    if rows == 0:
        for w in dw:
            if w is not None:
                w.zero_()
        if gate is not None:
            res["dgate"].zero_()
    else:
        need = ctypes.c_int64(0)
        _lib.call("tops_gated_norm_backward_workspace_bytes", rows, groups, C, ctypes.byref(need))
        ws = torch.empty(need.value, dtype=torch.uint8, device=x.device)
        x2, y2, g2, dh2, dn2 = (_rows(t, C) for t in (x, y, gate, dh, dn))
        ptr = _lib.ptr
        _lib.launch("tops_gated_norm_backward", x.device, dt, w_dt, rows, groups, C, kind == "layer", bool(post_norm),
                    bool(pre_norm), ptr(dh2), _pitch(dh2, C), ptr(dn2), _pitch(dn2, C), x2.data_ptr(), _pitch(x2, C),
                    y2.data_ptr(), _pitch(y2, C), ptr(g2), _pitch(g2, C), stats.data_ptr(), *map(ptr, weights[:4]),
                    dx.data_ptr(), res["dy"].data_ptr(), ptr(res.get("dgate")), *map(ptr, dw), ws.data_ptr())
    res.update({"d" + k: w for k, w in zip(named, dw) if w is not None})
    return res
