"""The sequence-local token block: what a model runs on its tokens or atoms around the pair trunk.

Each block updates a residual stream s (B, N, C) twice:

    q, k, v, g = n W_in                          n: the norm of s
    o          = window_attn(rotary(q), rotary(k), v)
    s, n       = gated_norm(s, o W_o, g)         post norm, gate, residual scale, add, next norm
    a, b, g    = n W_up
    s, n       = gated_norm(s, (silu(a) b) W_down, g)

so a block is two fused norms, one rotary, one attention and four library products.
:func:`forward` is differentiable in everything and takes whole sequences; :func:`step` takes
one token for each sequence against the keys and values kept in :func:`caches`, and gives what
:func:`forward` with the causal window gives at that token. :func:`forward` fills no caches: a
sequence enters them token by token. No counterpart in the reference.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import gated_norm as _gn
from . import rotary as _rot
from . import window_attn as _wa


def init(C, heads, kv_heads, head_dim, hidden, blocks, *, sections, base=10000.0, per_axis=False, interleaved=False,
         kind="layer", res_scale=1.0, dtype=torch.float32, device=None, generator=None):
    """Weights of ``blocks`` blocks (normal, variance 1 / fan-in) as one dict: ``first`` (the
    first norm's weight and bias), ``blocks`` (a dict each), and the shape of the heads. The
    positions' axes have ``sections`` frequencies each (:func:`rotary.frequencies`)."""

    def lin(out, inp):
        return (torch.randn(out, inp, generator=generator) * inp**-0.5).to(device=device, dtype=dtype)

    def vec(v):
        return torch.full((C,), float(v), dtype=dtype, device=device)

    def bias():
        return vec(0) if kind == "layer" else None

    def norms():
        return dict(post_weight=vec(1), post_bias=bias(), res_scale=vec(res_scale), pre_weight=vec(1), pre_bias=bias())

    qkv = (heads + 2 * kv_heads) * head_dim
    inv_freq, axis = _rot.frequencies(head_dim, sections, base=base, per_axis=per_axis, device=device)
    return {
        "heads": (heads, kv_heads, head_dim), "hidden": hidden, "kind": kind,
        "rotary": dict(inv_freq=inv_freq, axis=axis, interleaved=interleaved),
        "first": dict(weight=vec(1), bias=bias()),
        "blocks": [dict(w_in=lin(qkv + C, C), w_o=lin(C, heads * head_dim), attn=norms(), w_up=lin(2 * hidden + C, C),
                        w_down=lin(C, hidden), mlp=norms()) for _ in range(blocks)],
    }


def weights(pre):
    """The tensors of ``pre`` that a training step updates, in a fixed order."""
    out = [t for t in pre["first"].values() if t is not None]
    for b in pre["blocks"]:
        for t in b.values():
            out += [u for u in t.values() if u is not None] if isinstance(t, dict) else [t]
    return out


def _first_norm(s, pre, eps):
    w, b = pre["first"]["weight"], pre["first"]["bias"]
    if pre["kind"] == "layer":
        return F.layer_norm(s, s.shape[-1:], w, b, eps)
    return F.rms_norm(s, s.shape[-1:], w, eps)


def _project(n, b, pre):
    """q, k, v (..., heads, D) and the gate (..., C): views of one product."""
    hq, hk, D = pre["heads"]
    t = F.linear(n, b["w_in"])
    q, k, v, g = t.split([hq * D, hk * D, hk * D, n.shape[-1]], -1)
    return q.unflatten(-1, (hq, D)), k.unflatten(-1, (hk, D)), v.unflatten(-1, (hk, D)), g


def _transition(s, n, b, pre, eps):
    u, w, g = F.linear(n, b["w_up"]).split([pre["hidden"], pre["hidden"], n.shape[-1]], -1)
    return _gn.gated_norm(s, F.linear(F.silu(u) * w, b["w_down"]), g, kind=pre["kind"], eps=eps, **b["mlp"])


def forward(s, pre, positions, *, window, sinks=0, mask=None, eps=1e-5):
    """s (B, N, C), positions (axes, B, N) -> (s, n): the stream after the blocks and its norm.
    ``window``, ``sinks`` and ``mask`` (B, N) as in :func:`window_attn.window_attention`."""
    n = _first_norm(s, pre, eps)
    for b in pre["blocks"]:
        q, k, v, g = _project(n, b, pre)
        q, k = _rot.rotary(q, k, positions, **pre["rotary"])
        o = _wa.window_attention(q, k, v, window=window, sinks=sinks, mask=mask)
        s, n = _gn.gated_norm(s, F.linear(o.flatten(-2), b["w_o"]), g, kind=pre["kind"], eps=eps, **b["attn"])
        s, n = _transition(s, n, b, pre, eps)
    return s, n


def caches(pre, B, N, *, dtype, device=None):
    """Room for the keys and values of B sequences of up to N tokens, a pair for each block."""
    _, hk, D = pre["heads"]
    return [tuple(torch.empty(B, N, hk, D, dtype=dtype, device=device) for _ in range(2)) for _ in pre["blocks"]]


@torch.no_grad()
def step(s, pre, positions, cache, lengths, *, window, sinks=0, eps=1e-5):
    """One token for each sequence: s (B, C), positions (axes, B); its keys and values go to
    place ``lengths[b]`` (B,) int32 of the caches, which then hold ``lengths + 1`` tokens.
    ``window`` is a number of keys. Returns (s, n), each (B, C). A sequence whose place the caches
    do not have (they are full, or the length is negative) leaves them as they are and gets NaN."""
    x = s.unsqueeze(1)
    n = _first_norm(x, pre, eps)
    N = min((kc.shape[1] for kc, _ in cache), default=2**31 - 1)
    out = ((lengths < 0) | (lengths >= N)).unsqueeze(-1)
    now = lengths + 1
    for b, (kc, vc) in zip(pre["blocks"], cache):
        q, k, v, g = _project(n, b, pre)
        q, k = _rot.rotary(q, k, positions.unsqueeze(-1), **pre["rotary"])
        _wa.kernel.store(k[:, 0], v[:, 0], kc, vc, lengths)
        o = _wa.decode(q[:, 0], kc, vc, now, window=window, sinks=sinks)
        x, n = _gn.gated_norm(x, F.linear(o.flatten(-2), b["w_o"]).unsqueeze(1), g, kind=pre["kind"], eps=eps,
                              **b["attn"])
        x, n = _transition(x, n, b, pre, eps)
    return x[:, 0].masked_fill(out, float("nan")), n[:, 0].masked_fill(out, float("nan"))
