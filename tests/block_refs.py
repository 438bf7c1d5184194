"""The token block's operators in 64 bits, with the size of what rounding may do to each result.

A bound follows a kernel's roundings: half an ulp of the IO dtype for the final store (2^-25 where
an f16 is subnormal), ``u`` for the rounding of P and dS where they enter a 16-bit product; ``acc`` stands for the fp32 sums and
exponentials (2^-12 where a product is 16-bit: an exponential by a short polynomial is below
2^-13; 4 (terms) 2^-24 + 2^-17 in fp32)."""
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def store(value, dtype):
    """Half an ulp of the IO dtype at each value."""
    return (U[dtype] * value.abs()).clamp_min(2.0**-25 if dtype == torch.float16 else 2.0**-149)


def visible(Nq, Nk, left, right, sinks, mask=None, device=None):
    p = torch.arange(Nq, device=device)[:, None] + (Nk - Nq)
    j = torch.arange(Nk, device=device)[None]
    see = (j <= p + right) & ((j >= p - left) | (j < sinks))
    see = see[None, None]
    return see if mask is None else see & (mask != 0)[:, None, None]


def attention(q, k, v, window, sinks, mask=None, scale=None, dout=None):
    """{name: (value, bound)} of out, lse and, with dout, dq, dk, dv; 64 bits, any masked values."""
    dt, D = q.dtype, q.shape[3]
    u, low = U[dt], dt != torch.float32
    left, right = (window - 1, 0) if isinstance(window, int) else window
    scale = D**-0.5 if scale is None else scale
    B, Nq, Hq, _ = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    g = Hq // Hkv
    see = visible(Nq, Nk, left, right, sinks, mask, q.device).expand(B, Hq, Nq, Nk)
    up = lambda t: t.double().permute(0, 2, 1, 3)  # noqa: E731
    qd, kd, vd = up(q), up(k), up(v)
    if mask is not None:  # what masked keys hold takes no part
        gone = (mask == 0)[:, None, :, None]
        kd, vd = kd.masked_fill(gone, 0.0), vd.masked_fill(gone, 0.0)
    kd, vd = kd.repeat_interleave(g, 1), vd.repeat_interleave(g, 1)
    z = (qd @ kd.mT * scale).masked_fill(~see, -torch.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, 0.0, top)
    w = torch.exp(z - top)
    total = w.sum(-1, keepdim=True)
    P = w / torch.where(total > 0, total, 1.0)
    O = P @ vd
    acc = 2.0**-12 if low else 4 * (D + Nk) * 2.0**-24 + 2.0**-17
    uP = u if low else 0.0
    spread = P @ vd.abs()
    o_err = store(O, dt) + (uP + acc) * spread
    down = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    res = {"out": (down(O), down(o_err)), "lse": ((top + torch.log(total))[..., 0], None)}
    if dout is None:
        return res
    d = up(dout)
    dP = d @ vd.mT
    delta = (d * O).sum(-1, keepdim=True)
    dS = P * (dP - delta) * scale
    # delta comes from the stored out; P and dP carry the fp32 errors
    d_delta = (d.abs() * o_err).sum(-1, keepdim=True)
    ds_err = P * scale * (d_delta + acc * (d.abs() @ vd.abs().mT + delta.abs()) + acc * (dP - delta).abs()) + uP * dS.abs()
    per = lambda t: t.reshape(B, Hkv, g, Nk, D).sum(2)  # noqa: E731
    both = {"dq": (dS @ kd, (ds_err + acc * dS.abs()) @ kd.abs()),
            "dk": (per(dS.mT @ qd), per((ds_err + acc * dS.abs()).mT @ qd.abs())),
            "dv": (per(P.mT @ d), per(((uP + acc) * P).mT @ d.abs()))}
    res.update({n: (down(t), down(store(t, dt) + e)) for n, (t, e) in both.items()})
    return res


def assert_within(got, value, bound, what):
    """|got - value| <= bound element by element (1 % for the bound's own second-order terms)."""
    got = got.detach().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - value).abs() - (1.01 * bound + 1e-30)
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} over its bound (largest error {(got - value).abs().max().item():.3e})"


def gated_norm(x, y, gate, par, kind, eps, post_norm=True, pre_norm=True, dh=None, dn=None):
    """{name: value} of h, n and the gradients, by reverse differentiation in 64 bits, and
    {name: sum of the sizes of the terms} for the weights' gradients."""
    leaf = {"x": x, "y": y, "gate": gate, **par}
    leaf = {k: t.detach().double().requires_grad_() for k, t in leaf.items() if t is not None}

    def norm(t, w, b):
        t = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
        t = t if w is None else t * w
        return t if b is None else t + b

    get = leaf.get
    u = norm(get("y"), get("post_weight"), get("post_bias")) if post_norm else get("y")
    r = u if gate is None else u * torch.sigmoid(get("gate"))
    h = get("x") + (r if get("res_scale") is None else r * get("res_scale"))
    n = norm(h, get("pre_weight"), get("pre_bias")) if pre_norm else None
    res = {"h": h.detach()}
    if pre_norm:
        res["n"] = n.detach()
    if dh is None and dn is None:
        return res
    loss = 0 * h.sum()
    if dh is not None:
        loss = loss + (h * dh.double()).sum()
    if dn is not None and pre_norm:
        loss = loss + (n * dn.double()).sum()
    grads = torch.autograd.grad(loss, list(leaf.values()), allow_unused=True)
    res.update({"d" + k: torch.zeros_like(t) if gr is None else gr for (k, t), gr in zip(leaf.items(), grads)})
    return res


def rotary(t, positions, inv_freq, axis, interleaved, sign=1.0):
    P, D = inv_freq.numel(), t.shape[-1]
    t = t.double().clone()
    ang = positions[axis.long()].double().permute(1, 2, 0) * inv_freq.double()
    f = torch.arange(P, device=t.device)
    a, b = (2 * f, 2 * f + 1) if interleaved else (f, f + D // 2)
    c, s = torch.cos(ang)[:, :, None], sign * torch.sin(ang)[:, :, None]
    ta, tb = t[..., a].clone(), t[..., b].clone()
    size = t.abs()
    t[..., a], t[..., b] = ta * c - tb * s, ta * s + tb * c
    size[..., a] = size[..., b] = ta.abs() + tb.abs()
    return t, size
