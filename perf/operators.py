"""What is measured of the sequence-local token block: windowed attention with sinks, the norms
around a block fused with its gate and residual scale, and rotary positions with several axes.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, where ``own`` is true, through the package's public entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _attn(name, B, N, Hq, Hkv, D, left, right, sinks, mask, dtype, train):
    return {"name": name, "op": "attn", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "left": left, "right": right,
            "sinks": sinks, "mask": mask, "dtype": dtype, "train": train}


def _decode(name, B, N, Hq, Hkv, D, window, sinks, dtype):
    return {"name": name, "op": "decode", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "window": window,
            "sinks": sinks, "dtype": dtype}


def _norm(name, B, N, C, kind, gate, dtype, train):
    return {"name": name, "op": "norm", "B": B, "N": N, "C": C, "kind": kind, "gate": gate, "dtype": dtype,
            "train": train}


def _rotary(name, B, N, Hq, Hkv, D, sections, interleaved, dtype, train):
    return {"name": name, "op": "rotary", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "sections": sections,
            "interleaved": interleaved, "dtype": dtype, "train": train}


def listed():
    return [
        # a training step of the local attention over the 1024 tokens of one structure, the last 64 padded
        _attn("attn-train-1024-h4-d32", 1, 1024, 4, 4, 32, 64, 64, 0, "tail", "bf16", True),
        # reading a long sequence in: causal, four query heads to a key head, the first tokens stay visible
        _attn("attn-prefill-8192-h16-d128", 1, 8192, 16, 4, 128, 1023, 0, 4, "none", "bf16", False),
        # a batch of odd length with tokens missing here and there
        _attn("attn-prefill-1537-h6-d64", 3, 1537, 6, 2, 64, 199, 0, 5, "random", "f16", False),
        # a training step on two long sequences
        _attn("attn-train-4096-h16-d128", 2, 4096, 16, 4, 128, 511, 0, 4, "none", "bf16", True),
        # one token of one sequence: latency
        _decode("decode-1-w1024-d128", 1, 2048, 8, 2, 128, 1024, 4, "bf16"),
        # one token for each of 64 sequences of different lengths
        _decode("decode-64-w4096-d128", 64, 8192, 32, 8, 128, 4096, 4, "bf16"),
        # between two blocks, for the tokens of one serving step: latency
        _norm("norm-step-8x128", 8, 1, 128, "layer", "token", "bf16", False),
        # between two blocks of the pair stack, N = 1024, with gradients
        _norm("norm-pair-1024-c128", 1, 1024 * 1024, 128, "layer", "token", "bf16", True),
        # a single track of odd width, gated by sample, with gradients
        _norm("norm-train-3x1367-c771", 3, 1367, 771, "rms", "sample", "f16", True),
        # positions of one serving step
        _rotary("rotary-step-64x1-h32-d128", 64, 1, 32, 8, 128, "16,24,24", False, "bf16", False),
        # positions of two long sequences on three axes
        _rotary("rotary-2x8192-h32-d128", 2, 8192, 32, 8, 128, "16,24,24", False, "bf16", False),
        # a grid of 37 x 53, two axes on neighbouring channels, part of the head left as it is, with gradients
        _rotary("rotary-grid-3x1961-h6-d96", 3, 1961, 6, 2, 96, "20,20", True, "f16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    hkv = rng.choice([1, 2, 3, 4, 8])
    g = rng.choice([1, 1, 2, 3, 4, 8])
    return min(hkv * g, most // hkv * hkv), hkv


def draw(rng):
    op = rng.choice(["attn", "attn", "decode", "norm", "rotary"])
    dt = rng.choice(["bf16", "f16"])
    if op == "attn":
        hq, hkv = _heads(rng, 16)
        n = _log(rng, 17, 6000)
        b = max(1, min(4, _log(rng, 1, 4), 8192 // n))
        train = rng.random() < 0.5
        left = _log(rng, 1, 512 if train else 1024)
        right = 0 if rng.random() < 0.6 else _log(rng, 1, 128)
        return {k: v for k, v in _attn("", b, n, hq, hkv, rng.choice([32, 64, 128]), left, right,
                                       rng.choice([0, 0, 1, 4, 16, 70]), rng.choice(["none", "tail", "random"]), dt,
                                       train).items() if k != "name"}
    if op == "decode":
        hq, hkv = _heads(rng, 32)
        b = _log(rng, 1, 64)
        return {k: v for k, v in _decode("", b, _log(rng, 1, 8192), hq, hkv, rng.choice([32, 64, 128]),
                                         _log(rng, 1, 4096), rng.choice([0, 1, 4, 16]), dt).items() if k != "name"}
    if op == "norm":
        c = _log(rng, 33, 4100) if rng.random() < 0.4 else 8 * _log(rng, 4, 512)
        t = _log(rng, 1, min(300000, 2 ** 25 // c))
        b = min(t, _log(rng, 1, 8))
        return {k: v for k, v in _norm("", b, max(1, t // b), c, rng.choice(["layer", "rms"]),
                                       rng.choice(["token", "sample", "none"]), rng.choice(["bf16", "f16", "f32"]),
                                       rng.random() < 0.5).items() if k != "name"}
    hq, hkv = _heads(rng, 32)
    d = rng.choice([32, 64, 96, 128])
    n = _log(rng, 1, 8192)
    parts = {1: [d // 2], 2: [d // 4, d // 2 - d // 4], 3: [d // 8, 3 * d // 16, d // 2 - d // 8 - 3 * d // 16]}
    sections = parts[rng.choice([1, 2, 3])]
    if rng.random() < 0.3:
        sections[-1] = max(1, sections[-1] - 3)
    return {k: v for k, v in _rotary("", max(1, min(_log(rng, 1, 64), 8192 // n)), n, hq, hkv, d,
                                     ",".join(map(str, sections)), rng.random() < 0.5, dt, rng.random() < 0.4).items() if k != "name"}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _valid(case):
    """Tokens that a padded sequence has, one number for each of the batch: 64 tokens less each time,
    and from the third on an eighth of the length (so that late queries see no key at all)."""
    n = case["N"]
    return [max(1, n - 64 * (b + 1)) if b < 2 else max(1, n // 8) for b in range(case["B"])]


def _lengths(case):
    """Lengths of the sequences in a cache of N places: full, and shorter down to half."""
    n, b = case["N"], case["B"]
    return [max(1, n - i * n // (2 * b)) for i in range(b)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def r(*shape, sd=1.0, mean=0.0, dtype=dt):
        return torch.empty(*shape, device=dev, dtype=torch.float32).normal_(mean, sd, generator=g).to(dtype)

    s = {"case": case}
    op = case["op"]
    if op in ("attn", "decode", "rotary"):
        B, N, Hq, Hkv, D = (case[k] for k in ("B", "N", "Hq", "Hkv", "D"))
    if op == "attn":
        s.update(q=r(B, N, Hq, D), k=r(B, N, Hkv, D), v=r(B, N, Hkv, D))
        s["mask"] = None
        if case["mask"] == "tail":
            s["mask"] = torch.arange(N, device=dev) < torch.tensor(_valid(case), device=dev)[:, None]
        elif case["mask"] == "random":
            s["mask"] = torch.rand(B, N, device=dev, generator=g) < 0.9
        if case["train"]:
            s["dout"] = r(B, N, Hq, D)
    elif op == "decode":
        s.update(q=r(B, Hq, D), k=r(B, N, Hkv, D), v=r(B, N, Hkv, D),
                 lengths=torch.tensor(_lengths(case), device=dev, dtype=torch.int32))
    elif op == "norm":
        B, N, C = case["B"], case["N"], case["C"]
        s.update(x=r(B, N, C, sd=2.0), y=r(B, N, C, mean=0.1),
                 gate={"token": lambda: r(B, N, C), "sample": lambda: r(B, 1, C), "none": lambda: None}[case["gate"]](),
                 post_weight=r(C, sd=0.1, mean=1.0), post_bias=r(C, sd=0.1) if case["kind"] == "layer" else None,
                 res_scale=r(C, sd=0.1, mean=0.5), pre_weight=r(C, sd=0.1, mean=1.0),
                 pre_bias=r(C, sd=0.1) if case["kind"] == "layer" else None)
        if case["train"]:
            s.update(dh=r(B, N, C), dn=r(B, N, C))
    else:
        sections = [int(v) for v in case["sections"].split(",")]
        s.update(q=r(B, N, Hq, D), k=r(B, N, Hkv, D))
        if case["train"]:
            s.update(dq=r(B, N, Hq, D), dk=r(B, N, Hkv, D))
        s["positions"] = torch.randint(0, 8192, (len(sections), B, N), device=dev, generator=g,
                                       dtype=torch.int32)
        # one ladder of frequencies over the head; each section of it belongs to an axis
        p = sum(sections)
        s["inv_freq"] = (10000.0 ** (-torch.arange(p, dtype=torch.float64) * 2 / D)).float().to(dev)
        s["axis"] = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).int().to(dev)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return {"attn": _run_attn, "decode": _run_decode, "norm": _run_norm, "rotary": _run_rotary}[case["op"]](s, case)


def _visible(nq, nk, left, right, sinks, device):
    i = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None]
    return (j <= i + right) & ((j >= i - left) | (j < sinks))


def _run_attn(s, case):
    q, k, v, mask = s["q"], s["k"], s["v"], s["mask"]
    window, sinks = (case["left"], case["right"]), case["sinks"]
    if own:
        from triangleops_b200 import window_attn

        out, lse = window_attn.forward(q, k, v, window=window, sinks=sinks, mask=mask)
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = window_attn.backward(s["dout"], q, k, v, out, lse, window=window, sinks=sinks, mask=mask)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    g = Hq // Hkv
    scale = D ** -0.5
    qf = q.float().reshape(B, N, Hkv, g, D).permute(0, 2, 3, 1, 4)  # (B, Hkv, g, N, D)
    kf = k.float().permute(0, 2, 1, 3)[:, :, None]  # (B, Hkv, 1, N, D)
    vf = v.float().permute(0, 2, 1, 3)[:, :, None]
    see = _visible(N, N, *window, sinks, q.device)[None, None, None]
    if mask is not None:
        see = see & mask[:, None, None, None, :]
    p = (torch.matmul(qf, kf.transpose(-1, -2)) * scale).masked_fill_(~see, -math.inf)
    p = torch.exp(p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)))
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    o = torch.matmul(p, vf)
    out = o.permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D).to(q.dtype)
    if not case["train"]:
        return {"out": out}
    do = s["dout"].float().reshape(B, N, Hkv, g, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, vf.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2)
    return {"out": out, "dq": dq.permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D).to(q.dtype),
            "dk": dk.transpose(1, 2).to(q.dtype), "dv": dv.transpose(1, 2).to(q.dtype)}


def _run_decode(s, case):
    q, k, v, lengths = s["q"], s["k"], s["v"], s["lengths"]
    if own:
        from triangleops_b200 import window_attn

        return window_attn.decode(q, k, v, lengths, window=case["window"], sinks=case["sinks"])
    B, Hq, D = q.shape
    N, Hkv = k.shape[1], k.shape[2]
    qf = q.float().reshape(B, Hkv, Hq // Hkv, D)
    j = torch.arange(N, device=q.device)[None]
    n = lengths[:, None]
    see = (j < n) & ((j >= n - case["window"]) | (j < case["sinks"]))
    p = torch.matmul(qf, k.float().permute(0, 2, 3, 1)) * D ** -0.5
    p = p.masked_fill_(~see[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p, v.float().transpose(1, 2)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(B, Hq, D).to(q.dtype)


def _stats(t, kind):
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
    return mean, torch.rsqrt((t - mean).square().mean(-1, keepdim=True) + EPS)


def _norm_grad(d, xhat, rstd, w, kind):
    """Gradient of the norm's input, of its weight and of its bias, from that of its output."""
    dxh = d * w
    dx = dxh - xhat * (dxh * xhat).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - dxh.mean(-1, keepdim=True)
    return dx * rstd, (d * xhat).sum((0, 1)), d.sum((0, 1)) if kind == "layer" else None


def _run_norm(s, case):
    kind = case["kind"]
    names = ("post_weight", "post_bias", "res_scale", "pre_weight", "pre_bias")
    if own:
        from triangleops_b200 import gated_norm

        par = {n: s[n] for n in names}
        h, n, stats = gated_norm.forward(s["x"], s["y"], s["gate"], kind=kind, eps=EPS, **par)
        if not case["train"]:
            return {"h": h, "n": n}
        grads = gated_norm.backward(s["dh"], s["dn"], s["x"], s["y"], s["gate"], stats, kind=kind, **par)
        return {"h": h, "n": n, **grads}
    dt = s["x"].dtype
    x, y = s["x"].float(), s["y"].float()
    pw, pb, sc, nw, nb = (None if s[n] is None else s[n].float() for n in names)
    mean, rstd = _stats(y, kind)
    yhat = (y - mean) * rstd
    u = yhat * pw if pb is None else yhat * pw + pb
    sg = None if s["gate"] is None else torch.sigmoid(s["gate"].float())
    gu = u if sg is None else u * sg
    h = x + sc * gu
    hmean, hrstd = _stats(h, kind)
    hhat = (h - hmean) * hrstd
    n = hhat * nw if nb is None else hhat * nw + nb
    res = {"h": h.to(dt), "n": n.to(dt)}
    if not case["train"]:
        return res
    dx, dnw, dnb = _norm_grad(s["dn"].float(), hhat, hrstd, nw, kind)
    dx = dx + s["dh"].float()
    du = dx * sc
    if sg is not None:
        dg = du * u * sg * (1 - sg)
        if case["gate"] == "sample":
            dg = dg.sum(1, keepdim=True)
        res["dgate"] = dg.to(dt)
        du = du * sg
    dy, dpw, dpb = _norm_grad(du, yhat, rstd, pw, kind)
    res.update(dx=dx.to(dt), dy=dy.to(dt), dpost_weight=dpw.to(dt), dres_scale=(dx * gu).sum((0, 1)).to(dt),
               dpre_weight=dnw.to(dt))
    if kind == "layer":
        res.update(dpost_bias=dpb.to(dt), dpre_bias=dnb.to(dt))
    return res


def _turn(t, cos, sin, interleaved, dt):
    p = cos.shape[-1]
    half = t.shape[-1] // 2
    tf = t.float()
    out = tf.clone()
    if interleaved:
        a, b = tf[..., 0:2 * p:2], tf[..., 1:2 * p:2]
        out[..., 0:2 * p:2] = a * cos - b * sin
        out[..., 1:2 * p:2] = a * sin + b * cos
    else:
        a, b = tf[..., :p], tf[..., half:half + p]
        out[..., :p] = a * cos - b * sin
        out[..., half:half + p] = a * sin + b * cos
    return out.to(dt)


def _run_rotary(s, case):
    if own:
        from triangleops_b200 import rotary

        tab = dict(inv_freq=s["inv_freq"], axis=s["axis"], interleaved=case["interleaved"])
        qr, kr = rotary.forward(s["q"], s["k"], s["positions"], **tab)
        if not case["train"]:
            return {"q": qr, "k": kr}
        dq, dk = rotary.backward(s["dq"], s["dk"], s["positions"], **tab)
        return {"q": qr, "k": kr, "dq": dq, "dk": dk}
    pos = s["positions"].float()[s["axis"].long()].permute(1, 2, 0)  # (B, N, P)
    ang = (pos * s["inv_freq"])[:, :, None]
    cos, sin, il, dt = torch.cos(ang), torch.sin(ang), case["interleaved"], s["q"].dtype
    res = {"q": _turn(s["q"], cos, sin, il, dt), "k": _turn(s["k"], cos, sin, il, dt)}
    if case["train"]:
        res.update(dq=_turn(s["dq"], cos, -sin, il, dt), dk=_turn(s["dk"], cos, -sin, il, dt))
    return res


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _pairs(n, left, right, sinks, valid):
    """Visible (query, key) pairs of n queries over the first `valid` of n keys."""
    i = torch.arange(n)
    hi = torch.minimum(i + right, torch.tensor(valid - 1))
    lo = (i - left).clamp(min=0)
    own_ = (hi - lo + 1).clamp(min=0)
    early = (torch.minimum(torch.minimum(lo, hi + 1), torch.tensor(sinks))).clamp(min=0)
    return int((own_ + early).sum())


def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "f32" else 2
    if op == "attn":
        B, N, Hq, Hkv, D = (case[k] for k in ("B", "N", "Hq", "Hkv", "D"))
        valid = _valid(case) if case["mask"] == "tail" else [N] * B
        pairs = sum(_pairs(N, case["left"], case["right"], case["sinks"], m) for m in valid)
        pairs *= 0.9 if case["mask"] == "random" else 1
        q, kv = B * N * Hq * D * e, B * N * Hkv * D * e
        # forward: q k^T and p v. With gradients also do v^T, p^T do, ds k and ds^T q
        return {"bytes": (2 * q + 2 * kv) if not case["train"] else (4 * q + 4 * kv),
                "flops": pairs * Hq * D * (12 if case["train"] else 4)}
    if op == "decode":
        B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
        keys = 0
        for n in _lengths(case):
            lo = max(0, n - case["window"])
            keys += n - lo + min(lo, case["sinks"])
        return {"bytes": keys * Hkv * D * 2 * e + 2 * B * Hq * D * e, "flops": 4 * keys * Hq * D}
    if op == "norm":
        T, C = case["B"] * case["N"], case["C"]
        gate = {"token": T, "sample": case["B"], "none": 0}[case["gate"]] * C
        one = T * C
        if not case["train"]:
            return {"bytes": (4 * one + gate) * e, "flops": 20 * one}
        # read x, y, the gate, dh and dn; write h, n, dx, dy and the gate's gradient
        return {"bytes": (8 * one + 2 * gate) * e, "flops": 60 * one}
    one = case["B"] * case["N"] * (case["Hq"] + case["Hkv"]) * case["D"]
    n = 2 if case["train"] else 1
    return {"bytes": n * 2 * one * e + case["B"] * case["N"] * 4 * len(case["sections"].split(",")),
            "flops": n * 3 * one}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "decode": _exact_decode, "norm": _exact_norm,
            "rotary": _exact_rotary}[case["op"]](s, case)


def _softmax_rows(z, see):
    """Softmax over the seen entries of each row; a row that sees none is zero."""
    z = torch.where(see, z, torch.full_like(z, -math.inf))
    top = z.max(-1, keepdim=True).values
    w = torch.where(see, torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(z))
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, w / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(w))


def _exact_attn(s, case):
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    B, N, Hq, D = q.shape
    g = Hq // case["Hkv"]
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = torch.arange(N, device=q.device)
    gap = at[:, None] - at[None]  # query minus key
    band = (gap >= -case["right"]) & ((gap <= case["left"]) | (at[None] < case["sinks"]))
    for b in range(B):
        see = band if s["mask"] is None else band & s["mask"][b][None]
        for h in range(Hq):
            kv = h // g
            w = _softmax_rows(q[b, :, h] @ k[b, :, kv].T / math.sqrt(D), see)
            out[b, :, h] = w @ v[b, :, kv]
            if case["train"]:
                d = s["dout"][b, :, h].double()
                dw = d @ v[b, :, kv].T
                dz = w * (dw - (w * dw).sum(-1, keepdim=True)) / math.sqrt(D)
                dv[b, :, kv] += w.T @ d
                dk[b, :, kv] += dz.T @ q[b, :, h]
                dq[b, :, h] = dz @ k[b, :, kv]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"out": out}


def _exact_decode(s, case):
    q = s["q"].double()
    B, Hq, D = q.shape
    g = Hq // case["Hkv"]
    out = torch.zeros_like(q)
    for b, n in enumerate(_lengths(case)):
        keep = sorted(set(range(min(n, case["sinks"]))) | set(range(max(0, n - case["window"]), n)))
        keep = torch.tensor(keep, device=q.device, dtype=torch.long)
        kk, vv = s["k"][b, keep].double(), s["v"][b, keep].double()
        for h in range(case["Hkv"]):
            w = torch.softmax(q[b, h * g:(h + 1) * g] @ kk[:, h].T / math.sqrt(D), -1)
            out[b, h * g:(h + 1) * g] = w @ vv[:, h]
    return out


def _exact_norm(s, case):
    """The gradients by reverse differentiation of the definition, a block of tokens at a time."""
    layer = case["kind"] == "layer"
    names = [n for n in ("post_weight", "post_bias", "res_scale", "pre_weight", "pre_bias") if s[n] is not None]
    par = {n: s[n].double().requires_grad_(case["train"]) for n in names}
    B, N, C = s["x"].shape
    step = max(1, 2 ** 24 // C)
    outs = {k: [[] for _ in range(B)] for k in ("h", "n", "dx", "dy", "dgate")}
    total = {n: torch.zeros(C, dtype=torch.float64, device=s["x"].device) for n in names}

    def norm(t, w, b):
        t = t - t.mean(-1, keepdim=True) if layer else t
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w
        return t if b is None else t + b

    for b in range(B):
        for i in range(0, N, step):
            cut = {k: s[k][b, i:i + step].double().requires_grad_(case["train"]) for k in ("x", "y")}
            r = norm(cut["y"], par["post_weight"], par.get("post_bias"))
            if s["gate"] is not None:
                gate = s["gate"][b] if case["gate"] == "sample" else s["gate"][b, i:i + step]
                cut["gate"] = gate.double().requires_grad_(case["train"])
                r = r / (1 + torch.exp(-cut["gate"]))
            h = cut["x"] + par["res_scale"] * r
            n = norm(h, par["pre_weight"], par.get("pre_bias"))
            outs["h"][b].append(h.detach())
            outs["n"][b].append(n.detach())
            if case["train"]:
                got = torch.autograd.grad((h, n), [*cut.values(), *par.values()],
                                          (s["dh"][b, i:i + step].double(), s["dn"][b, i:i + step].double()))
                for k, t in zip(cut, got):
                    outs["d" + k][b].append(t)
                for k, t in zip(names, got[len(cut):]):
                    total[k] += t
    res = {k: torch.stack([torch.cat(t) for t in outs[k]]) for k in ("h", "n")}
    if case["train"]:
        res.update({k: torch.stack([torch.cat(t) for t in outs[k]]) for k in ("dx", "dy")})
        if case["gate"] == "token":
            res["dgate"] = torch.stack([torch.cat(t) for t in outs["dgate"]])
        elif case["gate"] == "sample":
            res["dgate"] = torch.stack([sum(t) for t in outs["dgate"]])
        res.update({"d" + k: t for k, t in total.items()})
    return res


def _exact_rotary(s, case):
    """Each pair of channels is a complex number, turned by its angle."""
    p = s["inv_freq"].shape[0]
    D = case["D"]
    ang = torch.stack([s["positions"][int(a)].double() * float(f) for a, f in zip(s["axis"], s["inv_freq"])], -1)
    first = torch.arange(p, device=ang.device) * 2 if case["interleaved"] else torch.arange(p, device=ang.device)
    second = first + 1 if case["interleaved"] else first + D // 2

    def turn(t, sign):
        t = t.double().clone()
        z = torch.complex(t[..., first], t[..., second]) * torch.polar(torch.ones_like(ang), sign * ang)[:, :, None]
        t[..., first], t[..., second] = z.real, z.imag
        return t

    res = {"q": turn(s["q"], 1), "k": turn(s["k"], 1)}
    if case["train"]:
        res.update(dq=turn(s["dq"], -1), dk=turn(s["dk"], -1))
    return res
