"""The norms around a block, its gate and residual scale, against the definition in 64 bits."""
import pytest
import torch

import block_refs as ref
from triangleops_b200 import gated_norm

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
WEIGHTS = ("post_weight", "post_bias", "res_scale", "pre_weight", "pre_bias")


def _inputs(device, dtype, shape, gate, weights=WEIGHTS, w_dtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, sd=1.0, mean=0.0: torch.randn(*s, generator=g) * sd + mean  # noqa: E731
    C = shape[-1]
    x, y = r(*shape, sd=2.0).to(device, dtype), r(*shape, mean=0.3).to(device, dtype)
    gt = None if gate is None else r(*gate).to(device, dtype)
    par = {n: (r(C, sd=0.2, mean=0.0 if n.endswith("bias") else 1.0).to(device, w_dtype or dtype) if n in weights else None)
           for n in WEIGHTS}
    return x, y, gt, par, r(*shape).to(device, dtype), r(*shape).to(device, dtype)


def _check(device, dtype, shape, gate, kind="layer", weights=WEIGHTS, w_dtype=None, post=True, pre=True, dh=True, dn=True,
           eps=1e-5, seed=0):
    x, y, gt, par, gh, gn = _inputs(device, dtype, shape, gate, weights, w_dtype, seed)
    gh, gn = gh if dh else None, gn if dn else None
    kw = dict(kind=kind, post_norm=post, pre_norm=pre)
    want = ref.gated_norm(x, y, gt, par, kind, eps, post, pre, gh, gn)
    h, n, stats = gated_norm.forward(x, y, gt, eps=eps, **kw, **par)
    got = {"h": h, "n": n, **gated_norm.backward(gh, gn, x, y, gt, stats, **kw, **par)}
    T = x.numel() // shape[-1]
    # what one fp32 ulp of x and y does to each result: a row without much spread magnifies it
    g = torch.Generator().manual_seed(1)
    ulp = lambda t: t.double() * (1 + 2.0**-23 * (torch.randint(0, 2, t.shape, generator=g) * 2 - 1).to(device))  # noqa: E731
    near = ref.gated_norm(ulp(x), ulp(y), gt, par, kind, eps, post, pre, gh, gn)
    for name, value in want.items():
        # half an ulp of the store, and fp32 arithmetic: 2^-17 of the largest value that takes
        # part (1 / std included), of a root of T such terms where tokens are summed
        terms = T if name[1:] in WEIGHTS else T / max(1, gt.numel() // shape[-1]) if name == "dgate" else 1
        size = max(4.0, value.abs().max().item(), *(t.abs().max().item() for t in want.values() if t.dim() > 1))
        ref.assert_within(got[name], value, ref.store(value, got[name].dtype) + 2.0**-17 * size * terms**0.5
                          + 4 * (near[name] - value).abs().max(), f"{name} {dtype} {shape} {kind}")
    assert (n is None) == (not pre)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", [(1, 64), (3, 128), (257, 128), (33, 96), (5, 7, 200), (19, 37), (40, 771), (9, 1024),
                                   (6, 4100), (3, 8192), (1500, 33), (700, 2)])
def test_matches_definition(device, dtype, kind, shape):
    _check(device, dtype, shape, shape, kind, seed=shape[-1])


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape,gate", [((3, 500, 128), (3, 1, 128)), ((2, 3, 40, 72), (2, 1, 1, 72)),
                                        ((2, 3, 40, 72), (2, 3, 1, 72)), ((900, 129), (1, 129)), ((600, 2, 64), (600, 1, 64)),
                                        ((1, 5000, 1032), (1, 1, 1032)), ((4, 30, 128), None)])
def test_gates_shared_by_tokens(device, dtype, shape, gate):
    _check(device, dtype, shape, gate, seed=len(shape))


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("kw", [
    dict(weights=()), dict(weights=("res_scale",), kind="rms"), dict(post=False), dict(pre=False), dict(dh=False),
    dict(dn=False), dict(weights=("post_bias", "pre_bias")), dict(weights=("post_weight", "pre_weight", "pre_bias"), kind="rms"),
    dict(w_dtype=FP), dict(eps=0.1), dict(post=False, pre=False, weights=("res_scale",)), dict(dh=False, pre=False)])
def test_parts(device, dtype, kw):
    _check(device, dtype, (70, 136), (70, 136), **kw)


@gpu
def test_constant_rows(device):
    """A row without spread: 1 / sqrt(eps), nothing infinite."""
    x, y, gt, par, gh, gn = _inputs(device, FP, (4, 128), (4, 128))
    x, y = torch.zeros_like(x), torch.full_like(y, 3.0)
    h, n, st = gated_norm.forward(x, y, gt, **par)
    g = gated_norm.backward(gh, gn, x, y, gt, st, **par)
    assert all(torch.isfinite(t).all() for t in (h, n, *g.values()))
    far = torch.full_like(x, 1e4) + torch.randn(4, 128, generator=torch.Generator().manual_seed(0)).to(device)
    want = ref.gated_norm(x, far, gt, par, "layer", 1e-5)
    h, _, _ = gated_norm.forward(x, far, gt, **par)  # far from zero: the spread is of the distances from the mean
    ref.assert_within(h, want["h"], torch.full_like(want["h"], 1e-2), "far mean")


@gpu
def test_gate_range(device):
    """A gate of +-100 is open or shut, one of +-infinity too."""
    x, y, _, par, gh, gn = _inputs(device, BF, (6, 64), None)
    gate = torch.tensor([100.0, -100.0, float("inf"), -float("inf"), 0.0, 15.0], device=device, dtype=BF)[:, None].expand(6, 64)
    h, n, st = gated_norm.forward(x, y, gate.contiguous(), **par)
    u = torch.nn.functional.layer_norm(y.double(), (64,), par["post_weight"].double(), par["post_bias"].double(), 1e-5)
    want = x.double() + par["res_scale"].double() * u * torch.sigmoid(gate.double())
    ref.assert_within(h, want, 2.0**-8 * want.abs() + 2.0**-14, "gated h")
    g = gated_norm.backward(gh, gn, x, y, gate.contiguous(), st, **par)
    assert all(torch.isfinite(t).all() for t in g.values())


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides(device, dtype):
    """Rows that are parts of wider ones, an expanded x, and pointers off 16 bytes."""
    C = 128
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(60, 3 * C + 4, generator=g).to(device, dtype)
    x, y, gt = wide[:, :C], wide[:, C:2 * C], wide[:, 2 * C + 4:3 * C + 4]
    par = {n: torch.randn(C, generator=g).to(device, dtype) for n in WEIGHTS}
    a = gated_norm.forward(x.contiguous(), y.contiguous(), gt.contiguous(), **par)
    for b in (gated_norm.forward(x, y, gt, **par), gated_norm.forward(x, wide[:, C + 1:2 * C + 1], gt, **par)):
        assert b[0].shape == x.shape
    for s, t in zip(a, gated_norm.forward(x, y, gt, **par)):
        torch.testing.assert_close(s, t, rtol=2.0**-7 if dtype == BF else 1e-6, atol=1e-5)
    row = x[:1].expand(60, C)
    c = gated_norm.forward(row.contiguous(), y.contiguous(), gt.contiguous(), **par)
    torch.testing.assert_close(c[0], gated_norm.forward(row, y, gt, **par)[0], rtol=2.0**-7 if dtype == BF else 1e-6, atol=1e-5)
    three = wide.view(3, 20, -1)[:, ::2]
    d = gated_norm.forward(three[..., :C], three[..., C:2 * C], None, **par)
    e = gated_norm.forward(three[..., :C].contiguous(), three[..., C:2 * C].contiguous(), None, **par)
    torch.testing.assert_close(d[1], e[1], rtol=2.0**-7 if dtype == BF else 1e-6, atol=1e-5)


@gpu
def test_repeatable_and_autograd(device):
    x, y, gt, par, gh, gn = _inputs(device, BF, (2, 3000, 128), (2, 1, 128))
    h, n, st = gated_norm.forward(x, y, gt, **par)
    a = gated_norm.backward(gh, gn, x, y, gt, st, **par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = gated_norm.backward(gh, gn, x, y, gt, st, **par)
    torch.cuda.current_stream().wait_stream(side)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    leaves = {"x": x, "y": y, "gate": gt, **par}
    leaves = {k: t.clone().requires_grad_() for k, t in leaves.items()}
    args = [leaves.pop(k) for k in ("x", "y", "gate")]
    h2, n2 = gated_norm.gated_norm(*args, **leaves)
    grads = torch.autograd.grad((h2, n2), [*args, *leaves.values()], (gh, gn))
    for k, t in zip(("x", "y", "gate", *leaves), grads):
        assert torch.equal(a["d" + k], t), k
    only = torch.autograd.grad(gated_norm.gated_norm(*args, **leaves)[0], [args[1], leaves["pre_weight"]], gh,
                               allow_unused=True)
    assert not only[1].any()


@gpu
def test_gradient_against_differences(device):
    """fp32, along one direction of everything that has a gradient."""
    x, y, gt, par, gh, gn = _inputs(device, FP, (30, 96), (30, 96))
    _, _, st = gated_norm.forward(x, y, gt, **par)
    grads = gated_norm.backward(gh, gn, x, y, gt, st, **par)
    at = {"x": x, "y": y, "gate": gt, **par}
    way = {k: torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(device) for i, (k, t) in enumerate(at.items())}

    def loss(e):
        p = {k: t + e * way[k] for k, t in at.items()}
        h, n, _ = gated_norm.forward(p.pop("x"), p.pop("y"), p.pop("gate"), **p)
        return ((h.double() * gh).sum() + (n.double() * gn).sum()).item()

    eps = 1e-2
    slope = (loss(eps) - loss(-eps)) / (2 * eps)
    terms = [(grads["d" + k].double() * way[k]) for k in at]
    size = sum(t.abs().sum().item() for t in terms)
    assert abs(slope - sum(t.sum().item() for t in terms)) <= 2e-3 * size


@gpu
def test_empty(device):
    x = torch.zeros(0, 64, dtype=BF, device=device)
    w = torch.ones(64, dtype=BF, device=device)
    h, n, st = gated_norm.forward(x, x, x, pre_weight=w)
    g = gated_norm.backward(h, n, x, x, x, st, pre_weight=w)
    assert h.shape == x.shape and not g["dpre_weight"].any()


def test_refusals():
    x = torch.zeros(4, 64)
    f = gated_norm.forward
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        f(x, x)
    with pytest.raises(AssertionError):
        f(x, x[:, :32])
    with pytest.raises(AssertionError):
        f(x, x, x[:3])
    with pytest.raises(AssertionError):
        f(x, x, x[:, :32])
    with pytest.raises(AssertionError):
        f(x, x, pre_weight=torch.ones(63))
    with pytest.raises(AssertionError):
        f(torch.zeros(1, 8193), torch.zeros(1, 8193))
    with pytest.raises(ValueError):
        f(x, x, kind="batch")
    with pytest.raises(ValueError):
        f(x.double(), x.double())
    with pytest.raises(ValueError):
        f(x.half(), x.half(), pre_weight=torch.ones(64).bfloat16())
    with pytest.raises(ValueError):
        f(x, x.half())
    with pytest.raises(ValueError):
        f(x.half(), x.half(), pre_weight=torch.ones(64), post_weight=torch.ones(64).half())
    with pytest.raises(AssertionError):
        gated_norm.backward(x, x, x, x, None, torch.zeros(3, 4))
    with pytest.raises(ValueError):
        gated_norm.backward(x.half(), x, x, x, None, torch.zeros(4, 4))
