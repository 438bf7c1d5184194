"""Rotary positions with several axes against the definition in 64 bits."""
import pytest
import torch

import block_refs as ref
from triangleops_b200 import rotary

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _inputs(device, dtype, B, N, Hq, Hk, D, axes, seed=0, most=5000):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(device, dtype)  # noqa: E731
    return r(B, N, Hq, D), r(B, N, Hk, D), torch.randint(-most, most, (axes, B, N), generator=g).int().to(device)


def _within(got, t, pos, tab, sign, what):
    value, size = ref.rotary(t, pos, tab["inv_freq"], tab["axis"], tab["interleaved"], sign)
    # the store, and a cosine and a sine of fp32 (2^-22) times the pair
    ref.assert_within(got, value, ref.store(value, t.dtype) + 2.0**-21 * size, what)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,Hq,Hk,D,sections", [
    (1, 1, 1, 1, 32, (16,)), (2, 37, 6, 2, 64, (16, 16)), (3, 130, 4, 1, 128, (16, 24, 24)), (1, 7, 2, 2, 96, (20, 20)),
    (2, 5, 3, 1, 10, (2, 1)), (1, 600, 8, 8, 48, (7, 0, 9)), (64, 1, 32, 8, 128, (64,)), (1, 3, 2, 1, 7, (3,)),
    (1, 9, 5, 5, 256, (128,)), (2, 21, 1, 3, 40, (4, 4, 4, 4)),
])
def test_matches_definition(device, dtype, interleaved, B, N, Hq, Hk, D, sections):
    q, k, pos = _inputs(device, dtype, B, N, Hq, Hk, D, len(sections), seed=D)
    inv_freq, axis = rotary.frequencies(D, sections, device=device)
    tab = dict(inv_freq=inv_freq, axis=axis, interleaved=interleaved)
    qo, ko = rotary.forward(q, k, pos, **tab)
    _within(qo, q, pos, tab, 1.0, "q")
    _within(ko, k, pos, tab, 1.0, "k")
    dq, dk = rotary.backward(q, k, pos, **tab)
    _within(dq, q, pos, tab, -1.0, "dq")
    _within(dk, k, pos, tab, -1.0, "dk")
    alone, none = rotary.forward(q, None, pos.long(), **tab)
    assert none is None and torch.equal(alone, qo)


@gpu
def test_far_positions(device):
    """fp32 at positions of millions: the angle keeps its digits."""
    q, k, pos = _inputs(device, FP, 1, 64, 2, 1, 64, 2, most=50_000_000)
    inv_freq, axis = rotary.frequencies(64, (16, 16), per_axis=True, device=device)
    tab = dict(inv_freq=inv_freq, axis=axis, interleaved=False)
    qo, _ = rotary.forward(q, k, pos, **tab)
    _within(qo, q, pos, tab, 1.0, "far q")


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides(device, dtype):
    B, N, H, D = 2, 50, 4, 64
    qkv = torch.randn(B, N, 3 * H * D, generator=torch.Generator().manual_seed(0)).to(device, dtype)
    q, k, _ = (t.view(B, N, H, D) for t in qkv.split(H * D, -1))
    pos = torch.arange(N, device=device, dtype=torch.int32).expand(2, B, N)
    inv_freq, axis = rotary.frequencies(D, (20, 12), device=device)
    tab = dict(inv_freq=inv_freq, axis=axis)
    a = rotary.forward(q.contiguous(), k.contiguous(), pos.contiguous(), **tab)
    odd = [torch.nn.functional.pad(t, (0, 1))[..., :D] for t in (q, k)]
    hf = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k)]
    last = [t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for t in (q, k)]
    for x, y in ((q, k), odd, hf, last):
        b = rotary.forward(x, y, pos, **tab)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
def test_autograd_and_differences(device):
    """The turn is linear: its gradient is its transpose."""
    q, k, pos = _inputs(device, FP, 2, 20, 3, 1, 32, 2)
    inv_freq, axis = rotary.frequencies(32, (6, 7), device=device)
    q, k = q.requires_grad_(), k.requires_grad_()
    qo, ko = rotary.rotary(q, k, pos, inv_freq=inv_freq, axis=axis, interleaved=True)
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    t = torch.randn_like(q)
    moved, _ = rotary.forward(q.detach() + t, k.detach(), pos, inv_freq=inv_freq, axis=axis, interleaved=True)
    slope = ((moved.double() - qo.detach().double()) * dq.double()).sum()
    assert abs(slope - (gq.double() * t.double()).sum()) <= 1e-5 * (gq.double() * t.double()).abs().sum()
    assert gk.shape == k.shape
    only_q, = torch.autograd.grad(rotary.rotary(q, None, pos, inv_freq=inv_freq, axis=axis)[0], q, dq)
    assert only_q.shape == q.shape


@gpu
def test_unknown_axis_and_empty(device):
    q, k, pos = _inputs(device, BF, 1, 5, 2, 1, 32, 1)
    inv_freq, axis = rotary.frequencies(32, (16,), device=device)
    bad = axis.clone()
    bad[3], bad[5] = 7, -1
    qo, _ = rotary.forward(q, k, pos, inv_freq=inv_freq, axis=bad)
    for f in (3, 5):
        assert torch.equal(qo[..., [f, 16 + f]], q[..., [f, 16 + f]])
    e, _ = rotary.forward(q[:, :0], k[:, :0], pos[:, :, :0], inv_freq=inv_freq, axis=axis)
    assert e.shape == (1, 0, 2, 32)


def test_frequencies():
    f, a = rotary.frequencies(128, (16, 24, 24))
    assert f.shape == (64,) and a.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    assert abs(f[32].item() - 0.01) < 1e-8
    f, a = rotary.frequencies(64, (8, 4), base=100.0, per_axis=True)
    assert f[8].item() == 1.0 and abs(f[4].item() - 0.1) < 1e-7
    with pytest.raises(AssertionError):
        rotary.frequencies(32, (16, 1))
    with pytest.raises(ValueError):
        rotary.frequencies(32, (16, -1))


def test_refusals():
    q = torch.zeros(1, 4, 2, 32)
    pos = torch.zeros(1, 1, 4, dtype=torch.int32)
    f, a = rotary.frequencies(32, (16,))
    ok = dict(inv_freq=f, axis=a)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary.forward(q, None, pos, **ok)
    with pytest.raises(AssertionError):
        rotary.forward(q, q[:, :3], pos, **ok)
    with pytest.raises(AssertionError):
        rotary.forward(q, None, pos[:, :, :3], **ok)
    with pytest.raises(AssertionError):
        rotary.forward(q[..., :16], None, pos, **ok)
    with pytest.raises(AssertionError):
        rotary.forward(q, None, pos, inv_freq=f, axis=a[:3])
    with pytest.raises(ValueError):
        rotary.forward(q, None, pos.float(), **ok)
    with pytest.raises(ValueError):
        rotary.forward(q, None, pos, inv_freq=f.double(), axis=a)
    with pytest.raises(ValueError):
        rotary.forward(q, q.half(), pos, **ok)
    with pytest.raises(ValueError):
        rotary.forward(q.double(), None, pos, **ok)
