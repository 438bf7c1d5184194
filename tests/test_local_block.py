"""The token block that runs windowed attention, the gated norms and rotary positions together."""
import pytest
import torch
import torch.nn.functional as F

import block_refs as ref
from triangleops_b200 import local_block

gpu = pytest.mark.gpu
KW = dict(C=96, heads=4, kv_heads=2, head_dim=32, hidden=160, blocks=2, sections=(6, 5, 5), res_scale=0.5)


def _setup(dtype, device, kind="layer", B=2, N=70, seed=0):
    g = torch.Generator().manual_seed(seed)
    pre = local_block.init(**KW, kind=kind, dtype=dtype, device=device, generator=g)
    s = torch.randn(B, N, KW["C"], generator=g).to(device, dtype)
    pos = torch.stack([torch.arange(N).expand(B, N), torch.randint(0, 3, (B, N), generator=g),
                       torch.arange(N).expand(B, N) % 7]).int().to(device)
    return pre, s, pos, g


def _plain(s, pre, pos, window, sinks, mask, kind, eps=1e-5):
    """The block in elementary operations, in the tensors' own precision."""
    def norm(t, w, b):
        t = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * w
        return t if b is None else t + b

    def join(s, y, g, p):
        h = s + p["res_scale"] * norm(y, p["post_weight"], p["post_bias"]) * torch.sigmoid(g)
        return h, norm(h, p["pre_weight"], p["pre_bias"])

    hq, hk, D = pre["heads"]
    tab = pre["rotary"]
    ang = pos[tab["axis"].long()].to(s.dtype).permute(1, 2, 0)[:, :, None] * tab["inv_freq"].to(s.dtype)
    left, right = (window - 1, 0) if isinstance(window, int) else window
    N = s.shape[1]
    see = ref.visible(N, N, left, right, sinks, mask, s.device)

    def turn(t):
        P = ang.shape[-1]
        a, b, rest = t[..., :P], t[..., D // 2:D // 2 + P], t[..., D // 2 + P:]
        return torch.cat([a * ang.cos() - b * ang.sin(), t[..., P:D // 2], a * ang.sin() + b * ang.cos(), rest], -1)

    n = norm(s, pre["first"]["weight"], pre["first"]["bias"])
    for b in pre["blocks"]:
        q, k, v, g = local_block._project(n, b, pre)
        q, k, v = (t.permute(0, 2, 1, 3) for t in (turn(q), turn(k), v))
        k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
        z = (q @ k.mT * D**-0.5).masked_fill(~see, -1e30)
        w = torch.softmax(z, -1) * see.any(-1, keepdim=True)
        o = (w @ v).permute(0, 2, 1, 3).flatten(-2)
        s, n = join(s, F.linear(o, b["w_o"]), g, b["attn"])
        u, w, g = F.linear(n, b["w_up"]).split([pre["hidden"]] * 2 + [s.shape[-1]], -1)
        s, n = join(s, F.linear(F.silu(u) * w, b["w_down"]), g, b["mlp"])
    return s, n


def _double(pre):
    if isinstance(pre, dict):
        return {k: _double(v) for k, v in pre.items()}
    if isinstance(pre, list):
        return [_double(v) for v in pre]
    return pre.detach().double() if isinstance(pre, torch.Tensor) and pre.is_floating_point() else pre


@gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("window,sinks,masked", [((9, 4), 2, True), (16, 3, False)])
def test_forward_and_gradients(device, kind, window, sinks, masked):
    """fp32 against the plain block in 64 bits, the gradients of every weight and of the input:
    two blocks of some hundred fp32 operations in a row, 1e-4 of each tensor's largest value."""
    pre, s, pos, g = _setup(torch.float32, device, kind)
    mask = (torch.rand(s.shape[:2], generator=g) < 0.8).to(device) if masked else None
    params = [s, *local_block.weights(pre)]
    for t in params:
        t.requires_grad_()
    out, n = local_block.forward(s, pre, pos, window=window, sinks=sinks, mask=mask)
    d, dn = torch.randn(out.shape, generator=g).to(device), torch.randn(out.shape, generator=g).to(device)
    torch.backends.cuda.matmul.allow_tf32 = False
    got = [out, n, *torch.autograd.grad((out, n), params, (d, dn))]
    pre64, s64 = _double(pre), s.detach().double()
    params64 = [s64, *local_block.weights(pre64)]
    for t in params64:
        t.requires_grad_()
    want = _plain(s64, pre64, pos, window, sinks, mask, kind)
    want = [*want, *torch.autograd.grad(want, params64, (d.double(), dn.double()))]
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a.double() - b).abs().max() <= 1e-4 * b.abs().max(), i


@gpu
def test_training_lowers_the_loss(device):
    """bf16: some steps of gradient descent on tokens shifted by one."""
    pre, s, pos, _ = _setup(torch.bfloat16, device)
    params = local_block.weights(pre)
    for t in params:
        t.requires_grad_()
    target = s.roll(1, 1)
    losses = []
    for _ in range(25):
        _, n = local_block.forward(s, pre, pos, window=8, sinks=1)
        loss = (n.float() - target.float()).square().mean()
        losses.append(loss.item())
        for t, g in zip(params, torch.autograd.grad(loss, params)):
            t.data.add_(g, alpha=-0.5)
    assert all(x == x for x in losses) and losses[-1] < 0.8 * losses[0], losses


@gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2.0**-4)])
def test_steps_equal_the_whole_sequence(device, dtype, tol):
    """Token by token against the caches, as reading the sequence in at once (bf16: four
    roundings of a stream of about 4 in size, 2^-6 each, in either)."""
    pre, s, pos, _ = _setup(dtype, device, B=3, N=40)
    whole, _ = local_block.forward(s, pre, pos, window=12, sinks=2)
    cache = local_block.caches(pre, 3, 48, dtype=dtype, device=device)
    for kc, vc in cache:
        kc.fill_(float("nan")), vc.fill_(float("nan"))
    lengths = torch.zeros(3, dtype=torch.int32, device=device)
    for t in range(40):
        out, _ = local_block.step(s[:, t], pre, pos[:, :, t], cache, lengths, window=12, sinks=2)
        lengths += 1
        assert (out.float() - whole[:, t].float()).abs().max() <= tol, t


def test_init_and_refusals():
    pre = local_block.init(**KW, kind="rms")
    assert len(local_block.weights(pre)) == 1 + 2 * (4 + 2 * 3)
    assert pre["blocks"][0]["w_in"].shape == ((4 + 4) * 32 + 96, 96)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        local_block.forward(torch.zeros(1, 4, 96), pre, torch.zeros(3, 1, 4, dtype=torch.int32), window=2)
