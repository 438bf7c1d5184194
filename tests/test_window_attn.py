"""Windowed attention with sinks against its definition in 64 bits: forward, gradients, one token."""
import pytest
import torch

import block_refs as ref
from triangleops_b200 import _lib, window_attn

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _inputs(device, dtype, B, Nq, Nk, Hq, Hkv, D, seed=0, sd=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * sd).to(device, dtype)  # noqa: E731
    return r(B, Nq, Hq, D), r(B, Nk, Hkv, D), r(B, Nk, Hkv, D), r(B, Nq, Hq, D)


def _check(device, dtype, B, Nq, Nk, Hq, Hkv, D, window, sinks, mask=None, seed=0, scale=None, poison=True, grads=True,
           sd=1.0):
    q, k, v, dout = _inputs(device, dtype, B, Nq, Nk, Hq, Hkv, D, seed, sd)
    want = ref.attention(q, k, v, window, sinks, mask, scale, dout if grads else None)
    if mask is not None and poison:  # what masked keys hold must not matter
        gone = (mask == 0)[..., None, None]
        k, v = k.masked_fill(gone, float("nan")), v.masked_fill(gone, float("inf"))
    kw = dict(window=window, sinks=sinks, mask=mask, scale=scale)
    out, lse = window_attn.forward(q, k, v, **kw)
    what = f"{dtype} {(B, Nq, Nk, Hq, Hkv, D)} window {window} sinks {sinks}"
    ref.assert_within(out, *want["out"], f"out {what}")
    torch.testing.assert_close(lse.double(), want["lse"][0], rtol=1e-3 if dtype != FP else 1e-5,
                               atol=1e-3 if dtype != FP else 1e-5)
    if grads:
        for name, got in zip(("dq", "dk", "dv"), window_attn.backward(dout, q, k, v, out, lse, **kw)):
            ref.assert_within(got, *want[name], f"{name} {what}")
    assert _lib.device_error()[0] == 0


# lengths of one token, on and around tile edges; head sizes on and off the tensor-core widths
@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("N,Hq,Hkv,D,window,sinks", [
    (1, 1, 1, 32, 1, 0),
    (2, 2, 1, 64, 1, 1),
    (37, 3, 1, 64, 8, 2),
    (64, 4, 4, 32, (16, 16), 0),
    (127, 2, 2, 128, 32, 4),
    (128, 4, 2, 128, (0, 0), 0),
    (129, 4, 1, 64, (5, 200), 3),
    (257, 2, 1, 16, 100, 7),
    (300, 2, 2, 40, 64, 1),
    (513, 8, 2, 128, 130, 4),
    (700, 2, 1, 64, (300, 17), 130),
    (1025, 1, 1, 96, 128, 200),
    (1100, 2, 2, 32, 2000, 0),
])
def test_matches_definition(device, dtype, N, Hq, Hkv, D, window, sinks):
    _check(device, dtype, 2, N, N, Hq, Hkv, D, window, sinks, seed=N)


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [7, 20, 160, 256])
def test_odd_heads(device, dtype, D):
    _check(device, dtype, 1, 70, 70, 2, 1, D, 24, 2, seed=D)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("Nq,Nk,window,sinks", [(1, 400, 100, 4), (5, 261, 64, 0), (130, 700, 256, 9), (64, 64, 64, 0),
                                               (200, 1000, (50, 30), 64)])
def test_queries_are_the_last_tokens(device, dtype, Nq, Nk, window, sinks):
    _check(device, dtype, 2, Nq, Nk, 4, 2, 64, window, sinks, seed=Nq)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("kind", ["tail", "random", "none_kept", "first_only", "late_only"])
def test_masks(device, dtype, D, kind):
    """Rows that a mask leaves empty, masked sinks, and NaN and infinity in masked places."""
    B, N = 3, 333
    g = torch.Generator().manual_seed(5)
    mask = torch.ones(B, N, dtype=torch.bool)
    if kind == "tail":
        for b, n in enumerate((N - 1, 129, 3)):
            mask[b, n:] = False
    elif kind == "random":
        mask = torch.rand(B, N, generator=g) < 0.6
    elif kind == "none_kept":
        mask[1] = False
    elif kind == "first_only":
        mask[:, 1:] = False
    else:
        mask[:, :300] = False
    for sinks in (0, 5):
        _check(device, dtype, B, N, N, 4, 2, D, (40, 7), sinks, mask.to(device), seed=9)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,N,Hq,Hkv,D,window,sinks", [(9, 700, 8, 2, 64, 100, 40), (3, 1300, 10, 5, 128, (50, 20), 0),
                                                       (40, 129, 8, 8, 32, 1, 1)])
def test_more_tiles_than_blocks(device, dtype, B, N, Hq, Hkv, D, window, sinks):
    """Blocks that take several tiles, over the ends of heads and sequences, some with no key at all."""
    mask = torch.rand(B, N, generator=torch.Generator().manual_seed(B)) < 0.8
    mask[1] = False
    _check(device, dtype, B, N, N, Hq, Hkv, D, window, sinks, mask.to(device), seed=N)


@gpu
def test_mask_types(device):
    q, k, v, _ = _inputs(device, BF, 2, 90, 90, 2, 2, 64)
    keep = (torch.rand(2, 90, generator=torch.Generator().manual_seed(1)) < 0.5).to(device)
    a, _ = window_attn.forward(q, k, v, window=32, mask=keep)
    for m in (keep.int(), keep.float() * 0.25, keep.to(torch.uint8) * 7, keep.t().contiguous().t()):
        assert torch.equal(a, window_attn.forward(q, k, v, window=32, mask=m)[0])


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_scores(device, dtype):
    """Scores of some hundreds: the running maximum moves, sums do not overflow."""
    _check(device, dtype, 1, 500, 500, 2, 1, 64, 200, 3, seed=3, sd=4.0, grads=False)
    _check(device, dtype, 1, 260, 260, 2, 1, 64, 200, 3, seed=3, scale=-0.5, grads=False)


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides(device, dtype):
    """Parts of one projection, heads before tokens, a batch taken from the end of a buffer, and
    strides that 16-byte loads cannot follow."""
    B, N, H, D = 2, 150, 4, 64
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(B, N, 3 * H * D, generator=g).to(device, dtype)
    q, k, v = (t.reshape(B, N, H, D) for t in qkv.split(H * D, -1))
    kw = dict(window=(40, 9), sinks=3)
    base, lse = window_attn.forward(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
    d = torch.randn(B, N, H, D, generator=g).to(device, dtype)
    grads = window_attn.backward(d, q.contiguous(), k.contiguous(), v.contiguous(), base, lse, **kw)

    def heads_first(t):
        return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)

    def odd(t):
        return torch.nn.functional.pad(t, (0, 3))[..., :D]

    def reversed_channels(t):
        return t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device=device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    for f in (lambda t: t, heads_first, odd, reversed_channels, shifted):
        a, l2 = window_attn.forward(f(q), f(k), f(v), **kw)
        want = ref.attention(q, k, v, (40, 9), 3, dout=d)
        ref.assert_within(a, *want["out"], "strided out")
        for name, x in zip(("dq", "dk", "dv"), window_attn.backward(f(d), f(q), f(k), f(v), a, l2, **kw)):
            ref.assert_within(x, *want[name], f"strided {name}")
    one = k[:, :, :1].expand(B, N, H, D)  # one key head for all, by a stride of zero
    a, _ = window_attn.forward(q, one, v, **kw)
    assert torch.equal(a, window_attn.forward(q, one.contiguous(), v, **kw)[0])
    assert len(grads) == 3


@gpu
def test_empty(device):
    for B, Nq, Nk in ((0, 5, 5), (2, 0, 0), (2, 0, 9)):
        q, k, v, d = _inputs(device, BF, B, Nq, Nk, 2, 2, 64)
        out, lse = window_attn.forward(q, k, v, window=4)
        dq, dk, dv = window_attn.backward(d, q, k, v, out, lse, window=4)
        assert out.shape == q.shape and dq.shape == q.shape and dk.shape == k.shape
        assert not dk.any() and not dv.any()


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_repeatable_on_other_streams(device, dtype):
    """The same bits each time, on a stream that is not the default, and from a CUDA graph."""
    q, k, v, d = _inputs(device, dtype, 2, 700, 700, 4, 2, 64)
    kw = dict(window=128, sinks=5)

    def step():
        out, lse = window_attn.forward(q, k, v, **kw)
        return (out, *window_attn.backward(d, q, k, v, out, lse, **kw))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_gradient_against_differences(device):
    """fp32: the loss along a direction, at two points on either side (its third derivative
    times eps^2 / 6 and 2e-6 of rounding over eps bound the difference)."""
    q, k, v, d = _inputs(device, FP, 1, 60, 60, 2, 1, 16, seed=4)
    kw = dict(window=(10, 3), sinks=2)
    t = [torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(device) for i, x in enumerate((q, k, v))]
    out, lse = window_attn.forward(q, k, v, **kw)
    grads = window_attn.backward(d, q, k, v, out, lse, **kw)
    eps = 1e-2
    loss = lambda e: (window_attn.forward(q + e * t[0], k + e * t[1], v + e * t[2], **kw)[0].double() * d.double()).sum()  # noqa: E731,E501
    slope = (loss(eps) - loss(-eps)) / (2 * eps)
    exact = sum((a.double() * b.double()).sum() for a, b in zip(grads, t))
    size = sum((a.double() * b.double()).abs().sum() for a, b in zip(grads, t))
    assert abs(slope - exact) <= 2e-3 * size


@gpu
def test_autograd(device):
    q, k, v, d = _inputs(device, BF, 2, 140, 140, 4, 2, 64)
    kw = dict(window=50, sinks=2)
    out, lse = window_attn.forward(q, k, v, **kw)
    want = window_attn.backward(d, q, k, v, out, lse, **kw)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(window_attn.window_attention(*leaves, **kw), leaves, d)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
def test_first_use_in_a_new_thread(device):
    """A thread that has made no CUDA call yet (as autograd's are)."""
    import threading

    q, k, v, d = _inputs(device, BF, 1, 200, 200, 2, 1, 64)
    want, lse = window_attn.forward(q, k, v, window=64, sinks=1)
    torch.cuda.synchronize()
    got = []

    def work(f):
        try:
            got.append(f())
        except Exception as e:  # noqa: BLE001
            got.append(e)

    for f in (lambda: window_attn.forward(q, k, v, window=64, sinks=1)[0],
              lambda: window_attn.backward(d, q, k, v, want, lse, window=64, sinks=1)[2]):
        t = threading.Thread(target=work, args=(f,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)
    assert torch.equal(got[1], window_attn.backward(d, q, k, v, want, lse, window=64, sinks=1)[2])


def _decode_ref(q, k, v, lengths, window, sinks):
    out, err = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        n = min(n, k.shape[1])
        if n <= 0:
            continue
        o, e = ref.attention(q[b:b + 1, None], k[b:b + 1, :n], v[b:b + 1, :n], window, sinks)["out"]
        out[b], err[b] = o[0, 0], e[0, 0]
    return out, err


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("N,Hq,Hkv,D,window,sinks", [
    (1, 1, 1, 32, 1, 0), (40, 4, 4, 32, 16, 2), (300, 8, 2, 128, 100, 4), (1000, 6, 2, 64, 2000, 0),
    (1500, 32, 8, 128, 700, 5), (515, 20, 1, 64, 129, 1), (2100, 40, 2, 128, 1, 0), (333, 3, 3, 40, 33, 300),
    (200, 2, 1, 24, 64, 3), (130, 2, 2, 7, 64, 3), (9000, 8, 2, 128, 9000, 0), (9001, 20, 1, 64, 6000, 7),
    (5000, 3, 3, 40, 4999, 1), (700, 64, 32, 128, 650, 9),
])
def test_decode(device, dtype, N, Hq, Hkv, D, window, sinks):
    B = 5
    q, k, v, _ = _inputs(device, dtype, B, N, N, Hq, Hkv, D, seed=N)
    q = q[:, 0].contiguous()
    lengths = torch.tensor([N, max(1, N // 2), 1, 0, N + 3], dtype=torch.int32, device=device)
    want = _decode_ref(q, k, v, lengths, window, sinks)
    for b, n in enumerate(lengths.tolist()):  # places no sequence has filled hold anything
        k[b, max(n, 0):], v[b, max(n, 0):] = float("nan"), float("nan")
    out = window_attn.decode(q, k, v, lengths, window=window, sinks=sinks)
    ref.assert_within(out, *want, f"decode {dtype} {(N, Hq, Hkv, D)} window {window} sinks {sinks}")
    assert not out[3].any()
    assert torch.equal(out, window_attn.decode(q, k, v, lengths.long(), window=window, sinks=sinks))


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_decode_strides_and_streams(device, dtype):
    """Caches stored heads first, and as halves of one buffer; a side stream; a graph."""
    B, N, Hq, Hkv, D = 3, 600, 8, 2, 64
    q, k, v, _ = _inputs(device, dtype, B, N, N, Hq, Hkv, D)
    q = q[:, 0]
    lengths = torch.tensor([600, 333, 64], dtype=torch.int32, device=device)
    kw = dict(window=200, sinks=4)
    a = window_attn.decode(q.contiguous(), k, v, lengths, **kw)
    both = torch.stack([k, v], 2)  # (B, N, 2, Hkv, D)
    assert torch.equal(a, window_attn.decode(q, both[:, :, 0], both[:, :, 1], lengths, **kw))
    hf = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v)]
    assert torch.equal(a, window_attn.decode(q, *hf, lengths, **kw))
    odd = [torch.nn.functional.pad(t, (0, 1))[..., :D] for t in (k, v)]
    ref.assert_within(window_attn.decode(q, *odd, lengths, **kw), *_decode_ref(q, k, v, lengths, 200, 4), "odd strides")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = window_attn.decode(q, k, v, lengths, **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, b)


@gpu
def test_decode_far_into_a_large_cache(device):
    """Keys beyond 2^32 bytes of the cache."""
    B, N, Hkv, D = 1, 17 * 2**20, 2, 64  # 4.6 GB each
    k = torch.zeros(B, N, Hkv, D, dtype=BF, device=device)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(1)
    n = N - 3
    tail = torch.randn(2, 1, 300, Hkv, D, generator=g).to(device, BF)
    k[:, n - 300:n], v[:, n - 300:n] = tail[0], tail[1]
    q = torch.randn(B, 4, D, generator=g).to(device, BF)
    out = window_attn.decode(q, k, v, torch.tensor([n], dtype=torch.int32, device=device), window=300)
    o, e = ref.attention(q[:, None], tail[0], tail[1], 300, 0)["out"]
    ref.assert_within(out, o[:, 0], e[:, 0], "far decode")


def test_refusals():
    q = torch.zeros(2, 8, 4, 32, dtype=BF)
    k = torch.zeros(2, 8, 2, 32, dtype=BF)
    f = window_attn.forward
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        f(q, k, k, window=4)
    with pytest.raises(AssertionError):
        f(q, k[:, :, :, :16], k, window=4)
    with pytest.raises(AssertionError):
        f(q, torch.zeros(2, 8, 3, 32, dtype=BF), torch.zeros(2, 8, 3, 32, dtype=BF), window=4)  # 4 % 3
    with pytest.raises(AssertionError):
        f(q, k[:, :7], k[:, :7], window=4)  # more queries than keys
    with pytest.raises(AssertionError):
        f(q[0], k, k, window=4)
    with pytest.raises(ValueError):
        f(q, k.half(), k.half(), window=4)
    with pytest.raises(ValueError):
        f(q.double(), k.double(), k.double(), window=4)
    for window in (0, -3, (-1, 2), (2, -1)):
        with pytest.raises(ValueError):
            f(q, k, k, window=window)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        window_attn.decode(q[:, 0], k, k, torch.ones(2, dtype=torch.int32), window=4)
    with pytest.raises(AssertionError):
        window_attn.decode(q[:, 0], k, k, torch.ones(3, dtype=torch.int32), window=4)
    with pytest.raises(ValueError):
        window_attn.decode(q[:, 0], k, k, torch.ones(2, dtype=torch.int32), window=(4, 0))
    with pytest.raises(AssertionError):
        window_attn.backward(q[:, :4], q, k, k, q, torch.zeros(2, 4, 8), window=4)
    with pytest.raises(AssertionError):
        window_attn.backward(q, q, k, k, q, torch.zeros(2, 8, 4), window=4)


@gpu
def test_refusals_on_device(device):
    q, k, v, _ = _inputs(device, BF, 2, 8, 8, 2, 2, 32)
    with pytest.raises(AssertionError):
        window_attn.forward(q, k, v, window=4, mask=torch.ones(2, 7, dtype=torch.bool, device=device))
    with pytest.raises(ValueError):
        window_attn.forward(q, k, v, window=4, sinks=-1)
    big = torch.zeros(1, 4, 1, 264, dtype=BF, device=device)
    with pytest.raises(AssertionError):
        window_attn.forward(big, big, big, window=4)
    with pytest.raises(AssertionError):
        window_attn.forward(q, k, v, window=4, out=torch.empty_like(q)[:, ::2])
