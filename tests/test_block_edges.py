"""The token block's operators at the edges of what they take: empty and oversized calls, narrow
ranges of a type, what nobody sees, and calls that C makes without Python's checks."""
import ctypes

import pytest
import torch

import block_refs as ref
from triangleops_b200 import _build, _lib, gated_norm, local_block, rotary, window_attn

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _c(name, *args):
    """The status of a C entry: tensors as their pointers, None as null, lists of int as int64 arrays."""
    def arg(a):
        if a is None or isinstance(a, torch.Tensor):
            return ctypes.c_void_p(_lib.ptr(a))
        if isinstance(a, list):
            return (ctypes.c_int64 * len(a))(*a)
        return ctypes.c_float(a) if isinstance(a, float) else a if not isinstance(a, int) else ctypes.c_int64(a)

    return getattr(_lib.lib(), name)(*map(arg, args))


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_no_queries_in_c(device, dtype):
    """Without queries a C caller has no q, k or v to give: the gradients are zero, nothing is read."""
    B, Nk, H, D = 2, 9, 2, 64
    dk, dv = (torch.full((B, Nk, H, D), float("nan"), dtype=dtype, device=device) for _ in range(2))
    assert _c("tops_window_attn_backward", _lib.dtype_code(dtype), B, 0, Nk, H, H, D, None, None, None, None, None, 3, 0, 0,
              1.0, None, None, None, None, None, None, dk, dv, ctypes.c_void_p(_lib.stream_ptr())) == _lib.OK
    assert not dk.any() and not dv.any()


def test_decode_workspace_of_no_sequences():
    """No division by the number of sequences, whatever the window."""
    need = ctypes.c_int64(-1)
    for window in (1, 4096, 9000, 2**40):
        assert _c("tops_window_attn_decode_workspace_bytes", 0, 10000, 4, 2, 64, window, 0, ctypes.byref(need)) == _lib.OK
        assert need.value == 0


@gpu
def test_decode_of_no_sequences(device):
    k = torch.zeros(0, 10000, 2, 64, dtype=BF, device=device)
    n = torch.zeros(0, dtype=torch.int32, device=device)
    assert window_attn.decode(torch.zeros(0, 4, 64, dtype=BF, device=device), k, k, n, window=9000).shape == (0, 4, 64)


@pytest.mark.parametrize("B,Hq,Hkv,N,D", [(2**32, 1, 1, 1, 8), (2**32 + 1, 1, 1, 1, 8), (1, 2**32, 2**32, 1, 8), (1, 2**31, 1, 1, 8),
                                          (2**31, 1, 1, 1, 64), (1, 2**26, 2**26, 1, 64)])
def test_sizes_past_31_bits_are_refused(B, Hq, Hkv, N, D):
    """The kernels count sequences, and the channels of a token, in 32 bits."""
    t, st, need = torch.zeros(16, dtype=BF), [8] * 9, ctypes.c_int64(0)
    assert _c("tops_window_attn_forward", _lib.BF16, B, N, N, Hq, Hkv, D, t, t, t, st, None, 3, 0, 0, 1.0, t, None,
              None) == _lib.ERR_SHAPE
    assert _c("tops_window_attn_backward", _lib.BF16, B, N, N, Hq, Hkv, D, t, t, t, st, None, 3, 0, 0, 1.0, t, [8] * 3, t, t,
              t, t, t, t, None) == _lib.ERR_SHAPE
    assert _c("tops_window_attn_backward_workspace_bytes", _lib.BF16, B, N, N, Hq, Hkv, D, 3, 0, 0,
              ctypes.byref(need)) == _lib.ERR_SHAPE
    assert _c("tops_window_attn_decode", _lib.BF16, B, N, Hq, Hkv, D, t, t, t, [8] * 8, t, 3, 0, 1.0, None, t,
              None) == _lib.ERR_SHAPE
    assert _c("tops_window_attn_decode_workspace_bytes", B, N, Hq, Hkv, D, 3, 0, ctypes.byref(need)) == _lib.ERR_SHAPE


@gpu
def test_step_without_room(device):
    """Lengths that have no place in the caches: these sequences get NaN, the others what they would
    get, and what the caches hold stays."""
    g = torch.Generator().manual_seed(0)
    pre = local_block.init(64, 4, 2, 16, 96, 2, sections=(4, 4), dtype=FP, device=device, generator=g)
    B, N = 5, 6
    s = torch.randn(B, 64, generator=g).to(device)
    pos = torch.arange(B, dtype=torch.int32, device=device).expand(2, B)
    full = local_block.caches(pre, B, N, dtype=FP, device=device)
    for pair in full:
        for c in pair:
            c.copy_(torch.randn(c.shape, generator=g))
    before = [[c.clone() for c in pair] for pair in full]
    lengths = torch.tensor([N, 3, -1, N - 1, 2**31 - 1], dtype=torch.int32, device=device)
    x, n = local_block.step(s, pre, pos, full, lengths, window=4, sinks=1)
    fit = [1, 3]
    some = [[c[fit] for c in pair] for pair in before]
    x2, n2 = local_block.step(s[fit], pre, pos[:, fit], some, lengths[fit], window=4, sinks=1)
    torch.testing.assert_close(x[fit], x2, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(n[fit], n2, rtol=1e-5, atol=1e-5)
    for b in range(B):
        assert (torch.isfinite if b in fit else torch.isnan)(torch.stack([x[b], n[b]])).all()
    for pair, old in zip(full, before):
        for c, o in zip(pair, old):
            same = (c == o).all(-1).all(-1)  # (B, N)
            for b in range(B):
                assert same[b].tolist() == [b not in fit or t != lengths[b].item() for t in range(N)]


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_store(device, dtype):
    """Any strides of what is stored and of the caches; lengths of either width."""
    g = torch.Generator().manual_seed(1)
    B, N, H, D = 4, 5, 3, 20
    k, v = (torch.randn(B, H, D, generator=g).to(device, dtype) for _ in range(2))
    lengths = torch.tensor([0, N - 1, N, 2], device=device)
    want = [torch.zeros(B, N, H, D, dtype=dtype, device=device) for _ in range(2)]
    for b, n in enumerate(lengths.tolist()):
        if n < N:
            want[0][b, n], want[1][b, n] = k[b], v[b]
    both = torch.zeros(B, N, 2, H, D, dtype=dtype, device=device)
    turned = [torch.zeros(B, D, H, N, dtype=dtype, device=device).permute(0, 3, 2, 1) for _ in range(2)]
    split = torch.cat([k, v], 1)
    for kc, vc, n in ((both[:, :, 0], both[:, :, 1], lengths), (*turned, lengths.int())):
        window_attn.kernel.store(split[:, :H], v.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, n)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_store_refusals():
    k, c, n = torch.zeros(2, 3, 8), torch.zeros(2, 4, 3, 8), torch.zeros(2, dtype=torch.int32)
    store = window_attn.kernel.store
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        store(k, k, c, c, n)
    for bad in ((k, k[:, :2], c, c, n), (k, k, c[:1], c, n), (k, k, c, c[:, :3], n), (k, k, c, c, n[:1]), (k[0], k[0], c, c, n)):
        with pytest.raises(AssertionError):
            store(*bad)
    with pytest.raises(ValueError):
        store(k, k, c.half(), c.half(), n)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,N,H,window,sinks", [(65537, 2, 1, 2, 0), (65540, 3, 2, 1, 1), (8200, 140, 8, 2, 1)])
def test_gradients_of_many_sequences(device, dtype, B, N, H, window, sinks):
    """More sequences than a grid's second and third dimensions count, with and without sinks' late queries."""
    g = torch.Generator(device=device).manual_seed(N)
    q, k, v, d = (torch.randn(B, N, H, 8, device=device, generator=g).to(dtype) for _ in range(4))
    kw = dict(window=window, sinks=sinks)
    out, lse = window_attn.forward(q, k, v, **kw)
    got = dict(zip(("dq", "dk", "dv"), window_attn.backward(d, q, k, v, out, lse, **kw)), out=out)
    rows = torch.tensor([0, 1, B // 2, B - 2, B - 1], device=device)
    want = ref.attention(q[rows], k[rows], v[rows], window, sinks, dout=d[rows])
    for name, t in got.items():
        ref.assert_within(t[rows], *want[name], f"{name} {dtype} {(B, N, H)}")


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("low", [-16.0, -17.0, -20.0])
def test_probabilities_far_below_the_largest(device, dtype, low):
    """A first key that takes nearly all and holds zeros, and some thousand keys e^-16 to e^-20 below
    it that make the result: they count, although f16 has nothing below 2^-24. (Held at 2^8 times its
    size, a probability is off by 2^-33 of the largest at most; one token's at 2^15, by 2^-40.)"""
    N, D = 2048, 64
    g = torch.Generator().manual_seed(7)
    q = torch.ones(1, N, 1, D).to(device, dtype)
    k = torch.full((1, N, 1, D), low / 64).to(device, dtype)  # scores of `low`, exact in either type
    k[:, 0] = 0.0
    v = (1 + torch.rand(1, N, 1, D, generator=g)).to(device, dtype)
    v[:, 0] = 0.0
    want = ref.attention(q, k, v, N, 1, scale=1.0)
    value, bound = want["out"]
    sums = v.double().cumsum(1) if dtype == HF else torch.zeros_like(value)
    out, lse = window_attn.forward(q, k, v, window=N, sinks=1, scale=1.0)
    ref.assert_within(out, value, bound + 2.0**-33 * sums, "out")
    torch.testing.assert_close(lse.double(), want["lse"][0], rtol=1e-5, atol=1e-5)
    # the last query alone, through the one-token form
    n = torch.tensor([N], dtype=torch.int32, device=device)
    one = window_attn.decode(q[:, -1].contiguous(), k, v, n, window=N, sinks=1, scale=1.0)
    ref.assert_within(one, value[:, -1], (bound + 2.0**-40 * sums)[:, -1], "one token")


def _norm_error(got, value):
    return (torch.linalg.vector_norm(got.double() - value) / torch.linalg.vector_norm(value)).item()


@gpu
@pytest.mark.parametrize("N,Nq,Hq,Hkv,D,window,sinks,masked", [(2048, 2048, 2, 1, 64, 512, 4, False),
                                                              (1500, 700, 2, 2, 128, (200, 20), 0, True),
                                                              (1000, 1000, 4, 1, 32, (40, 0), 140, True)])
@pytest.mark.parametrize("dout,v_sd", [(1e-6, 1.0), (1e-4, 1.0), (1e-3, 1.0), (1.0, 1.0), (500.0, 30.0), (1.0, 1e-4)])
def test_f16_gradients_of_any_size(device, dout, v_sd, N, Nq, Hq, Hkv, D, window, sinks, masked):
    """Gradients far below and above 1: f16 products keep their digits. The 2-norm may be off by the
    store and by one 16-bit factor of a product (2^-11 of the value each), and by half of f16's
    smallest step for each element. What masked keys and queries that see nothing hold sizes nothing."""
    g = torch.Generator().manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(1, Nq, Hq, D).to(device, HF), r(1, N, Hkv, D).to(device, HF), (r(1, N, Hkv, D) * v_sd).to(device, HF)
    d = (r(1, Nq, Hq, D) * dout).to(device, HF)
    mask = None
    if masked:
        mask = torch.rand(1, N, generator=g).to(device) < 0.8
        mask[:, -60:] = False
        v = v.masked_fill(~mask[..., None, None], 60000.0)
    want = ref.attention(q, k, v, window, sinks, mask, dout=d)
    kw = dict(window=window, sinks=sinks, mask=mask)
    out, lse = window_attn.forward(q, k, v, **kw)
    for name, got in zip(("dq", "dk", "dv"), window_attn.backward(d, q, k, v, out, lse, **kw)):
        value = want[name][0]
        fits = value.abs() < 65520.0  # what rounds to infinity is infinite
        assert torch.equal(torch.isfinite(got), fits), name
        got, value = got[fits], value[fits]
        off = torch.linalg.vector_norm(got.double() - value).item()
        size = torch.linalg.vector_norm(value).item()
        assert off <= 2.0**-10 * size + 2.0**-25 * value.numel() ** 0.5, (name, off / size)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients_of_q_and_k_lose_only_their_own_rounding(device, dtype):
    """dS enters its products with twice the type's digits: dQ and dK are no farther from the 64-bit
    values than these rounded (one more rounding of that size would add in squares: 1.4 times)."""
    g = torch.Generator().manual_seed(3)
    q, k, v, d = (torch.randn(2, 1024, h, 64, generator=g).to(device, dtype) for h in (4, 2, 2, 4))
    want = ref.attention(q, k, v, 256, 4, dout=d)
    out, lse = window_attn.forward(q, k, v, window=256, sinks=4)
    dq, dk, _ = window_attn.backward(d, q, k, v, out, lse, window=256, sinks=4)
    for name, got in (("dq", dq), ("dk", dk)):
        value = want[name][0]
        assert _norm_error(got, value) <= 1.2 * _norm_error(value.to(dtype), value), name


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("N,D,sinks,window", [(200, 64, 0, (30, 5)), (700, 128, 3, (100, 0)), (130, 32, 1, (8, 8))])
def test_what_a_query_that_sees_nothing_holds(device, dtype, N, D, sinks, window):
    """NaN and infinity in q and in the gradient of queries whose keys are all masked reach nothing."""
    g = torch.Generator().manual_seed(N)
    q, k, v, d = (torch.randn(2, N, h, D, generator=g).to(device, dtype) for h in (4, 2, 2, 4))
    mask = torch.ones(2, N, dtype=torch.bool)
    mask[0, :sinks] = mask[1, :sinks] = False  # (a kept sink is seen by all)
    mask[0, N // 2:] = False
    mask[1, 40:40 + window[0] + window[1] + 9] = False
    mask = mask.to(device)
    see = ref.visible(N, N, *window, sinks, mask, device)[:, 0].any(-1)  # (B, N)
    assert (~see).any(1).all()
    want = ref.attention(q, k, v, window, sinks, mask, dout=d)
    kw = dict(window=window, sinks=sinks, mask=mask)
    gone = ~see[..., None, None]
    q, d = q.masked_fill(gone, float("nan")), d.masked_fill(gone, float("nan"))
    d[..., 1::2] = d[..., 1::2].masked_fill(gone, float("inf"))
    out, lse = window_attn.forward(q, k, v, **kw)
    ref.assert_within(out, *want["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), window_attn.backward(d, q, k, v, out, lse, **kw)):
        ref.assert_within(got, *want[name], f"{name} {dtype}")


def _stand_ins(monkeypatch):
    """The launchers as graph-less functions of the CPU with gradients of the right shapes (the values take no part)."""
    monkeypatch.setattr(window_attn.kernel, "forward", lambda q, k, v, **kw: (q * 2, q.sum(-1)))
    monkeypatch.setattr(window_attn.kernel, "backward", lambda d, q, k, v, o, lse, **kw: (d * 2, k * 0, v * 0))
    monkeypatch.setattr(gated_norm.kernel, "forward", lambda x, y, g, **kw: (x + y, x * 2 if kw["pre_norm"] else None, x))
    monkeypatch.setattr(gated_norm.kernel, "backward", lambda dh, dn, x, y, g, st, **kw: dict(
        dx=x * 2, dy=y * 2, **{"d" + w: t * 1 for w, t in kw.items() if isinstance(t, torch.Tensor)}))
    for f in ("forward", "backward"):
        monkeypatch.setattr(rotary.kernel, f, lambda q, k, pos, **kw: (q * 2, None if k is None else k * 2))


def test_second_derivatives_are_refused(monkeypatch):
    """A gradient of a gradient would lose the terms that run through the first one: an error, whether
    the graph reaches it by the incoming gradient or by the inputs; first gradients are as they were."""
    _stand_ins(monkeypatch)
    x, w = torch.randn(3, 4, requires_grad=True), torch.randn(4, requires_grad=True)
    inv, axis, pos = torch.ones(2), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 1, 3, dtype=torch.int32)
    calls = {
        "window_attention": lambda t: window_attn.window_attention(t, t, t, window=2),
        "gated_norm": lambda t: gated_norm.gated_norm(t, t, post_weight=w)[0],
        "gated_norm without a second norm": lambda t: gated_norm.gated_norm(t, t, pre_norm=False)[0],
        "rotary": lambda t: rotary.rotary(t, None, pos, inv_freq=inv, axis=axis)[0],
    }
    for what, f in calls.items():
        once, = torch.autograd.grad(f(x).square().sum(), x)
        assert not once.requires_grad and once.shape == x.shape
        grad, = torch.autograd.grad(f(x * x).square().sum(), x, create_graph=True)
        assert grad.requires_grad
        with pytest.raises(RuntimeError, match="no second derivatives"):
            torch.autograd.grad(grad.square().sum(), x)
        if what != "rotary":  # (a turn's gradient does not depend on what is turned)
            grad, = torch.autograd.grad(f(x).sum(), x, create_graph=True)
            with pytest.raises(RuntimeError, match="no second derivatives"):
                torch.autograd.grad((grad * grad).sum() + x.sum(), x)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,P", [(1024, 512), (784, 392), (768, 384), (896, 448), (1024, 100)])
def test_rotary_of_one_wide_head(device, dtype, D, P):
    """Many tokens a block of one head: their angles fit the block's shared memory."""
    B, N = 2, 4800
    g = torch.Generator(device=device).manual_seed(D)
    q = torch.randn(B, N, 1, D, device=device, generator=g).to(dtype)
    pos = torch.randint(-500, 500, (1, B, N), device=device, generator=g, dtype=torch.int32)
    inv_freq, axis = rotary.frequencies(D, (P,), device=device)
    got, _ = rotary.forward(q, None, pos, inv_freq=inv_freq, axis=axis)
    value, size = ref.rotary(q, pos, inv_freq, axis, False)
    ref.assert_within(got, value, ref.store(value, dtype) + 2.0**-21 * size, f"{dtype} {D}")


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_lengths_past_32_bits(device, dtype):
    """A 64-bit length counts as what it is, not as its low 32 bits."""
    B, N, D = 5, 40, 32
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(*s, generator=g).to(device, dtype) for s in ((B, 2, D), (B, N, 2, D), (B, N, 2, D)))
    far = torch.tensor([2**32 + 3, 2**40, -(2**32) + 7, 2**31 + 1, 12], device=device)
    near = torch.tensor([N, N, 0, N, 12], dtype=torch.int32, device=device)
    kw = dict(window=16, sinks=1)
    assert torch.equal(window_attn.decode(q, k, v, far, **kw), window_attn.decode(q, k, v, near, **kw))
    old = k.clone(), v.clone()
    window_attn.kernel.store(q, q, k, v, far)
    for c, o in zip((k, v), old):
        o[4, 12] = q[4]
        assert torch.equal(c, o)


@gpu
def test_first_use_of_a_thread_inside_a_capture(device):
    """A thread whose first call of the operators is captured into a graph, as autograd's may be."""
    import threading

    q, k, v, d = (torch.randn(1, 200, 2, 64, device=device).to(BF) for _ in range(4))
    kw = dict(window=64, sinks=1)
    want = window_attn.forward(q, k, v, **kw)
    want = (*want, *window_attn.backward(d, q, k, v, *want, **kw))
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=stream):
                out, lse = window_attn.forward(q, k, v, **kw)
                grads = window_attn.backward(d, q, k, v, out, lse, **kw)
            graph.replay()
            torch.cuda.synchronize()
            got.extend(t.clone() for t in (out, lse, *grads))
            graph.reset()
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not isinstance(got[0], Exception), got
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows_in_c():
    """Zero rows are no error at the gated norm's C entries, and nothing has to be there."""
    need = ctypes.c_int64(-1)
    assert _c("tops_gated_norm_backward_workspace_bytes", 0, 3, 64, ctypes.byref(need)) == _lib.OK and need.value == 0
    none = [None] * 6
    assert _c("tops_gated_norm_forward", _lib.BF16, _lib.BF16, 0, 3, 64, 1, 1, 1, 1e-5, None, 64, None, 64, None, 64, *none[:5],
              None, None, None, None) == _lib.OK
    assert _c("tops_gated_norm_backward", _lib.BF16, _lib.F32, 0, 3, 64, 1, 1, 1, None, 64, None, 64, None, 64, None, 64,
              None, 64, *([None] * 15)) == _lib.OK
    assert _c("tops_window_attn_decode_workspace_bytes", 2, 0, 4, 2, 64, 9000, 0, ctypes.byref(need)) == _lib.OK
    assert need.value == 0


@gpu
def test_no_rows_on_the_device(device):
    w = [torch.full((64,), float("nan"), device=device) for _ in range(5)]
    gate = torch.full((3, 64), float("nan"), dtype=BF, device=device)
    assert _c("tops_gated_norm_backward", _lib.BF16, _lib.F32, 0, 3, 64, 1, 1, 1, None, 64, None, 64, None, 64, None, 64, None,
              64, *([None] * 7), gate, *w, None, ctypes.c_void_p(_lib.stream_ptr())) == _lib.OK
    assert not any(t.any() for t in (gate, *w))
    k = torch.zeros(2, 0, 2, 64, dtype=BF, device=device)
    n = torch.tensor([0, 5], dtype=torch.int32, device=device)
    q = torch.ones(2, 4, 64, dtype=BF, device=device)
    assert not window_attn.decode(q, k, k, n, window=9000).any()
    window_attn.kernel.store(q[:, :2], q[:, 2:], k, k, n)


def test_the_extension_is_of_this_torch(monkeypatch, tmp_path):
    """Another torch or Python than the one that it was compiled against, or none on record: built again."""
    _lib.bind()
    assert not _build.needs_bind()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _build.needs_bind()
    monkeypatch.undo()
    assert not _build.needs_bind()
    monkeypatch.setattr(_build, "BIND_STAMP", str(tmp_path / "none"))
    assert _build.needs_bind()


@pytest.mark.parametrize("B,N,Hq,Hkv,D,left,sinks", [(1, 131072, 4, 1, 128, 1, 8192), (2, 65536, 32, 8, 128, 1, 8192),
                                                     (4, 8192, 16, 4, 64, 511, 4), (1, 2**20, 8, 8, 128, 1023, 128),
                                                     (1, 300, 2, 2, 32, 9, 40)])
def test_backward_workspace_with_sinks(B, N, Hq, Hkv, D, left, sinks):
    """What the header says of it, at 148 SMs: the sinks' parts do not grow with the queries without limit."""
    need = ctypes.c_int64(0)
    assert _c("tops_window_attn_backward_workspace_bytes", _lib.BF16, B, N, N, Hq, Hkv, D, left, 0, sinks,
              ctypes.byref(need)) == _lib.OK
    stats = 2 * B * Hq * (-(-N // 128) * 128 + 64) * 4 + 16
    rows = -(-sinks // 128) * 128  # (whole tiles of sinks)
    parts = B * Hkv * 2 * (1 + Hq // Hkv) * rows * max(64, D) * 4 + 148 * 2**20
    assert stats <= need.value <= stats + parts


@gpu
def test_many_sinks_and_late_queries(device):
    """So many sinks and queries that a block of late queries walks more than its share of a tile's own."""
    B, N, H, D, sinks = 2, 7000, 8, 32, 300
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v, d = (torch.randn(B, N, H, D, device=device, generator=g).to(BF) for _ in range(4))
    kw = dict(window=2, sinks=sinks)
    out, lse = window_attn.forward(q, k, v, **kw)
    grads = window_attn.backward(d, q, k, v, out, lse, **kw)
    at = (slice(1, 2), slice(None), slice(5, 6))
    want = ref.attention(q[at], k[at], v[at], 2, sinks, dout=d[at])
    for name, got in zip(("dq", "dk", "dv"), grads):
        ref.assert_within(got[at], *want[name], name)


def _odd(t):
    """The same values one element off 16 bytes, rows an odd number of elements apart."""
    flat = torch.zeros(t.numel() // t.shape[-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    flat[:, 1:-2] = t.reshape(-1, t.shape[-1])
    return flat[:, 1:-2].view(t.shape)


def _part(t):
    """The same values as a part of wider rows, which 16-byte loads can follow."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 64, dtype=t.dtype, device=t.device)
    wide[..., 32:-32] = t
    return wide[..., 32:-32]


def _channels_first(t):
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


def _one_row(t):
    """Its first row for all, by a stride of zero."""
    return t.reshape(-1, t.shape[-1])[:1].expand(t.numel() // t.shape[-1], t.shape[-1]).view(t.shape)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("C", [128, 771])
@pytest.mark.parametrize("lay", [_odd, _part, _channels_first, _one_row])
@pytest.mark.parametrize("which", ["x", "y", "gate", "dh", "dn", "all"])
def test_gated_norm_strides(device, dtype, C, lay, which):
    """Each input by itself, and all of them, in other strides: values forward and backward. Bounds: the
    store, fp32 arithmetic of 2^-17 of the largest value that takes part, of a root of T such terms in sums."""
    T = 60
    g = torch.Generator().manual_seed(C)
    t = {n: (torch.randn(3, T // 3, C, generator=g) * (2.0 if n == "x" else 1.0)).to(device, dtype)
         for n in ("x", "y", "gate", "dh", "dn")}
    par = {n: (torch.randn(C, generator=g) * 0.2 + (not n.endswith("bias"))).to(device, dtype)
           for n in ("post_weight", "post_bias", "res_scale", "pre_weight", "pre_bias")}
    for n in t:
        if which in (n, "all"):
            t[n] = lay(t[n])
    want = ref.gated_norm(t["x"], t["y"], t["gate"], par, "layer", 1e-5, dh=t["dh"], dn=t["dn"])
    h, n, stats = gated_norm.forward(t["x"], t["y"], t["gate"], **par)
    got = {"h": h, "n": n, **gated_norm.backward(t["dh"], t["dn"], t["x"], t["y"], t["gate"], stats, **par)}
    for name, value in want.items():
        terms = T if name[1:] in par else 1
        size = max(4.0, value.abs().max().item(), *(v.abs().max().item() for v in want.values() if v.dim() > 1))
        ref.assert_within(got[name], value, ref.store(value, dtype) + 2.0**-17 * size * terms**0.5, f"{name} {which}")


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("lay", [_odd, _part, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                                 lambda t: t[:, :1].expand_as(t)])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout", "all"])
def test_window_attention_strides(device, dtype, lay, which):
    """Each input by itself in other strides, with gradients."""
    g = torch.Generator().manual_seed(4)
    t = {n: torch.randn(2, 150, 2 if n in "kv" else 4, 64, generator=g).to(device, dtype) for n in ("q", "k", "v", "dout")}
    for n in t:
        if which in (n, "all"):
            t[n] = lay(t[n])
    q, k, v, d = t.values()
    want = ref.attention(q, k, v, (40, 9), 3, dout=d)
    out, lse = window_attn.forward(q, k, v, window=(40, 9), sinks=3)
    ref.assert_within(out, *want["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), window_attn.backward(d, q, k, v, out, lse, window=(40, 9), sinks=3)):
        ref.assert_within(got, *want[name], name)


def test_flags_without_a_truth_value():
    """An error of the argument's own, not of an interpreter that finds one left behind."""
    both = torch.ones(2)
    q, pos, f, a = torch.zeros(1, 4, 2, 32), torch.zeros(1, 1, 4, dtype=torch.int32), torch.ones(16), torch.zeros(16).int()
    x, w = torch.zeros(4, 64), torch.zeros(4, 4)
    for call in (lambda: rotary.forward(q, None, pos, inv_freq=f, axis=a, interleaved=both),
                 lambda: gated_norm.forward(x, x, post_norm=both), lambda: gated_norm.forward(x, x, pre_norm=both),
                 lambda: gated_norm.backward(x, x, x, x, None, w, post_norm=both)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()


def test_builds_of_two_processes_do_not_share_a_file(monkeypatch, tmp_path):
    """Ranks that start together may all compile: each writes a file of its own and moves it into place whole."""
    import os
    import types

    written = []

    def compiler(cmd, **_):
        written.append(cmd[cmd.index("-o") + 1])
        with open(written[-1], "w") as f:
            f.write(cmd[0])
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    for name in ("LIB_PATH", "BIND_PATH", "BIND_STAMP"):
        monkeypatch.setattr(_build, name, str(tmp_path / name))
    monkeypatch.setattr(_build.subprocess, "run", compiler)
    for pid in (11, 12):
        monkeypatch.setattr(os, "getpid", lambda pid=pid: pid)
        _build.build(force=True)
        _build.build_bind(force=True)
    assert len(set(written)) == 4
    assert sorted(os.listdir(tmp_path)) == ["BIND_PATH", "BIND_STAMP", "LIB_PATH"]
