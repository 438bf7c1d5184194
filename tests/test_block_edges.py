"""The token block's operators at the edges of what they take: empty and oversized calls, narrow
ranges of a type, what nobody sees, and calls that C makes without Python's checks."""
import ctypes

import pytest
import torch

import block_refs as ref
from triangleops_b200 import _lib, window_attn

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
