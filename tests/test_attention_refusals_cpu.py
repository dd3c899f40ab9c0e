"""Calls of attend and attend_cached whose constants leave fp32 are refused (no GPU)."""
import ctypes

import pytest
import torch

from flashdiffusion_b200 import attention, native

BAD = [dict(cap=1e19), dict(cap=3e38), dict(cap=1e300), dict(cap=9e-4), dict(scale=1e31), dict(scale=-1e39),
       dict(scale=float("inf"))]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_python(bad):
    q, k = torch.zeros(2, 8, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16)
    name = next(iter(bad))
    with pytest.raises(ValueError, match=name):
        attention.attend(q, k, k, **bad)
    with pytest.raises(ValueError, match=name):
        attention.attend_cached(q, k, k, torch.ones(2, dtype=torch.int32), **bad)


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_c(bad):
    n = 4096
    a = native.AttentionArgs(q=n, k=n, v=n, o=n, scale=1.0, cap=0.0, dtype=native.DTYPE_BF16, batch=1, q_len=8, k_len=8,
                             heads=4, kv_heads=2, dim=64)
    for name, x in bad.items():
        setattr(a, name, x)
    lib = native.load()
    assert lib.fd_attention_forward(ctypes.byref(a), None, 0, None) == native.FD_ERR_ARG
    assert next(iter(bad)).encode() in lib.fd_last_error()
