"""Workspace sizes of the attention entry points, asked on the host (no GPU)."""
import ctypes

import pytest

from flashdiffusion_b200 import native


def _bytes(backward, **kw):
    n = 4096                     # no pointer is read
    a = native.AttentionArgs(q=n, k=n, v=n, o=n, d_o=n, dq=n, dk=n, dv=n, lse=n, scale=1.0, cap=0.0,
                             dtype=native.DTYPE_BF16, batch=1, q_len=8, k_len=8, heads=4, kv_heads=2, dim=64)
    for name, x in kw.items():
        setattr(a, name, x)
    return native.load().fd_attention_workspace_bytes(ctypes.byref(a), backward)


SIZES = [(1, 2048, 2048, 16, 4, 128), (1, 2048, 2048, 4, 1, 128), (1, 4096, 4096, 8, 2, 128), (1, 1024, 1024, 32, 8, 128),
         (1, 1900, 1900, 8, 4, 128), (1, 7900, 7900, 4, 1, 64), (2, 200, 16384, 2, 1, 64), (1, 3000, 140, 2, 2, 64),
         (1, 512, 16384, 8, 2, 256), (1, 4, 9000, 8, 2, 128), (3, 77, 77, 4, 4, 96)]


@pytest.mark.parametrize("dtype", [native.DTYPE_BF16, native.DTYPE_F16, native.DTYPE_F32])
@pytest.mark.parametrize("b,sq,sk,h,hk,d", SIZES)
def test_a_window_that_reaches_every_key_is_no_window(b, sq, sk, h, hk, d, dtype):
    """Sized as the kernels are launched: a window of at least q_len + k_len keys is taken for none there."""
    kw = dict(batch=b, q_len=sq, k_len=sk, heads=h, kv_heads=hk, dim=d, dtype=dtype, causal=1)
    for backward in (0, 1):
        want = _bytes(backward, **kw)
        for window in (sq + sk, sq + sk + 1, 2 * (sq + sk), 2 ** 31 - 1):
            assert _bytes(backward, window=window, **kw) == want, (backward, window)


def test_sizes_are_for_these_calls():
    """The first size above is one whose gradients are cut into parts: their fp32 sums are in the workspace."""
    whole = _bytes(1, q_len=2048, k_len=2048, heads=16, kv_heads=4, dim=128, causal=1)
    assert whole >= 2 * 2 * 4 * 2048 * 4 * 128
