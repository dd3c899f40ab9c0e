"""Refusals of the attention and rotary operators, and their host-side parts (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from flashdiffusion_b200 import attention, native, rope


def _heads(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("bad", [
    dict(q=_heads(2, 8, 4, 64, dtype=torch.float64)),
    dict(q=_heads(2, 8, 4, 64, dtype=torch.float16)),
    dict(q=_heads(8, 4, 64)),
    dict(q=_heads(3, 8, 4, 64)),
    dict(q=_heads(2, 8, 3, 64)),
    dict(q=_heads(2, 8, 4, 32)),
    dict(v=_heads(2, 7, 2, 64)),
    dict(q=_heads(2, 8, 4, 264), k=_heads(2, 8, 2, 264), v=_heads(2, 8, 2, 264)),
    dict(scale=float("nan")), dict(cap=-1.0), dict(cap=1e-9), dict(cap=float("inf")),
    dict(window=0, causal=True), dict(window=4),
    dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4, dtype=torch.float64)),
    dict(slopes=torch.zeros(4, requires_grad=True)),
], ids=str)
def test_attend_refuses(bad):
    args = dict(q=_heads(2, 8, 4, 64), k=_heads(2, 8, 2, 64), v=_heads(2, 8, 2, 64)) | bad
    with pytest.raises((ValueError, TypeError, RuntimeError)) as e:
        attention.attend(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    assert "no CUDA" not in str(e.value) or "window" in bad     # refused for what it is, not for the missing device


def test_attend_without_a_gpu_raises():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    with pytest.raises(RuntimeError, match="B200"):
        attention.attend(_heads(1, 8, 4, 64), _heads(1, 8, 2, 64), _heads(1, 8, 2, 64))
    with pytest.raises(RuntimeError, match="B200"):
        rope.apply_rotary(_heads(1, 8, 4, 64), positions=torch.arange(8), freqs=torch.ones(32, dtype=torch.float64))


def test_spans_refuse():
    i32 = dict(dtype=torch.int32)
    with pytest.raises(TypeError):
        attention.Spans(torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError):
        attention.Spans(torch.zeros(4, **i32), torch.zeros(5, **i32))
    with pytest.raises(TypeError):
        attention.document_spans(torch.zeros(3), 10)
    with pytest.raises(TypeError):
        attention.prefix_spans(torch.zeros(2, 2, **i32), 10)


def test_packed_arguments_are_the_c_structures():
    """The packers and the ctypes structures lay the same values out the same way."""
    a = native.AttentionArgs()
    values = list(range(1, 100))
    flat = []
    for name, kind in native.AttentionArgs._fields_:
        n = 3 if kind is native._L3 else 1
        take, values = values[:n], values[n:]
        setattr(a, name, native._L3(*take) if n > 1 else (float(take[0]) if kind is ctypes.c_double else take[0]))
        flat += [float(x) if kind is ctypes.c_double else x for x in take]
    assert native.PACK_ATTENTION(*flat) == bytes(a)
    r, values, flat = native.RotaryArgs(), list(range(1, 100)), []
    for name, kind in native.RotaryArgs._fields_:
        n = {native._L3: 3, native._L2: 2}.get(kind, 1)
        take, values = values[:n], values[n:]
        setattr(r, name, kind(*take) if n > 1 else (float(take[0]) if kind is ctypes.c_double else take[0]))
        flat += [float(x) if kind is ctypes.c_double else x for x in take]
    assert native.PACK_ROTARY(*flat) == bytes(r)


def _args(**kw):
    n = 4096
    a = native.AttentionArgs(q=n, k=n, v=n, o=n, scale=1.0, cap=0.0, dtype=native.DTYPE_BF16, batch=1, q_len=8,
                             k_len=8, heads=4, kv_heads=2, dim=64)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("bad", [
    dict(dtype=native.DTYPE_F64), dict(batch=-1), dict(q_len=-1), dict(k_len=-2), dict(dim=0), dict(dim=257),
    dict(kv_heads=3), dict(kv_heads=0), dict(heads=0), dict(batch=70000), dict(heads=65536 * 2), dict(o_low=4100), dict(scale=float("nan")), dict(cap=-1.0),
    dict(cap=float("nan")), dict(first=4096), dict(end=4096), dict(window=-1), dict(window=3),
    dict(first=4096, end=4096, causal=1), dict(q=None), dict(k=None), dict(o=None), dict(q_len=(1 << 30) + 1),
], ids=str)
def test_c_entry_refuses_before_any_launch(bad):
    lib = native.load()
    a = _args(**bad)
    assert lib.fd_attention_forward(ctypes.byref(a), None, 0, None) == native.FD_ERR_ARG
    assert b"fd_attention" in lib.fd_last_error()
    assert lib.fd_attention_backward(ctypes.byref(a), None, 0, None) == native.FD_ERR_ARG


def test_c_entries_check_workspace_and_gradients():
    lib = native.load()
    a = _args()
    assert lib.fd_attention_backward(ctypes.byref(a), None, 0, None) == native.FD_ERR_ARG      # no d_o, lse
    a = _args(d_o=4096, dq=4096, dk=4096, dv=4096, lse=4096)
    assert lib.fd_attention_workspace_bytes(ctypes.byref(a), 1) >= 4 * 8 * 4
    assert lib.fd_attention_backward(ctypes.byref(a), None, 0, None) == native.FD_ERR_WORKSPACE
    big = lib.fd_attention_workspace_bytes(ctypes.byref(a), 1)
    assert lib.fd_attention_backward(ctypes.byref(a), ctypes.c_void_p(4100), big, None) == native.FD_ERR_ARG
    assert lib.fd_attention_forward(None, None, 0, None) == native.FD_ERR_ARG
    assert lib.fd_attention_workspace_bytes(None, 0) == 0
    assert lib.fd_attention_document_spans(None, 1, None, 8, 1, 0, None, None, None) == native.FD_ERR_ARG
    assert lib.fd_attention_document_spans(ctypes.c_void_p(4096), 1, None, 8, 0, 3, None, None, None) == native.FD_ERR_ARG
    assert lib.fd_attention_prefix_spans(None, 1, 4, 4, None, None, None) == native.FD_ERR_ARG
    assert lib.fd_attention_prefix_spans(None, 70000, 4, 4, None, None, None) == native.FD_ERR_ARG
    # nothing to do is not an error
    empty = _args(batch=0)
    assert lib.fd_attention_forward(ctypes.byref(empty), None, 0, None) == native.FD_OK


def test_rotary_c_entry_refuses_very_wide_heads():
    lib = native.load()
    a = native.RotaryArgs(q=4096, qo=4096, positions=4096, freqs=4096, magnitude=1.0, dtype=native.DTYPE_BF16,
                          position_dtype=native.DTYPE_I64, batch=1, tokens=4, heads=2, dim=4098, rot=64)
    assert lib.fd_rotary(ctypes.byref(a), None) == native.FD_ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(rot=3), dict(rot=0), dict(rot=66), dict(layout=2), dict(position_dtype=native.DTYPE_F16),
    dict(dtype=native.DTYPE_F64), dict(tokens=-1), dict(q=None), dict(positions=None), dict(freqs=None),
    dict(kv_heads=2),
], ids=str)
def test_rotary_c_entry_refuses(bad):
    lib = native.load()
    n = 4096
    a = native.RotaryArgs(q=n, qo=n, positions=n, freqs=n, magnitude=1.0, dtype=native.DTYPE_BF16,
                          position_dtype=native.DTYPE_I64, batch=1, tokens=4, heads=2, dim=64, rot=64)
    for name, x in bad.items():
        setattr(a, name, x)
    assert lib.fd_rotary(ctypes.byref(a), None) == native.FD_ERR_ARG
    assert b"fd_rotary" in lib.fd_last_error()


@pytest.mark.parametrize("bad", [
    dict(q=_heads(2, 8, 4, 64, dtype=torch.float64)), dict(k=_heads(2, 7, 4, 64)), dict(k=_heads(2, 8, 4, 32)),
    dict(layout="pairs"), dict(freqs=torch.ones(33, dtype=torch.float64)), dict(freqs=torch.ones(32)),
    dict(positions=torch.zeros(8, dtype=torch.float16)), dict(positions=torch.zeros(7, dtype=torch.int64)),
    dict(magnitude=float("inf")), dict(positions=torch.zeros(8, dtype=torch.float64, requires_grad=True)),
    dict(freqs=torch.zeros(0, dtype=torch.float64)),
], ids=str)
def test_apply_rotary_refuses(bad):
    args = dict(q=_heads(2, 8, 4, 64), k=None, positions=torch.arange(8), freqs=torch.ones(32, dtype=torch.float64)) | bad
    with pytest.raises((ValueError, TypeError)):
        rope.apply_rotary(args.pop("q"), args.pop("k"), **args)


@pytest.mark.parametrize("bad", [dict(rot=5), dict(rot=8, factor=2.0), dict(rot=8, scaling="parts", factor=2.0),
                                 dict(rot=8, scaling="more"), dict(rot=2, scaling="base", factor=2.0),
                                 dict(rot=8, base=-1.0), dict(rot=8, scaling="linear", factor=0.5)], ids=str)
def test_rotary_frequencies_refuse(bad):
    with pytest.raises(ValueError):
        rope.rotary_frequencies(**bad)


def test_rotary_frequencies_values(monkeypatch):
    monkeypatch.setattr(native, "require_device", lambda device=None: torch.device("cpu"))
    f = rope.rotary_frequencies(64).numpy()
    np.testing.assert_allclose(f, 10000.0 ** (-np.arange(32) / 32), rtol=1e-14)
    np.testing.assert_allclose(rope.rotary_frequencies(64, scaling="linear", factor=4.0).numpy(), f / 4, rtol=1e-14)
    g = rope.rotary_frequencies(64, scaling="base", factor=4.0).numpy()
    assert g[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 4, rel=1e-12) and np.all(np.diff(g / f) < 0)
    p = rope.rotary_frequencies(64, scaling="parts", factor=8.0, trained=4096).numpy()
    turns = 4096 * f / (2 * np.pi)
    np.testing.assert_array_equal(p[turns >= 32], f[turns >= 32])
    np.testing.assert_allclose(p[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    assert np.all(np.diff(p) < 0)
    assert rope.rotary_magnitude(1.0) == 1.0
