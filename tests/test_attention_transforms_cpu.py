"""Derivatives and records that a call of the kernels would drop: refused, not lost (no GPU: the library is stubbed)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from flashdiffusion_b200 import attention, native, rope

Q, K, V = (torch.randn(1, 8, 2, 16) for _ in range(3))
POS, FREQS, LENGTHS = torch.arange(8.0), torch.ones(8, dtype=torch.float64), torch.tensor([8], dtype=torch.int32)
SLOPES = torch.ones(2)

CALLS = {
    "attend-q": (Q, lambda x: attention.attend(x, K, V)),
    "attend-k": (K, lambda x: attention.attend(Q, x, V)),
    "attend-v": (V, lambda x: attention.attend(Q, K, x)),
    "attend-slopes": (SLOPES, lambda x: attention.attend(Q, K, V, slopes=x)),
    "cached": (Q, lambda x: attention.attend_cached(x, K, V, LENGTHS)),
    "rotary-q": (Q, lambda x: rope.apply_rotary(x, K, positions=POS, freqs=FREQS)[0]),
    "rotary-k": (K, lambda x: rope.apply_rotary(Q, x, positions=POS, freqs=FREQS)[1]),
    "rotary-positions": (POS, lambda x: rope.apply_rotary(Q, positions=x, freqs=FREQS)),
    "rotary-in-place": (Q, lambda x: rope.apply_rotary(x, positions=POS, freqs=FREQS, inplace=True)),
}


@pytest.fixture(autouse=True)
def stub(monkeypatch):
    class Library:
        def __getattr__(self, name):
            return lambda *args: native.FD_OK

    monkeypatch.setattr(native, "require_device", lambda device=None: torch.device("cpu"))
    monkeypatch.setattr(native, "load", lambda: Library())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    x, f = CALLS[name]
    with fwd.dual_level():
        before = x.clone()
        d = fwd.make_dual(before, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(d)
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            f(d)
        assert torch.equal(before, x)
        f(x.clone())                                   # no tangent: not refused for the level alone
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


def test_tangents_of_an_incoming_gradient_are_refused():
    for f in (lambda x: attention.attend(x, K, V), lambda x: rope.apply_rotary(x, positions=POS, freqs=FREQS)):
        leaf = Q.clone().requires_grad_(True)
        o = f(leaf)
        with fwd.dual_level():
            g = fwd.make_dual(torch.ones_like(o), torch.ones_like(o))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(o, leaf, g)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    x, f = CALLS[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(f, x.clone(), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(f)(x.clone())


@pytest.mark.filterwarnings("ignore")
def test_tracing_of_spans_is_refused():
    for f in (lambda x: attention.document_spans(x, 8).end, lambda x: attention.prefix_spans(x, 8).end):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, torch.tensor([0, 8], dtype=torch.int32), check_trace=False)
