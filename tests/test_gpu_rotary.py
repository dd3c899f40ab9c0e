"""apply_rotary against complex multiplication in 64 bits, its gradients and its layouts.

Bound: the angle is exact to 2^-25 turns (its fp32 fraction) and sincospi to 2 half steps, so cos and sin are off by
at most 2 pi 2^-25 + 2^-23 < 4e-7 absolute; two products and a sum in fp32 add 3 * 2^-24 of |a| + |b|; one rounding to
the type, u |y|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _exact(x, pos, freqs, layout, mag, sign=1.0):
    x, rot = x.detach().double(), 2 * freqs.numel()
    ang = sign * pos.double().reshape(pos.shape if pos.dim() == 2 else (1,) + pos.shape)[..., None] * freqs
    c, s = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]
    y, size = x.clone(), torch.zeros_like(x)
    lo, hi = ((slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else
              (slice(0, rot, 2), slice(1, rot, 2)))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = mag * (a * c - b * s), mag * (a * s + b * c)
    size[..., lo] = size[..., hi] = mag * (a.abs() + b.abs())
    return y, size


def _check(got, x, pos, freqs, layout, mag, sign=1.0):
    y, size = _exact(x, pos, freqs, layout, mag, sign)
    u = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tol = u * y.abs() * 1.001 + size * (4e-7 + 4 * 2.0 ** -24) + 2.0 ** -25 * (got.dtype == torch.float16)
    assert ((got.double() - y).abs() <= tol).all(), float(((got.double() - y).abs() - tol).max())
    rot = 2 * freqs.numel()
    assert torch.equal(got[..., rot:], x.detach()[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,s,h,hk,d,rot", [(1, 1, 1, 0, 2, 2), (2, 5, 3, 1, 128, 128), (3, 33, 8, 2, 96, 64),
                                            (1, 700, 2, 2, 80, 48), (2, 9, 5, 5, 34, 30), (16, 1, 32, 8, 128, 128),
                                            (1, 3001, 2, 1, 64, 64)])
def test_values_and_gradients(layout, dtype, b, s, h, hk, d, rot):
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    g = torch.Generator(device="cuda").manual_seed(b * 1000 + s)
    q = torch.randn(b, s, h, d, device="cuda", generator=g).to(dtype).requires_grad_(True)
    k = torch.randn(b, s, hk, d, device="cuda", generator=g).to(dtype).requires_grad_(True) if hk else None
    pos = torch.randint(-5000, 2 ** 20, (b, s), device="cuda", generator=g)
    f = rotary_frequencies(rot)
    out = apply_rotary(q, k, positions=pos, freqs=f, layout=layout, magnitude=1.25)
    out = [out] if k is None else list(out)
    leaves = [q] if k is None else [q, k]
    gs = [torch.randn(o.shape, device="cuda", generator=g).to(dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, gs)
    for x, o, go, dx in zip(leaves, out, gs, grads):
        assert o.dtype == dtype and dx.dtype == dtype
        _check(o.detach(), x, pos, f, layout, 1.25)
        _check(dx, go, pos, f, layout, 1.25, -1.0)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_position_types_and_shared_positions(kind):
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    x = torch.randn(2, 40, 3, 64, device="cuda")
    f = rotary_frequencies(64)
    pos = torch.arange(40, device="cuda").to(kind) * 3
    if kind.is_floating_point:
        pos = pos + 0.25
    _check(apply_rotary(x, positions=pos, freqs=f), x, pos, f, "half", 1.0)
    packed = apply_rotary(x[0], positions=pos, freqs=f)
    _check(packed[None], x[:1], pos, f, "half", 1.0)


def test_fractional_positions_far_out():
    """A position of 10^6 + 1/3 needs more than fp32's 24 bits."""
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    x = torch.randn(1, 1000, 1, 64, device="cuda")
    f = rotary_frequencies(64)
    pos = 1e6 + torch.arange(1000, device="cuda", dtype=torch.float64) / 3
    _check(apply_rotary(x, positions=pos, freqs=f, layout="interleaved"), x, pos, f, "interleaved", 1.0)


def test_strides_in_place_and_inverse():
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    f = rotary_frequencies(64)
    base = torch.randn(2, 3, 50, 66, device="cuda", dtype=torch.bfloat16)
    for x in (base.transpose(1, 2)[..., 1:65], base.transpose(1, 2)[..., :64], base.transpose(1, 2)[:, ::2, :, 2:],
              base.transpose(1, 3)[:, :64].transpose(1, 3)[:, :1].expand(2, 7, 50, 64).transpose(1, 2)):
        pos = torch.arange(x.shape[1], device="cuda", dtype=torch.int32)
        y = apply_rotary(x, positions=pos, freqs=f)
        _check(y, x, pos, f, "half", 1.0)
    qkv = torch.randn(2, 10, 3, 4, 64, device="cuda")
    q, k, v = qkv.unbind(2)
    keep, kv = qkv.clone(), v.clone()
    pos = torch.arange(10, device="cuda")
    rq, rk = apply_rotary(q, k, positions=pos, freqs=f, inplace=True)
    assert rq.data_ptr() == q.data_ptr() and torch.equal(v, kv)
    _check(q, keep[:, :, 0], pos, f, "half", 1.0)
    _check(k, keep[:, :, 1], pos, f, "half", 1.0)
    back = apply_rotary(q.clone(), positions=pos, freqs=f, inverse=True)
    assert (back - keep[:, :, 0]).abs().max() < 1e-5
    with pytest.raises(ValueError):
        apply_rotary(q.clone().requires_grad_(True), positions=pos, freqs=f, inplace=True)
    with pytest.raises(ValueError):
        apply_rotary(q[:, :1].expand(2, 10, 4, 64), positions=pos, freqs=f, inplace=True)


def test_empty_and_agreement_with_the_window_encoder():
    """One sample per window: the heads' rotation equals fd_rope_windows' rows."""
    import numpy as np

    from flashdiffusion_b200.rope import ROPE, apply_rotary, rotary_frequencies
    f = rotary_frequencies(8)
    assert apply_rotary(torch.empty(0, 3, 8, device="cuda"), positions=torch.arange(0, device="cuda"),
                        freqs=f).shape == (0, 3, 8)
    series = np.random.default_rng(0).standard_normal((40, 8))
    enc = ROPE(series, L=1, rank=2, center=False, precision="f16")
    x = torch.as_tensor(series, dtype=torch.float32, device="cuda")[:, None]
    y = apply_rotary(x, positions=torch.arange(40, device="cuda"), freqs=f, layout="interleaved")
    np.testing.assert_allclose(y[:, 0].cpu().numpy(), enc.Y_, atol=3e-6)


def test_gradient_against_differences():
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    f = rotary_frequencies(6)
    x = torch.randn(1, 3, 2, 8, device="cuda", requires_grad=True)
    w = torch.randn(1, 3, 2, 8, device="cuda")
    pos = torch.tensor([0, 5, 11], device="cuda")
    loss = lambda t: (apply_rotary(t, positions=pos, freqs=f, magnitude=1.1) * w).double().sum()  # noqa: E731
    g = torch.autograd.grad(loss(x), x)[0]
    e = torch.randn_like(x)
    # the map is linear: any step is exact up to fp32 rounding of 48 terms of size about 1
    diff = (loss(x.detach() + e) - loss(x.detach() - e)) / 2
    assert abs(float(diff) - float((g * e).double().sum())) < 48 * 2.0 ** -22 * 8


def test_in_place_is_seen_by_autograd_and_refused_twice():
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    x = torch.randn(1, 6, 4, 64, device="cuda")
    pos, f = torch.arange(6, device="cuda"), rotary_frequencies(64)
    w = torch.ones_like(x, requires_grad=True)
    y = w * x                                       # saves x
    with torch.no_grad():
        apply_rotary(x[:, :, :2], x[:, :, 2:], positions=pos, freqs=f, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(ValueError, match="same memory"):
        apply_rotary(x, x, positions=pos, freqs=f, inplace=True)
    with torch.inference_mode():
        z = torch.randn(1, 6, 4, 64, device="cuda")
        want = apply_rotary(z, positions=pos, freqs=f)
        assert torch.equal(apply_rotary(z, positions=pos, freqs=f, inplace=True), want)
