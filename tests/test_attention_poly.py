"""The polynomials compiled into the attention and rotary kernels, in fp32 Horner arithmetic on the host: their stated
errors, and how near they come to a least-squares fit of their degree on Chebyshev nodes.  CPU only."""
import os
import re

import numpy as np

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashdiffusion_b200", "csrc")
F32 = np.float32


def _source(name, start, end):
    text = open(os.path.join(CSRC, name)).read()
    text = text[text.index(start):]
    return text[:text.index(end)]


def _numbers(text):
    return [float(x) for x in re.findall(r"-?\d+\.\d+(?=f\b)", text)]


def _horner(coefficients, y):
    """fmaf from the highest coefficient down: one rounding a step."""
    p = np.full_like(y, F32(coefficients[-1]))
    for c in coefficients[-2::-1]:
        p = (p.astype(np.float64) * y + np.float64(F32(c))).astype(F32)
    return p


def _times(p, x):
    return (p.astype(np.float64) * x).astype(F32)


def _fit_error(f, powers, reach):
    """Largest error of the least-squares fit of these powers on 4000 Chebyshev nodes."""
    x = reach * np.cos(np.pi * (np.arange(4000) + 0.5) / 4000)
    x = x[x > 0]
    a = np.stack([x ** k for k in powers], 1)
    return np.abs(a @ np.linalg.lstsq(a, f(x), rcond=None)[0] - f(x)).max()


def test_tanh():
    text = _source("fd_attn_tc.cuh", "b0 = ptx::both2(", "shrink =")
    c = [_numbers(line)[0] for line in text.splitlines() if "both2(" in line]
    assert len(c) == 4
    u = np.linspace(-0.45, 0.45, 400001).astype(F32)
    t = _times(_horner(c, _times(u, u)), u)
    exact = np.tanh(u.astype(np.float64))
    error = np.abs(t - exact)
    assert error.max() < 9.1e-8
    # towards zero it is the product itself, to the first coefficient's distance from one and a rounding
    assert (error <= (1e-6 + 3 * 2.0 ** -24) * np.abs(exact) + 1e-30).all()
    # the fit's own error is a third of the bound: the rest are fp32 steps
    assert error.max() < 4 * _fit_error(np.tanh, (1, 3, 5, 7), 0.45) + 3 * 2.0 ** -25


def test_what_is_left_of_the_tanh_where_coefficients_are_lost():
    """The limits on |c s| where the highest coefficients leave the normal numbers: the rest is good to 1e-8 there."""
    text = _source("fd_attn_tc.cuh", "const float flat", ";")
    at = _numbers(text)
    assert at == [0.45, 0.1, 0.037, 0.003]
    steps = [float(x) for x in re.findall(r"flat >= (\d+e-\d+)f", text)]
    assert steps == [2e-5, 2e-7, 1e-11]
    c = [1.0, 1 / 3, 2 / 15, 17 / 315]
    for k, (u, flat) in enumerate(zip(at[1:], steps)):
        lost = 3 - k                                            # the coefficient that may go below this slope
        assert c[lost] * u ** (2 * lost + 1) < 1e-8
        # and above it, it is a normal number, as are the powers on the way to it, for the smallest cap, 1e-3
        assert 0.04 * flat ** (2 * lost + 1) * min(1.0, 1e-3 * 1.44) > 2.0 ** -126


def test_sine_and_cosine():
    text = _source("fd_rotary.cu", "const float s = h * fmaf", "const float a = k & 1")
    sine, cosine = (_numbers(line)[::-1] for line in text.strip().splitlines())
    # the multiplications' order in the source: highest first
    assert len(sine) == 4 and len(cosine) == 4 and cosine[0] == 1.0
    rng = np.random.default_rng(0)
    quarter = np.concatenate([rng.uniform(-1e6, 1e6, 400000), np.linspace(-2, 2, 40001)])
    near = np.rint(quarter)
    rest = quarter - near
    h = rest.astype(F32)
    y = _times(h, h)
    s, c = _times(_horner(sine, y), h), _horner(cosine, y)
    k = near.astype(np.int64) & 3
    sin = np.choose(k, [s, c, -s, -c])
    cos = np.choose(k, [c, -s, -c, s])
    for got, want in ((sin, np.sin(np.pi / 2 * (rest + k))), (cos, np.cos(np.pi / 2 * (rest + k)))):
        error = np.abs(got - want)
        assert error.max() < 1.1e-7 and (error ** 2).mean() ** 0.5 < 3.2e-8
    assert _fit_error(lambda x: np.sin(np.pi / 2 * x), (1, 3, 5, 7), 0.5) < 4e-8
    assert _fit_error(lambda x: np.cos(np.pi / 2 * x) - 1, (2, 4, 6), 0.5) < 8e-8


def test_the_exponential_is_the_tile_kernels():
    """exp2_fma2 has the coefficients of exp2_poly2, whose fit and error are tested beside the tile kernels."""
    pick = lambda text: [x for x in _numbers(text) if x not in (12582912.0, 125.0, -125.0)]  # noqa: E731
    mine = pick(_source("fd_attn_tc.cuh", "uint64_t exp2_fma2", "unpack2"))
    tile = pick(_source("fd_tc_common.cuh", "uint64_t exp2_poly2", "unpack2"))
    assert len(mine) == 5 and mine == sorted(set(tile), key=tile.index)
