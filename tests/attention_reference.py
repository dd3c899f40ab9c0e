"""Softmax attention over key spans from its definition in 64 bits, with elementwise bounds on a kernel's rounding.

Rounding model (u = half a step of the tensors' type, w = 2^-24):
  scores    summed in fp32 over D products and scaled: within e_s = 2 (D + 8) w |scale| sum |q||k| + 8 w (|s| + 1),
            the tanh and the bias included (both are fp32 evaluations of a few steps, the tanh with slope <= 1;
            a short polynomial or MUFU exponential adds 1e-6 cap)
  weights   p = exp(s - lse) relative to exact: 2 e_s' + 8e-6 (e_s' the row's largest; the exponential itself is
            good to 4e-6, twice for numerator and sum), and rounded once to the tensors' type: u
  output    one rounding, u, of a sum of p v
  ds        p (dp - delta): delta is summed from the rounded output, dp like a score without the scale; rounded: u
Sums of up to n terms in fp32 add 2 n w of their absolute sum; with n <= 4096 here that stays below 5e-4.
"""
import torch

W = 2.0 ** -24


def spans_of(sq, sk, b, causal=False, window=None, first=None, end=None, lengths=None):
    i = torch.arange(sq)
    n = torch.full((b, 1), sk) if lengths is None else lengths.long().clamp(0, sk)[:, None]
    pos = n - sq + i[None]
    if first is not None:
        lo, hi = first.long().expand(b, sq), end.long().expand(b, sq)
    else:
        hi = pos + 1 if causal else n.expand(b, sq)
        lo = (pos - window + 1) if window else torch.zeros_like(pos)
    return lo.clamp(min=0), torch.minimum(hi, n.expand(b, sq)), pos


def reference(q, k, v, lo, hi, pos, scale=None, cap=0.0, slopes=None, do=None):
    """dict of o, lse and, with do, dq, dk, dv (fp64, CPU), and of the bound on each ("o_tol" and so on)."""
    u = torch.finfo(q.dtype).eps / 2
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    do = None if do is None else do.detach().cpu().double()
    out = {n: torch.zeros(B, Sq, H, D, dtype=torch.float64) for n in ("o", "o_tol", "dq", "dq_tol")}
    out |= {n: torch.zeros(B, Sk, Hk, D, dtype=torch.float64) for n in ("dk", "dk_tol", "dv", "dv_tol")}
    out |= {n: torch.zeros(B, H, Sq, dtype=torch.float64) for n in ("lse", "lse_tol")}
    j = torch.arange(Sk)[None, :]
    for b in range(B):
        see = (j >= lo[b].cpu()[:, None]) & (j < hi[b].cpu()[:, None])
        empty = ~see.any(1)
        for h in range(H):
            hk = h * Hk // H
            Q, K, V = q[b, :, h], k[b, :, hk], v[b, :, hk]
            # what lies in masked places must not matter: take it out of the exact products
            seen = see.any(0)
            K, V = torch.where(seen[:, None], K, 0.0), torch.where(seen[:, None], V, 0.0)
            Q = torch.where(empty[:, None], 0.0, Q)
            z = scale * (Q @ K.T)
            es = 2 * (D + 8) * W * abs(scale) * (Q.abs() @ K.abs().T)
            bend = torch.ones_like(z)
            s = z
            if cap:
                t = torch.tanh(z / cap)
                s, bend = cap * t, 1 - t * t
                es = es + 1e-6 * cap
            if slopes is not None:
                s = s - float(slopes[h]) * (pos[b].cpu()[:, None] - j).abs()
            es = es + 8 * W * (s.abs() + z.abs() + 1)
            es = torch.where(see, es, 0.0).amax(1, keepdim=True)
            s = torch.where(see, s, float("-inf"))
            lse = torch.logsumexp(s, 1)
            p = torch.where(see & ~empty[:, None], torch.exp(s - lse[:, None]), 0.0)
            n = float(Sk)
            rel = 2 * es + 8e-6 + 2 * n * W
            o = p @ V
            out["o"][b, :, h] = o
            o_tol = u * o.abs() + (u + rel) * (p @ V.abs()) + 1e-30
            out["o_tol"][b, :, h] = o_tol
            out["lse"][b, h] = lse
            out["lse_tol"][b, h] = (es[:, 0] + 8e-6 + 2 * n * W) + 8 * W * lse.abs().nan_to_num(posinf=0.0)
            if do is None:
                continue
            G = torch.where(empty[:, None], 0.0, do[b, :, h])
            out["dv"][b, :, hk] += p.T @ G
            m = float(Sq * (H // Hk))
            out["dv_tol"][b, :, hk] += (p * (u + rel + 2 * m * W)).T @ G.abs()
            dp = G @ V.T
            dl = (G * o).sum(1, keepdim=True)
            dl_tol = (G.abs() * o_tol).sum(1, keepdim=True) + 2 * D * W * (G * o).abs().sum(1, keepdim=True)
            dp_tol = 2 * (D + 8) * W * (G.abs() @ V.abs().T)
            ds = p * (dp - dl) * bend * scale
            # a type with few exponent bits loses what is below its smallest step of a scaled ds
            ds_tol = abs(scale) * p * bend * ((rel + u) * (dp.abs() + dl.abs()) + dl_tol + dp_tol)
            if cap:
                ds_tol = ds_tol + abs(scale) * p * (dp - dl).abs() * (4e-6 + 2 * es / cap)
            out["dq"][b, :, h] = ds @ K
            out["dq_tol"][b, :, h] = u * out["dq"][b, :, h].abs() + ds_tol @ K.abs() + 2 * n * W * (ds.abs() @ K.abs())
            out["dk"][b, :, hk] += ds.T @ Q
            out["dk_tol"][b, :, hk] += ds_tol.T @ Q.abs() + 2 * m * W * (ds.abs().T @ Q.abs())
    out["dk_tol"] += u * out["dk"].abs()
    out["dv_tol"] += u * out["dv"].abs()
    return out


def check(name, got, ref, floor=0.0):
    """Every element of got within ref[name + "_tol"] (times 1 + 1e-3 for the bounds' own rounding, plus floor)."""
    got, want, tol = got.detach().cpu().double(), ref[name], ref[name + "_tol"] * 1.001 + floor
    same = (got == want)
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), float(((got - want).abs() / tol.clamp(min=1e-300))[bad].max()),
                           got[bad][:4], want[bad][:4], bad.nonzero()[:4])
