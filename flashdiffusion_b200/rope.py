"""RoPE-DMAP encoder on Hankel windows (reference ``FD/ROPE.py``), on the GPU.

The reference builds the dense K x K Gram, distance and kernel matrices of the
rotated window vectors and hands the dense symmetric operator to ARPACK.  Here
the rotation is a per-row preprocessing kernel (``fd_rope_windows``: Hankel
windows read in place from the series, centred, pairs rotated in fp64) and
everything after it is the existing never-materialised operator:

  fit     : rotated windows Y -> DiffusionMap(beta, alpha).fit(Y) (two prepasses:
            q = K 1, d = (K q^-alpha) q^-alpha) -> device Lanczos on
            d^-1/2 K_alpha d^-1/2 = diag(rscale) K diag(rscale) -> psi = d^-1/2 phi
  encode  : rotated query windows -> two Q != K prepasses (row sums, then with
            the training weights q_T^-alpha) -> one block pass with
            V = psi / lambda (the Nystrom formula of ``FD/ROPE.py:489-526``)

``G_`` and ``Kmat_`` (dense K x K in the reference) are never formed and are
None here; every other learned attribute keeps its name and meaning.  The
+1e-18 guards of the reference are kept where they change a result (row sums
of far query windows).

``apply_rotary`` is the same rotation for the query and key heads of a learned
model: 16- or 32-bit tensors, adjacent or split pairs, part of the head,
frequencies scaled for long contexts (``rotary_frequencies``), with gradients.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from . import native
from .dmap import DiffusionMap
from .kernel import GaussianOperator

__all__ = ["ROPE", "make_hankel_windows", "make_window_positions", "apply_rotary", "rotary_frequencies",
           "rotary_magnitude"]

_WINDOW_POSITION = {"start": 0, "center": 1, "end": 2}


def make_hankel_windows(F_tX, L: int, step: int = 1) -> np.ndarray:
    """(K, L, D) Hankel windows W[T, c] = F[T + c step], K = N - (L-1) step (``FD/ROPE.py:31-57``)."""
    F = np.asarray(F_tX, dtype=float)
    if F.ndim == 1:
        F = F[:, None]
    L, step = int(L), int(step)
    if L <= 0:
        raise ValueError("L must be positive.")
    if step <= 0:
        raise ValueError("step must be positive.")
    K = F.shape[0] - (L - 1) * step
    if K <= 0:
        raise ValueError(f"Need N={F.shape[0]} >= (L-1)*step+1 = {(L - 1) * step + 1}")
    idx = np.arange(K)[:, None] + step * np.arange(L)[None, :]
    return F[idx]


def make_window_positions(sample_positions, L: int, step: int = 1, mode: str = "sample",
                          window_position: str = "end") -> np.ndarray:
    """(K, L) sample positions, or (K,) one per window (``FD/ROPE.py:60-106``)."""
    pos = np.asarray(sample_positions, dtype=float)
    if pos.ndim != 1:
        raise ValueError("sample_positions must be one-dimensional.")
    K = len(pos) - (L - 1) * step
    if K <= 0:
        raise ValueError("Not enough positions for windows.")
    P = pos[np.arange(K)[:, None] + step * np.arange(L)[None, :]]
    if mode == "sample":
        return P
    if mode != "window":
        raise ValueError("mode must be 'sample' or 'window'.")
    if window_position not in _WINDOW_POSITION:
        raise ValueError("window_position must be 'start', 'center', or 'end'.")
    return P[:, (0, L // 2, L - 1)[_WINDOW_POSITION[window_position]]]


class ROPE:
    """RoPE-DMAP encoder (``FD/ROPE.py:109-590``); fits on construction like the reference.

    Extra keyword ``precision`` selects the operator tiles ("ramp": 16-bit then
    fp32-class Lanczos stage, the default; "f16", "fp32", "f16x3").
    """

    def __init__(self, F_tX, L: int, rank: int = 20, beta: float | None = None, alpha: float = 1.0,
                 center: bool = True, scale: bool = False, drop_first: bool = True, step: int = 1,
                 sample_positions=None, rope_mode: str = "sample", window_position: str = "end",
                 pos_scale: float = 1.0, base: float = 10000.0, freqs=None, n_freqs: int | None = None,
                 beta_sample_pairs: int = 20000, seed: int = 0, precision: str = "ramp"):
        R = np.asarray(F_tX, dtype=float)
        if R.ndim == 1:
            R = R[:, None]
        self.center, self.scale = bool(center), bool(scale)
        self.mu_ = R.mean(axis=0, keepdims=True) if self.center else np.zeros((1, R.shape[1]))
        sd = R.std(axis=0, keepdims=True) if self.scale else np.ones((1, R.shape[1]))
        self.sigma_ = np.where(sd == 0, 1.0, sd)
        self.R_raw_ = R
        self.R_ = (R - self.mu_) / self.sigma_
        self.N_, self.D_ = R.shape
        self.L, self.step = int(L), int(step)
        self.K_ = self.N_ - (self.L - 1) * self.step
        if self.K_ <= 0:
            raise ValueError(f"N={self.N_} too small for L={self.L}, step={self.step}")
        self.rank_req_ = int(rank)
        self.beta_in_ = beta
        self.alpha_ = float(alpha)
        self.drop_first_ = bool(drop_first)
        if rope_mode not in ("sample", "window"):
            raise ValueError("rope_mode must be 'sample' or 'window'.")
        if window_position not in _WINDOW_POSITION:
            raise ValueError("window_position must be 'start', 'center', or 'end'.")
        self.rope_mode_ = rope_mode
        self.window_position_ = window_position
        self.pos_scale_ = float(pos_scale)
        self.base_ = float(base)
        self.freqs_in_ = None if freqs is None else np.asarray(freqs, dtype=float)
        self.n_freqs_ = None if n_freqs is None else int(n_freqs)
        if sample_positions is None:
            sample_positions = np.arange(self.N_, dtype=float)
        self.sample_positions_ = np.asarray(sample_positions, dtype=float)
        if self.sample_positions_.shape != (self.N_,):
            raise ValueError(f"sample_positions must have shape ({self.N_},).")
        self.beta_sample_pairs_ = int(beta_sample_pairs)
        self.rng_ = np.random.default_rng(int(seed))
        self.precision = precision
        self.G_ = None          # dense Gram: never formed
        self.Kmat_ = None       # dense kernel: never formed
        self.W_TcX_ = None
        self.Pos_ = None
        self.beta_ = self.lam_ = self.phi_ = self.psi_ = self.freqs_ = None
        self.K_T_ = self.d_T_ = self.inv_sqrt_d_ = self.r2_T_ = None
        self.dm_ = None
        self.fit()

    # ---- RoPE internals ---------------------------------------------------------
    def _freqs(self, dim: int) -> np.ndarray:
        """Frequency of each adjacent pair (``FD/ROPE.py:231-259``)."""
        n_pairs = dim // 2
        if n_pairs == 0:
            return np.zeros((0,))
        if self.freqs_in_ is not None:
            f = self.freqs_in_[:n_pairs]
            return np.concatenate([f, np.zeros(n_pairs - f.size)]) if f.size < n_pairs else f
        m = np.arange(n_pairs, dtype=float)
        f = self.base_ ** (-2.0 * m / max(2, 2 * n_pairs))
        if self.n_freqs_ is not None:
            f = f * (np.arange(n_pairs) < max(0, min(self.n_freqs_, n_pairs)))
        return f

    def _rotate(self, F, sT, sC, pos, pT, pC, K) -> torch.Tensor:
        """fd_rope_windows on device copies of F (raw, uncentred) and the positions."""
        dev = native.require_device()
        L, D = self.L, self.D_
        freqs = self._freqs(D if self.rope_mode_ == "sample" else L * D)
        self.freqs_ = freqs
        if self.pos_scale_ == 0.0:
            freqs = np.zeros(0)
        Fd = torch.as_tensor(np.ascontiguousarray(F, dtype=np.float64), device=dev)
        Pd = torch.as_tensor(np.ascontiguousarray(pos, dtype=np.float64), device=dev)
        fd_ = torch.as_tensor(np.ascontiguousarray(freqs, dtype=np.float64), device=dev)
        mu = torch.as_tensor(self.mu_.ravel(), dtype=torch.float64, device=dev)
        sg = torch.as_tensor(self.sigma_.ravel(), dtype=torch.float64, device=dev)
        Y = torch.empty((K, L * D), dtype=torch.float32, device=dev)
        c_w = (0, L // 2, L - 1)[_WINDOW_POSITION[self.window_position_]]
        native.check(native.load().fd_rope_windows(
            native._ptr(Fd), sT, sC, native._ptr(Pd), pT, pC, K, D, L, 1 if self.rope_mode_ == "window" else 0,
            c_w, self.pos_scale_, native._ptr(fd_) if freqs.size else None, int(freqs.size), native._ptr(mu),
            native._ptr(sg), native._ptr(Y), native._stream(dev)))
        return Y

    def _choose_beta(self, Y: torch.Tensor) -> float:
        """Median rule on seeded off-diagonal pairs, beta = 1/(median + 1e-12) (``FD/ROPE.py:347-369``)."""
        if self.beta_in_ is not None:
            return float(self.beta_in_)
        K = self.K_
        M = min(self.beta_sample_pairs_, K * (K - 1) // 2)
        if M <= 0:
            return 1.0
        ii = self.rng_.integers(0, K, size=M)
        jj = self.rng_.integers(0, K, size=M)
        keep = ii != jj
        ii, jj = ii[keep], jj[keep]
        if ii.size == 0:
            return 1.0
        a = torch.as_tensor(ii, device=Y.device)
        b = torch.as_tensor(jj, device=Y.device)
        d2 = ((Y[a].double() - Y[b].double()) ** 2).sum(1).cpu().numpy()
        return 1.0 / (np.median(d2) + 1e-12)

    # ---- training -----------------------------------------------------------------
    def fit(self) -> "ROPE":
        D, L, step = self.D_, self.L, self.step
        self.Pos_ = make_window_positions(self.sample_positions_, L, step, self.rope_mode_, self.window_position_)
        # windows read in place from the raw series (the kernel centres them)
        if self.rope_mode_ == "sample":
            Y = self._rotate(self.R_raw_, D, step * D, self.sample_positions_, 1, step, self.K_)
        else:
            c_w = (0, L // 2, L - 1)[_WINDOW_POSITION[self.window_position_]]
            Y = self._rotate(self.R_raw_, D, step * D, self.sample_positions_[c_w * step:], 1, 0, self.K_)
        self._Y = Y
        self.r2_T_ = (Y.double() ** 2).sum(1).cpu().numpy()
        self.beta_ = self._choose_beta(Y)
        k = min(self.rank_req_ + (1 if self.drop_first_ else 0), self.K_ - 1)
        dm = DiffusionMap(beta=self.beta_, alpha=self.alpha_, n_components=max(k, 1), precision=self.precision)
        dm.fit(Y)
        self.dm_ = dm
        if k <= 0:
            self.lam_ = np.zeros((0,))
            self.phi_ = np.zeros((self.K_, 0))
            self.psi_ = np.zeros((self.K_, 0))
        else:
            dm.transform()
            w, V = dm.eigenvalues_, dm.eigenvectors_
            if self.drop_first_ and w.size > 0:
                w, V = w[1:], V[:, 1:]
            self.lam_, self.phi_ = w, V
        # q(T) and d(T) of the fitted (most precise) state
        self.K_T_ = dm.D_ + 1e-18
        self.d_T_ = dm.D_alpha_ + 1e-18
        self.inv_sqrt_d_ = 1.0 / np.sqrt(self.d_T_)
        if k > 0:
            self.psi_ = self.inv_sqrt_d_[:, None] * self.phi_
        return self

    @property
    def Y_(self) -> np.ndarray:
        """Rotated training window vectors (K, L*D)."""
        return self._Y.double().cpu().numpy()

    # ---- encoding / Nystrom ---------------------------------------------------------
    def _prepare_query_windows(self, W_BLX, positions=None):
        """Validate query windows and build their positions (``FD/ROPE.py:446-487``)."""
        W = np.asarray(W_BLX, dtype=float)
        if W.ndim == 2:
            W = W[None, :, :]
        if W.ndim != 3:
            raise ValueError("Expected query windows with shape (B,L,D) or (L,D).")
        if W.shape[1:] != (self.L, self.D_):
            raise ValueError(f"Expected window shape (*,{self.L},{self.D_}), got {W.shape}")
        B = W.shape[0]
        if self.rope_mode_ == "sample":
            if positions is None:
                Pos = np.tile(np.arange(self.L, dtype=float), (B, 1))
            else:
                Pos = np.asarray(positions, dtype=float)
                if Pos.ndim == 1 and Pos.shape[0] == self.L:
                    Pos = np.tile(Pos[None, :], (B, 1))
                if Pos.shape != (B, self.L):
                    raise ValueError(f"For sample mode, positions must have shape ({B},{self.L}) or ({self.L},).")
            return W, Pos
        if positions is None:
            Pos = np.zeros((B,))
        else:
            Pos = np.asarray(positions, dtype=float)
            if Pos.ndim == 0:
                Pos = np.full((B,), float(Pos))
            if Pos.shape != (B,):
                raise ValueError(f"For window mode, positions must have shape ({B},) or scalar.")
        return W, Pos

    def encode_windows(self, W_BLX, positions=None) -> np.ndarray:
        """Nystrom coordinates (B, r) of query windows (``FD/ROPE.py:489-526``)."""
        if self.psi_ is None or self.lam_ is None or self.psi_.shape[1] == 0:
            B = 1 if np.asarray(W_BLX).ndim == 2 else np.asarray(W_BLX).shape[0]
            return np.zeros((B, 0))
        W, Pos = self._prepare_query_windows(W_BLX, positions)
        B, L, D = W.shape
        if self.rope_mode_ == "sample":
            Yq = self._rotate(W, L * D, D, Pos, L, 1, B)
        else:
            Yq = self._rotate(W, L * D, D, Pos, 1, 0, B)
        return self._nystrom(Yq)

    def _nystrom(self, Yq: torch.Tensor) -> np.ndarray:
        st = self.dm_._best_state()
        op = GaussianOperator(Yq, st.X, self.beta_, st.op.precision, shift=st.op.shift)
        dev = op.device
        a = self.alpha_
        wT = torch.as_tensor(self.K_T_ ** (-a), dtype=torch.float32, device=dev)
        Kq = op.apply(out_dtype=torch.float64)[:, 0] + 1e-18                 # row sums of k(q, T)
        wq = Kq ** (-a)
        dq = wq * op.apply(wT, out_dtype=torch.float64)[:, 0] + 1e-18        # sum_T k_alpha(q, T)
        lam_safe = np.maximum(self.lam_, 1e-12)
        V = torch.as_tensor(self.psi_ / lam_safe[None, :], dtype=torch.float64, device=dev)
        out = op.apply(V.contiguous(), col_scale=wT, row_scale=(wq / dq).float().contiguous(),
                       out_dtype=torch.float64)
        return out.cpu().numpy()

    def encode_window(self, W_cX, positions=None) -> np.ndarray:
        return self.encode_windows(np.asarray(W_cX)[None, :, :], positions=positions)[0]

    def encode_series(self, F_aX, sample_positions=None) -> np.ndarray:
        """Encode every Hankel window of a new series (``FD/ROPE.py:537-580``); windows read in place."""
        F = np.asarray(F_aX, dtype=float)
        if F.ndim == 1:
            F = F[:, None]
        N, D = F.shape
        if D != self.D_:
            raise ValueError(f"Expected D={self.D_}, got D={D}.")
        if sample_positions is None:
            sample_positions = np.arange(N, dtype=float)
        sample_positions = np.asarray(sample_positions, dtype=float)
        if sample_positions.shape != (N,):
            raise ValueError(f"sample_positions must have shape ({N},).")
        K = N - (self.L - 1) * self.step
        if K <= 0:
            raise ValueError(f"Need N={N} >= (L-1)*step+1 = {(self.L - 1) * self.step + 1}")
        if self.psi_ is None or self.psi_.shape[1] == 0:
            return np.zeros((K, 0))
        if self.rope_mode_ == "sample":
            Yq = self._rotate(F, D, self.step * D, sample_positions, 1, self.step, K)
        else:
            c_w = (0, self.L // 2, self.L - 1)[_WINDOW_POSITION[self.window_position_]]
            Yq = self._rotate(F, D, self.step * D, sample_positions[c_w * self.step:], 1, 0, K)
        return self._nystrom(Yq)

    @property
    def embedding_(self) -> np.ndarray:
        return self.psi_

    def fit_transform(self) -> np.ndarray:
        return self.psi_


# ---- rotary positions of query and key heads --------------------------------------

_LAYOUTS = {"half": 0, "interleaved": 1}
_ROTARY_DTYPES = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16, torch.bfloat16: native.DTYPE_BF16}
_POSITION_DTYPES = {torch.int32: native.DTYPE_I32, torch.int64: native.DTYPE_I64, torch.float32: native.DTYPE_F32,
                    torch.float64: native.DTYPE_F64}


def rotary_frequencies(rot: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       trained: int | None = None, slow: float = 1.0, fast: float = 32.0,
                       device=None) -> torch.Tensor:
    """(rot/2,) float64 radians per position of each pair: base^(-2p/rot), scaled for contexts ``factor`` times longer.

    scaling None      unscaled (``factor`` must be 1)
            "linear"  every frequency divided by ``factor``
            "base"    base raised to base * factor^(rot/(rot-2)): the fastest pair keeps its frequency, the
                      slowest is divided by ``factor``
            "parts"   pairs that make at most ``slow`` turns within the ``trained`` length are divided by
                      ``factor``, those with at least ``fast`` turns are kept, linear in the turns between
    """
    rot = int(rot)
    if rot < 2 or rot % 2:
        raise ValueError(f"rot must be even and at least 2 (got {rot})")
    if not base > 0 or not factor >= 1 or not math.isfinite(base) or not math.isfinite(factor):
        raise ValueError(f"base must be positive and factor at least 1 (got {base}, {factor})")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts' (got {scaling!r})")
    if scaling is None and factor != 1:
        raise ValueError("factor needs a scaling")
    if scaling == "base":
        if rot < 4:
            raise ValueError("scaling='base' needs rot >= 4")
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if trained is None or trained <= 0 or not 0 <= slow < fast:
            raise ValueError("scaling='parts' needs the trained length and 0 <= slow < fast")
        keep = np.clip((trained * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return torch.as_tensor(f, device=native.require_device(device))


def rotary_magnitude(factor: float) -> float:
    """Factor on the rotated coordinates that goes with scaling="parts": 0.1 ln(factor) + 1."""
    if not factor >= 1:
        raise ValueError(f"factor must be at least 1 (got {factor})")
    return 0.1 * math.log(factor) + 1.0


_NO_STRIDES = (0, 0, 0)


def _rotate_heads(xs, positions, freqs, layout, magnitude, inverse, inplace):
    """fd_rotary on one or two (B, S, H, D) tensors; returns the rotated tensors."""
    xs = [x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous() for x in xs]
    outs = xs if inplace else [torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]
    q, qo = xs[0], outs[0]
    b, s, h, d = q.shape
    if len(xs) > 1:
        k, ko = xs[1], outs[1]
        kp, kop, ks, kos, hk = k.data_ptr(), ko.data_ptr(), k.stride()[:3], ko.stride()[:3], k.shape[2]
    else:
        kp = kop = hk = 0
        ks = kos = _NO_STRIDES
    args = native.PACK_ROTARY(q.data_ptr(), kp, qo.data_ptr(), kop, *q.stride()[:3], *ks, *qo.stride()[:3], *kos,
                              positions.data_ptr(), *positions.stride(), freqs.data_ptr(), magnitude,
                              _ROTARY_DTYPES[q.dtype], _POSITION_DTYPES[positions.dtype], layout, inverse,
                              b, s, h, hk, d, 2 * freqs.numel())
    native.call(native.load().fd_rotary, q.device, args)
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, freqs, layout, magnitude, inverse, *xs):
        ctx.save_for_backward(positions, freqs)
        ctx.how = (layout, magnitude, inverse)
        return tuple(_rotate_heads(xs, positions, freqs, layout, magnitude, inverse, False))

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("apply_rotary has no second derivative: call backward without create_graph")
        native.refuse_duals("the gradient of apply_rotary", *grads)
        positions, freqs = ctx.saved_tensors
        layout, magnitude, inverse = ctx.how
        return (None,) * 5 + tuple(_rotate_heads(grads, positions, freqs, layout, magnitude, not inverse, False))


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None = None, *, positions: torch.Tensor, freqs: torch.Tensor,
                 layout: str = "half", magnitude: float = 1.0, inverse: bool = False, inplace: bool = False):
    """Rotate the heads of ``q`` (and ``k``) by their tokens' positions, in one launch.

    q (B, S, H, D) or (S, H, D), k the same with its own number of heads; float32, float16 or bfloat16,
    any strides with contiguous coordinates.  ``positions`` (S,) or (B, S), integer or floating (fractional
    positions are exact to fp64).  ``freqs``: (R/2,) float64 radians per position, R <= D
    (``rotary_frequencies``); pair p turns by positions * freqs[p] and coordinates R.. are copied.

    layout "half" pairs coordinate p with p + R/2, "interleaved" 2p with 2p + 1 (as ROPE does).  ``magnitude``
    scales the rotated coordinates, ``inverse`` turns the other way.  ``inplace`` overwrites q and k (no
    gradients; q and k must not overlap).  Forward-mode tangents and tracing are refused.  Returns the rotated q,
    or (q, k).
    """
    xs = (q,) if k is None else (q, k)
    for name, x in zip("qk", xs):
        if not isinstance(x, torch.Tensor) or x.dtype not in _ROTARY_DTYPES:
            raise TypeError(f"{name} must be a float32, float16 or bfloat16 tensor")
    shape, device = q.shape, q.device
    if not 3 <= len(shape) <= 4 or k is not None and (len(k.shape) != len(shape) or k.dtype != q.dtype or k.device != device):
        raise ValueError("q and k must be (S, H, D) or (B, S, H, D) tensors of one type on one device")
    if k is not None and (k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1]):
        raise ValueError(f"q {tuple(shape)} and k {tuple(k.shape)} may differ in their heads only")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved' (got {layout!r})")
    if not isinstance(freqs, torch.Tensor) or freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("freqs must be a one-dimensional float64 tensor")
    if not 1 <= freqs.shape[0] <= shape[-1] // 2:
        raise ValueError(f"freqs has {freqs.shape[0]} pairs, a head of {shape[-1]} coordinates takes 1 to "
                         f"{shape[-1] // 2}")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITION_DTYPES:
        raise TypeError("positions must be an int32, int64, float32 or float64 tensor")
    if not math.isfinite(magnitude):
        raise ValueError(f"magnitude must be finite (got {magnitude})")
    lead = shape[:-2]
    if positions.shape != lead and positions.shape != lead[-1:]:
        raise ValueError(f"positions {tuple(positions.shape)} must be {tuple(lead)} or {tuple(lead[-1:])}")
    if positions.device != device or freqs.device != device:
        raise ValueError("q, positions and freqs must be on one device")
    if positions.requires_grad or freqs.requires_grad:
        raise ValueError("apply_rotary has no gradient for positions and freqs: detach them")
    native.refuse_duals("apply_rotary", q, k, positions, freqs)
    native.require_device(device)
    grad = torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad)
    if inplace and grad:
        raise ValueError("inplace=True has no gradient: detach q and k, or rotate out of place")
    flat = len(shape) == 3
    x4 = [x[None] for x in xs] if flat else xs
    pos = positions if len(positions.shape) == 2 else positions[None].expand(x4[0].shape[0], -1)
    freqs = freqs.contiguous()
    if inplace:
        if any(x.stride(-1) != 1 and x.shape[-1] > 1 for x in x4):
            raise ValueError("inplace=True needs contiguous coordinates")
        for x in x4:
            if any(x.stride(i) == 0 and x.shape[i] > 1 for i in range(3)):
                raise ValueError("inplace=True cannot write to an expanded tensor")
        if k is not None and k.numel() and q.data_ptr() == k.data_ptr():
            raise ValueError("inplace=True would rotate the same memory as q and as k")
    args = (pos, freqs, _LAYOUTS[layout], float(magnitude), bool(inverse))
    out = _Rotary.apply(*args, *x4) if grad else _rotate_heads(x4, *args, inplace)
    if inplace:    # autograd sees the change, as of any operation in place
        torch.autograd.graph.increment_version([x for x in xs if not x.is_inference()])
    if flat:
        out = [o[0] for o in out]
    return out[0] if k is None else (out[0], out[1])
