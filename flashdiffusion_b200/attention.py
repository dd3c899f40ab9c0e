"""Softmax attention over key spans: the learned-model form of the Q != K kernel.

``FlashDiffusion`` sums values with the weights exp(-beta ||q_i - k_j||^2) and
leaves normalisation to given row scales.  ``attend`` is the row-stochastic
operator with exp(score) in their place, for batches of 16- or 32-bit heads and
with gradients:

  s_ij = scale q_i.k_j, or cap tanh(scale q_i.k_j / cap), minus slope_h |pos_i - j|
  o_i  = sum_j softmax_j(s_ij) v_j       over the span first_i <= j < end_i

Every mask offered is a span of keys for each row: causal, sliding window,
documents packed into one row (``document_spans``), prefixes seen by all rows
(``prefix_spans``), or any spans of the caller's own (``Spans``).  Rows with an
empty span give zeros and no gradient; keys outside a row's span never reach it,
whatever their memory holds.

``attend_cached`` is the form for the newest tokens of each sequence against a
key/value cache of which ``lengths`` rows are in use.

Everything runs on the current stream and may be captured into a graph.  Where a
captured step takes gradients of leaves (``backward`` into ``.grad``), run its
warm-up on a side stream, or drop every output of earlier eager steps first: a
leaf whose gradient node was made on the default stream, and is kept alive by
such an output, pulls that stream into the capture, which torch cannot do.  Forward-mode tangents (``torch.func.jvp``, dual tensors) and tracing
(``torch.jit.trace``, ``make_fx``) are refused.

16-bit heads are summed by the tensor core in fp32, from weights of 16 bits (``attend_cached`` splits them in two), and
its adder rounds toward zero: beside its rounding an output can come out low by 6e-9 of its weighted sum of |v| for each
key, 1e-4 at 16384 keys of values of one sign, and a gradient for each row that it sums likewise.  Gradients of fp16
heads hold dS at one power of two for a sequence and key head, so that very large values or output gradients there cost
the smallest dS bits.

The kernels' waits are bounded.  One that gives up (after two seconds, which nothing but a fault of the device or of
these kernels should bring about) raises no error by itself, since a call does not wait for the GPU: it leaves NaN in
the rows that were not finished and a mark that ``flashdiffusion_b200.native.check_status(device)`` turns into an
``FDError``.  A program that wants to know calls that where it waits for results anyway, once a step say.
"""

from __future__ import annotations

import torch

from . import native

__all__ = ["attend", "attend_cached", "Spans", "document_spans", "prefix_spans"]

_DTYPES = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16, torch.bfloat16: native.DTYPE_BF16}
MAX_DIM = 256


class Spans:
    """Keys first[.., i] <= j < end[.., i] seen by query row i: int32 device tensors (q_len,) or (batch, q_len).

    Values are clamped to the keys that exist; end <= first is a row that sees nothing.
    """

    def __init__(self, first: torch.Tensor, end: torch.Tensor):
        for t in (first, end):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
                raise TypeError("first and end must be int32 tensors")
        if first.shape != end.shape or first.dim() not in (1, 2) or first.device != end.device:
            raise ValueError("first and end must be (q_len,) or (batch, q_len) tensors of one shape and device")
        first, end = (t[None] if t.dim() == 1 else t for t in (first, end))
        self.first, self.end = first.contiguous(), end.contiguous()

    @property
    def batch(self) -> int:
        return self.first.shape[0]

    @property
    def q_len(self) -> int:
        return self.first.shape[1]


def _int32(name: str, t: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1:
        raise TypeError(f"{name} must be a one-dimensional int32 tensor")
    native.require_device(t.device)
    return t.contiguous()


def document_spans(offsets: torch.Tensor, rows: int, *, causal: bool = True, window: int | None = None,
                   prefix: torch.Tensor | None = None) -> Spans:
    """Spans of a packed batch: document d holds rows offsets[d] .. offsets[d + 1] of ``rows``.

    A row sees its own document up to itself (all of it with causal=False), at most ``window`` rows back,
    or also the first prefix[d] rows of the document (``prefix``: one length per document, without a
    window).  Rows outside all documents (padding behind the last one) see nothing.
    """
    offsets = _int32("offsets", offsets)
    if offsets.numel() < 1:
        raise ValueError("offsets needs at least one entry")
    rows, window = int(rows), _window(window, causal)
    if rows < 0:
        raise ValueError(f"rows must not be negative (got {rows})")
    if prefix is not None:
        prefix = _int32("prefix", prefix)
        if prefix.numel() != offsets.numel() - 1 or prefix.device != offsets.device:
            raise ValueError(f"prefix needs one length for each of the {offsets.numel() - 1} documents")
        if window or not causal:
            raise ValueError("a prefix needs causal=True and no window")
    first = torch.empty((1, rows), dtype=torch.int32, device=offsets.device)
    end = torch.empty_like(first)
    native.call(native.load().fd_attention_document_spans, offsets.device, offsets.data_ptr(), offsets.numel() - 1,
                native._ptr(prefix), rows, int(causal), window, first.data_ptr(), end.data_ptr())
    return Spans(first, end)


def prefix_spans(prefix: torch.Tensor, q_len: int, k_len: int | None = None) -> Spans:
    """Spans of rows that see the first prefix[b] keys of sequence b and all keys up to their own position."""
    prefix = _int32("prefix", prefix)
    q_len = int(q_len)
    k_len = q_len if k_len is None else int(k_len)
    first = torch.empty((prefix.numel(), q_len), dtype=torch.int32, device=prefix.device)
    end = torch.empty_like(first)
    native.call(native.load().fd_attention_prefix_spans, prefix.device, prefix.data_ptr(), prefix.numel(), q_len, k_len,
                first.data_ptr(), end.data_ptr())
    return Spans(first, end)


def _window(window, causal) -> int:
    if window is None:
        return 0
    if int(window) < 1:
        raise ValueError(f"window must be at least 1 (got {window})")
    if not causal:
        raise ValueError("a window needs causal=True")
    return min(int(window), 2**31 - 1)


def _loadable(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels take it: contiguous coordinates, and 16-bit heads that the tensor-core kernels could take
    at 16-byte steps in memory.  A copy is made of what is not: it costs one pass over t."""
    n0, n1, n2, d = t.shape
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 and d > 1:
        return t.contiguous()
    if t.dtype == torch.float32 or d % 8:
        return t
    if (t.data_ptr() % 16 or n0 > 1 and (s0 % 8 or not s0) or n1 > 1 and (s1 % 8 or not s1)
            or n2 > 1 and (s2 % 8 or not s2)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


_NO_GRADIENTS = (0,) * 16


def _arguments(q, k, v, o, lse, low, how, gradients=_NO_GRADIENTS) -> bytes:
    """fd_attention_args, packed; lse and low are addresses, 0 for none."""
    spans, causal, window, lengths, slopes, scale, cap = how
    b, sq, h, d = q.shape
    if spans is None:
        first = end = step = 0
    else:
        first, end, step = spans.first.data_ptr(), spans.end.data_ptr(), sq if spans.batch > 1 else 0
    return native.PACK_ATTENTION(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], o.data_ptr(),
        *o.stride()[:3], lse or 0, low or 0, first, end, step,
        0 if lengths is None else lengths.data_ptr(), 0 if slopes is None else slopes.data_ptr(), scale, cap,
        _DTYPES[q.dtype], causal, window, b, sq, k.shape[1], h, k.shape[2], d, *gradients)


def _call(fn, args, backward, q):
    if torch._C._cuda_getDevice() != q.device.index:      # sizes depend on the number of SMs of the current device
        with torch.cuda.device(q.device):
            return _call(fn, args, backward, q)
    # the caching allocator's own buffer for each call: streams and captured graphs never share it
    nbytes = native.load().fd_attention_workspace_bytes(args, backward)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    native.call(fn, q.device, args, ws.data_ptr() if nbytes else 0, nbytes)


def _forward(q, k, v, how, want_lse):
    """(output, lse or None) of heads that are loadable."""
    o = _like(q)
    lse = _lse_like(q) if want_lse else None
    _call(native.load().fd_attention_forward, _arguments(q, k, v, o, lse.data_ptr() if want_lse else 0, 0, how), 0, q)
    return o, lse


def _lse_like(q):
    return q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)


def _kept(kept, lse, low_at):
    """Addresses of lse and of o's low bits (0: none)."""
    at = kept.data_ptr()
    return at if lse is None else lse.data_ptr(), 0 if low_at is None else at + low_at


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, how, return_lse):
        q, k, v = _loadable(q), _loadable(k), _loadable(v)
        b, sq, h, d = q.shape
        # one buffer for what the gradients want besides o: lse (unless it is an output), and for 16-bit heads whose
        # forward pass is on the tensor cores eight more bits of o
        rows = b * sq * h
        low = rows * d if q.dtype is not torch.float32 and d % 8 == 0 else 0
        ctx.low_at = (0 if return_lse else (rows + 1) // 2 * 8) if low else None
        kept = torch.empty((0 if return_lse else (rows + 1) // 2 * 8) + low, dtype=torch.uint8, device=q.device)
        o, lse = _like(q), _lse_like(q) if return_lse else None
        _call(native.load().fd_attention_forward, _arguments(q, k, v, o, *_kept(kept, lse, ctx.low_at), how), 0, q)
        spans, slopes = how[0], how[4]
        if spans is None and slopes is None:
            ctx.save_for_backward(q, k, v, o, kept, lse)
        else:    # what the gradients read again: autograd notices if it was changed in between
            ctx.save_for_backward(q, k, v, o, kept, lse, *(() if spans is None else (spans.first, spans.end)),
                                  *(() if slopes is None else (slopes,)))
        ctx.how = how
        if not return_lse:
            return o
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, do, *_):
        if torch.is_grad_enabled():
            raise RuntimeError("attend has no second derivative: call backward without create_graph")
        native.refuse_duals("the gradient of attend", do)
        q, k, v, o, kept, lse = ctx.saved_tensors[:6]
        do = _loadable(do)
        dq, dk, dv = _like(q), _like(k), _like(v)
        args = _arguments(q, k, v, o, *_kept(kept, lse, ctx.low_at), ctx.how,
                          (do.data_ptr(), *do.stride()[:3], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                           *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3]))
        _call(native.load().fd_attention_backward, args, 1, q)
        return dq, dk, dv, None, None


def _check(q, k, v, slopes, scale, cap, names):
    # the usual call is found in order by these comparisons; _explain says what is wrong with any other
    qs, ks = q.shape, k.shape
    if not (ks == v.shape and q.dtype is k.dtype is v.dtype and q.dtype in _DTYPES and q.device == k.device == v.device
            and len(qs) == len(ks) and 3 <= len(qs) <= 4 and qs[-1] == ks[-1] and qs[:-3] == ks[:-3]
            and 1 <= qs[-1] <= MAX_DIM and ks[-2] >= 1 and qs[-2] >= 1 and qs[-2] % ks[-2] == 0):
        _explain(q, k, v, names)
    h = qs[-2]
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or tuple(slopes.shape) != (h,):
            raise ValueError(f"slopes must be a float32 tensor of {h} values")
        if slopes.device != q.device:
            raise ValueError("slopes must be on the device of the heads")
        if slopes.requires_grad:
            raise ValueError("there is no gradient for slopes: detach them")
    scale = qs[-1] ** -0.5 if scale is None else float(scale)
    cap = 0.0 if cap is None else float(cap)
    if not abs(scale) <= 1e30:
        raise ValueError(f"scale must be finite and at most 1e30 (got {scale})")
    if cap and not 1e-3 <= cap <= 1e18:
        raise ValueError(f"cap must be None or 1e-3 to 1e18 (got {cap})")
    native.refuse_duals("attention", q, k, v, slopes)
    native.require_device(q.device)
    return scale, cap


def _explain(q, k, v, names):
    for name, t in zip(names, (q, k, v)):
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be a float32, float16 or bfloat16 tensor")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{names[0]}, {names[1]} and {names[2]} must have one type and device")
        if t.dim() != q.dim() or t.dim() not in (3, 4):
            raise ValueError(f"{name} {tuple(t.shape)} must be (S, H, D) or (B, S, H, D), as {names[0]} is")
    if k.shape != v.shape:
        raise ValueError(f"{names[1]} {tuple(k.shape)} and {names[2]} {tuple(v.shape)} must have one shape")
    if q.shape[-1] != k.shape[-1] or q.shape[:-3] != k.shape[:-3]:
        raise ValueError(f"{names[0]} {tuple(q.shape)} and {names[1]} {tuple(k.shape)} differ in batch or head size")
    if not 1 <= q.shape[-1] <= MAX_DIM:
        raise ValueError(f"heads of 1 to {MAX_DIM} coordinates (got {q.shape[-1]})")
    raise ValueError(f"{q.shape[-2]} query heads are no multiple of {k.shape[-2]} key heads")


def _tensors(names, ts):
    for name, t in zip(names, ts):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a float32, float16 or bfloat16 tensor")


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, causal: bool = False,
           window: int | None = None, cap: float | None = None, slopes: torch.Tensor | None = None,
           spans: Spans | None = None, return_lse: bool = False):
    """softmax(scores) v over each row's span of keys; differentiable in q, k and v.

    q (B, Sq, H, D), k and v (B, Sk, Hk, D) with H a multiple of Hk (query head h reads key head h // (H/Hk)),
    or all three without the batch axis; float16, bfloat16 or float32, D <= 256, any strides with contiguous
    coordinates.  Query row i stands at position Sk - Sq + i.

    scale    of the products, D^-1/2 by default
    causal   keys up to the row's own position; ``window``: at most that many of them
    spans    a ``Spans`` in the place of causal and window
    cap      scores become cap tanh(score / cap); 1e-3 to 1e18
    slopes   (H,) float32: slope times the distance |position - j| is subtracted from the scores
    Returns the output (as q), or (output, lse): lse (B, H, Sq) float32 is the natural log of the sum of
    exp(scores), -inf for rows that see nothing; it carries no gradient.  A row that sees keys, but none above a score of
    -infinity, is NaN.
    """
    _tensors(("q", "k", "v"), (q, k, v))
    scale, cap = _check(q, k, v, slopes, scale, cap, ("q", "k", "v"))
    flat = q.dim() == 3
    if flat:
        q, k, v = q[None], k[None], v[None]
    if spans is not None:
        if not isinstance(spans, Spans):
            raise TypeError("spans must be a Spans")
        if causal or window is not None:
            raise ValueError("spans replace causal and window")
        if spans.batch not in (1, q.shape[0]) or spans.q_len != q.shape[1] or spans.first.device != q.device:
            raise ValueError(f"spans ({spans.batch}, {spans.q_len}) on {spans.first.device} do not fit "
                             f"q {tuple(q.shape)} on {q.device}")
    slopes = None if slopes is None else slopes.contiguous()
    how = (spans, bool(causal), _window(window, causal), None, slopes, scale, cap)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o = _Attend.apply(q, k, v, how, return_lse)
        o, lse = o if return_lse else (o, None)
    else:
        o, lse = _forward(_loadable(q), _loadable(k), _loadable(v), how, return_lse)
    if flat:
        o, lse = o[0], None if lse is None else lse[0]
    return (o, lse) if return_lse else o


def attend_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                  scale: float | None = None, window: int | None = None, cap: float | None = None,
                  slopes: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention of the newest tokens of each sequence against a cache; no gradients.

    q (B, N, H, D): the last N tokens of each sequence, which stand at positions lengths[b] - N .. lengths[b] - 1;
    k_cache, v_cache (B, capacity, Hk, D) with the first lengths[b] rows in use (the new tokens' among them),
    lengths (B,) int32 on the device (clamped to the capacity; a row at a negative position sees nothing).
    Rows of the cache behind lengths[b] are never looked at.  scale, window, cap, slopes and return_lse as in
    ``attend``.
    """
    _tensors(("q", "k_cache", "v_cache"), (q, k_cache, v_cache))
    scale, cap = _check(q, k_cache, v_cache, slopes, scale, cap, ("q", "k_cache", "v_cache"))
    if q.dim() != 4:
        raise ValueError(f"q must be (B, N, H, D) (got {tuple(q.shape)})")
    lengths = _int32("lengths", lengths)
    if tuple(lengths.shape) != (q.shape[0],) or lengths.device != q.device:
        raise ValueError(f"lengths must hold {q.shape[0]} values on {q.device}")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise ValueError("attend_cached has no gradient: detach its inputs, or use attend")
    slopes = None if slopes is None else slopes.contiguous()
    o, lse = _forward(_loadable(q), _loadable(k_cache), _loadable(v_cache),
                      (None, True, _window(window, True), lengths, slopes, scale, cap), return_lse)
    return (o, lse) if return_lse else o
