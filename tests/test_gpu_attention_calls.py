"""Calls of attend and attend_cached that their documentation allows, against the same bits by another call or the
definition in 64 bits (tests/attention_reference.py)."""
import pytest
import torch

from tests.attention_reference import check, reference, spans_of

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
# fp16 holds nothing finer than 2^-25 absolute: outputs that small, and the ds values they are summed from
FLOOR = {BF: 0.0, HF: 2.0 ** -25, SF: 0.0}


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    """A bounded wait that gives up leaves its mark in the status word and its results unfinished."""
    yield
    from flashdiffusion_b200 import native
    native.check_status()


def _inputs(b, sq, sk, h, hk, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return mk(b, sq, h, d), mk(b, sk, hk, d), mk(b, sk, hk, d), mk(b, sq, h, d)


def _step(q, k, v, do, **kw):
    from flashdiffusion_b200.attention import attend
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o, lse = attend(q, k, v, return_lse=True, **kw)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {"o": o.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _compare(out, ref, dtype):
    for name in out:
        check(name, out[name], ref, 0.0 if name == "lse" else FLOOR[dtype])


@pytest.fixture
def guarded(monkeypatch):
    """Workspaces of exactly the size asked for, with bytes behind them that must not change."""
    from flashdiffusion_b200 import attention, native

    def call(fn, args, backward, q):
        n = native.load().fd_attention_workspace_bytes(args, backward)
        ws = torch.full((n + (32 << 20),), 0xA5, dtype=torch.uint8, device=q.device)
        native.call(fn, q.device, args, ws.data_ptr(), n)
        assert (ws[n:] == 0xA5).all()

    monkeypatch.setattr(attention, "_call", call)


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("b,s,h,hk,d,window", [(1, 1024, 32, 8, 128, 4096), (1, 2048, 16, 4, 128, 4096),
                                               (1, 2048, 4, 1, 128, 4096), (1, 1900, 8, 4, 128, 2 ** 31 - 1),
                                               (1, 3000, 4, 1, 64, 6000)])
def test_a_window_that_reaches_every_key_is_no_window(guarded, b, s, h, hk, d, window, dtype):
    """Sizes whose gradients are cut into parts with fp32 sums of their own in the workspace."""
    q, k, v, do = _inputs(b, s, s, h, hk, d, dtype, seed=s)
    want = _step(q, k, v, do, causal=True)
    got = _step(q, k, v, do, causal=True, window=window)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype,kw", [
    (1, 300, 3001, 2, 1, 128, BF, dict(causal=True)), (1, 1500, 1500, 4, 1, 64, HF, dict(causal=True, window=700)),
    (1, 2100, 140, 1, 1, 80, BF, dict()), (1, 3, 5000, 8, 2, 128, HF, dict()), (1, 200, 3000, 2, 1, 256, BF, dict()),
    (2, 100, 130, 2, 1, 48, SF, dict(causal=True)), (1, 100, 2000, 2, 1, 20, BF, dict()), (3, 77, 77, 4, 4, 64, HF, dict()),
], ids=str)
def test_workspaces_are_not_left(guarded, b, sq, sk, h, hk, d, dtype, kw):
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=sk)
    lo, hi, pos = spans_of(sq, sk, b, causal=kw.get("causal", False), window=kw.get("window"))
    _compare(_step(q, k, v, do, **kw), reference(q, k, v, lo, hi, pos, do=do), dtype)


def _spans(kind, sq, sk):
    """Keyword arguments and the keys that no row sees (rows that see nothing are the caller's to find)."""
    from flashdiffusion_b200.attention import Spans, document_spans
    if kind == "documents":
        spans = document_spans(torch.tensor([0, 100, sk - 190], dtype=torch.int32, device="cuda"), sq)
    elif kind == "holes":        # rows in no order that see keys 3 .. 9, 40 .. 59 and 260 .. 399
        i = torch.arange(sq)
        first = torch.where(i % 3 == 0, 3, torch.where(i % 3 == 1, 40, 260)).int()
        end = torch.where(i % 3 == 0, 10, torch.where(i % 3 == 1, 60, 400)).int()
        end[5::7] = 0
        spans = Spans(first.cuda(), end.cuda())
    else:                        # the last rows of a window: keys before it are never seen
        return dict(causal=True, window=50), torch.arange(sk) < sk - sq - 49, torch.zeros(sq, dtype=torch.bool)
    first, end = spans.first[0].cpu(), spans.end[0].cpu()
    j = torch.arange(sk)
    return dict(spans=spans), ~((j >= first[:, None]) & (j < end[:, None])).any(0), end <= first


@pytest.mark.parametrize("bad", [6e4, -6e4], ids=str)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (HF, 128), (SF, 48)], ids=str)
@pytest.mark.parametrize("kind,sq,sk", [("documents", 400, 400), ("holes", 2300, 500), ("window", 130, 700)])
def test_masked_places_hold_large_numbers(kind, sq, sk, dtype, d, bad):
    """Finite and large where NaN and infinities are looked for elsewhere: the same bits, gradients too."""
    q, k, v, do = _inputs(1, sq, sk, 4, 2, d, dtype, seed=71)
    kw, unseen, empty = _spans(kind, sq, sk)
    assert unseen.any()
    want = _step(q, k, v, do, **kw)
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    for t in (k2, v2):
        t[:, unseen] = bad
    for t in (q2, do2):
        t[:, empty] = bad
    got = _step(q2, k2, v2, do2, **kw)
    for n in got:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
def test_sequences_and_key_heads_do_not_touch_each_other(dtype):
    """A sequence's and a key head's results are the same bits whatever the others hold."""
    b, s, h, hk, d = 2, 500, 4, 2, 64
    q, k, v, do = _inputs(b, s, s, h, hk, d, dtype, seed=73)
    want = _step(q, k, v, do, causal=True)
    v2, do2 = v.clone(), do.clone()
    v2[1, :, 1] *= 1000
    do2[1, :, 2:] *= 16
    got = _step(q, k, v2, do2, causal=True)
    for n in got:
        x, y = (t[n].transpose(1, 2) if n != "lse" else t[n] for t in (got, want))       # (batch, head, row ..)
        one = 1 if n in ("dk", "dv") else 2                                                # heads of key head 0
        assert torch.equal(x[0], y[0]) and torch.equal(x[1, :one], y[1, :one]), n
    lo, hi, pos = spans_of(s, s, b, causal=True)
    ref = reference(q, k, v2, lo, hi, pos, do=do2)
    if dtype is HF:
        # |dS| reaches 16 sqrt(64) 1000 sqrt(64) here, so some exact gradients leave fp16: its largest number is 65504,
        # and from half a step (16) above it on, less the bound, every value in reach rounds to an infinity
        for n in ("dq", "dk", "dv"):
            over = ref[n].abs() - ref[n + "_tol"] * 1.001 >= 65504 + 16
            assert (got[n].cpu().double()[over] == ref[n][over].sign() * float("inf")).all()
            ref[n][over] = got[n].cpu().double()[over]
    _compare(got, ref, dtype)


def test_a_wait_that_gave_up_is_reported():
    """As the module says: the mark stays through later calls, and check_status raises for it once."""
    from flashdiffusion_b200 import attention, native
    q, k, v, do = _inputs(1, 200, 200, 2, 1, 64, BF)
    native.check(native.load().fd_selftest_wait_timeout(10_000_000, native._stream(q.device)))
    _step(q, k, v, do)
    with pytest.raises(native.FDError) as e:
        native.check_status(q.device)
    assert e.value.code == native.FD_ERR_TIMEOUT
    native.check_status(q.device)
    assert "check_status" in attention.__doc__


# forward kernels: whole and cut key axes of both tile heights, few rows, fp32 and odd heads by tiles and by rows
SIZES = [(1, 300, 700, 2, 1, 64, BF), (1, 300, 700, 2, 1, 128, HF), (4, 700, 300, 40, 4, 64, BF), (1, 200, 2000, 2, 1, 256, BF),
         (1, 140, 3000, 1, 1, 128, BF), (1, 3, 700, 4, 2, 128, HF), (2, 8, 5000, 4, 2, 64, BF), (1, 300, 700, 2, 1, 48, SF),
         (1, 300, 700, 2, 1, 20, BF), (1, 2, 700, 2, 1, 40, SF)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype", SIZES, ids=str)
def test_a_row_of_minus_infinities_has_no_softmax(b, sq, sk, h, hk, d, dtype, causal):
    """An infinite coordinate of q against keys of the other sign: NaN whatever the mask, and the other rows as ever."""
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=81)
    k[..., 0] = -1
    kw = dict(causal=causal, cap=None)
    want = _step(q, k, v, do, **kw)
    at = sq // 2
    if causal and sk < sq:
        at = max(at, sq - sk)                     # a row that sees something
    q[:, at, :, 0] = float("inf")
    got = _step(q, k, v, do, **kw)
    other = torch.arange(sq, device="cuda") != at
    assert got["o"][:, at].isnan().all() and got["lse"][:, :, at].isnan().all() and got["dq"][:, at].isnan().all()
    assert torch.equal(got["o"][:, other], want["o"][:, other]) and torch.equal(got["dq"][:, other], want["dq"][:, other])
    assert torch.equal(got["lse"][:, :, other], want["lse"][:, :, other])


@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype", SIZES, ids=str)
def test_keys_at_minus_infinity_weigh_nothing(b, sq, sk, h, hk, d, dtype):
    """The first keys of all rows at score -infinity (whole tiles of them): as if they were masked."""
    from flashdiffusion_b200.attention import attend
    q, k, v, _ = _inputs(b, sq, sk, h, hk, d, dtype, seed=83)
    q[..., 0], away = 1, 2 * sk // 3
    k[:, :away, :, 0] = float("-inf")
    o, lse = attend(q, k, v, return_lse=True)
    first = torch.full((1, sq), away)
    lo, hi, pos = spans_of(sq, sk, b, first=first, end=torch.full((1, sq), sk))
    ref = reference(q, k, v, lo, hi, pos)
    check("o", o, ref, FLOOR[dtype])
    check("lse", lse, ref)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (BF, 256), (SF, 32)], ids=str)
def test_a_cached_row_of_minus_infinities_has_no_softmax(dtype, d):
    from flashdiffusion_b200.attention import attend_cached
    lengths = torch.tensor([0, 1, 130, 900], dtype=torch.int32, device="cuda")
    q, k, v, _ = _inputs(4, 2, 900, 4, 2, d, dtype, seed=85)
    k[..., 0] = -1
    q[:, 1, :, 0] = float("inf")
    o, lse = attend_cached(q, k, v, lengths, return_lse=True)
    assert (o[0] == 0).all() and (lse[0] == float("-inf")).all()
    assert o[1:, 1].isnan().all() and lse[1:, :, 1].isnan().all()
    assert (o[1, 0] == 0).all() and o[2:, 0].isfinite().all() and lse[2:, :, 0].isfinite().all()


@pytest.mark.parametrize("new,h,hk,d", [(1, 8, 4, 128), (1, 4, 4, 64), (3, 8, 4, 64), (4, 16, 4, 128)])
@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("above", [15.0, 17.0])
def test_small_weights_of_a_cache_are_kept(above, dtype, new, h, hk, d):
    """The newest tokens' keys `above` nats over all others, with values of zero: the output is the small weights' alone.
    2^-24 of the largest weight is below fp16's own range, and here the many small ones are all there is.  So many
    sequences that one warp goes on from the newest keys to a quarter of the others."""
    from flashdiffusion_b200.attention import attend_cached
    b, keys = 160, 600
    q, k, v, _ = _inputs(b, new, keys, h, hk, d, dtype, seed=87)
    q[..., 0], k[..., 0] = 4, 0
    q[..., 1:] /= 16
    k[:, -new:, :, 0] = above * d ** 0.5 / 4
    v[:, -new:] = 0
    v = v.abs()
    n = torch.full((b,), keys, dtype=torch.int32, device="cuda")
    lo, hi, pos = spans_of(new, keys, b, causal=True, lengths=n.cpu())
    ref = reference(q, k, v, lo, hi, pos)
    o, lse = attend_cached(q, k, v, n, return_lse=True)
    # beside the definition's bounds: fp16 holds a weight to 2^-25 at 2^7 times the largest, and the sum of weights is at
    # least the largest, so each value may come with 2^-32 too much or too little
    check("o", o, ref, 2.0 ** -32 * float(v.double().sum(1).max()) + FLOOR[dtype])
    check("lse", lse, ref)


@pytest.mark.parametrize("bad", [6e4, float("inf"), float("nan")], ids=str)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (SF, 48)], ids=str)
@pytest.mark.parametrize("kind,sq,sk", [("documents", 400, 400), ("holes", 2300, 500), ("window", 130, 700)])
def test_masked_places_hold_anything_under_a_wide_cap(kind, sq, sk, dtype, d, bad):
    """All visible scores well inside their cap, masked ones beyond it: the same bits."""
    q, k, v, do = _inputs(1, sq, sk, 4, 2, d, dtype, seed=91)
    kw, unseen, empty = _spans(kind, sq, sk)
    kw["cap"] = 50.0
    want = _step(q, k, v, do, **kw)
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    for t in (k2, v2):
        t[:, unseen] = bad
    for t in (q2, do2):
        t[:, empty] = bad
    got = _step(q2, k2, v2, do2, **kw)
    for n in got:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype,d,new", [(BF, 128, 1), (HF, 64, 3), (BF, 256, 1), (SF, 64, 2)], ids=str)
def test_a_cache_holds_anything_behind_a_row_under_a_wide_cap(dtype, d, new):
    """Several new tokens: the keys of later ones are hidden from the earlier, whatever they hold, and the end of the
    cache from all."""
    from flashdiffusion_b200.attention import attend_cached
    q, k, v, _ = _inputs(2, new, 300, 4, 2, d, dtype, seed=93)
    n = torch.tensor([290, 17], dtype=torch.int32, device="cuda")
    want = attend_cached(q, k, v, n, cap=50.0)
    k2, v2 = k.clone(), v.clone()
    for b, m in ((0, 290), (1, 17)):
        k2[b, m - new + 1:] = v2[b, m - new + 1:] = 6e4
    got = attend_cached(q, k2, v2, n, cap=50.0)
    assert torch.equal(got[:, 0], want[:, 0])


@pytest.mark.parametrize("cap", [1e4, 1e6, 1e12])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype", SIZES, ids=str)
def test_a_very_wide_cap_changes_nothing(b, sq, sk, h, hk, d, dtype, cap):
    """Scores of a few units: cap tanh(s / cap) is s to within s (s / cap)^2 / 3, some 1e-6 at the smallest cap here."""
    from flashdiffusion_b200.attention import attend
    q, k, v, _ = _inputs(b, sq, sk, h, hk, d, dtype, seed=95)
    lo, hi, pos = spans_of(sq, sk, b, causal=True)
    o, lse = attend(q, k, v, causal=True, cap=cap, return_lse=True)
    ref = reference(q, k, v, lo, hi, pos)
    check("o", o, ref, FLOOR[dtype])
    check("lse", lse, ref)


@pytest.mark.parametrize("cap", [20.0, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype", SIZES, ids=str)
def test_wide_caps_over_their_whole_range(b, sq, sk, h, hk, d, dtype, cap):
    """Scores up to 0.44 of the cap, large heads and a small scale: the coefficients of a series of the tanh in the raw
    products leave fp32's normal numbers one by one."""
    from flashdiffusion_b200.attention import attend
    q, k, v, _ = _inputs(b, sq, sk, h, hk, d, dtype, seed=97)
    q, k = q * 1000, k * 1000
    lo, hi, pos = spans_of(sq, sk, b)
    top = max(float((q[:, :, i].double() @ k[:, :, i * hk // h].double().transpose(1, 2)).abs().max()) for i in range(h))
    scale = 0.44 * cap / top
    lse = attend(q, k, v, cap=cap, scale=scale, return_lse=True)[1]
    check("lse", lse, reference(q, k, v, lo, hi, pos, cap=cap, scale=scale))


@pytest.mark.parametrize("d", [64, 136, 256])
@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("rows", [1, 130])
def test_rows_that_cancel(rows, dtype, d):
    """Queries that look at two keys whose values differ little: dS = P (dP - delta) is the small difference of large
    numbers."""
    from flashdiffusion_b200.attention import attend
    g = torch.Generator("cuda").manual_seed(57)
    q, k = (torch.randn(1, n, 1, d, device="cuda", generator=g).to(dtype) for n in (rows, 2))
    u = torch.finfo(dtype).eps / 2
    v = torch.ones(1, 2, 1, d, device="cuda", dtype=dtype)
    v[0, 1] += 4 * u
    do = torch.ones(1, rows, 1, d, device="cuda", dtype=dtype)
    lo, hi, pos = spans_of(rows, 2, 1)
    ref = reference(q, k, v, lo, hi, pos, do=do)
    dq, = torch.autograd.grad(attend(q.requires_grad_(True), k, v), q, do)
    # p (1 - p) <= 1/4, dP - delta <= 4 u d.  delta is off by d 2 (2^-8 u of the kept bits and 2^-20 of fp32 steps), P by
    # 2^-15, and dS is rounded once.  Where the weights of P V are rounded to 16 bits (all but few rows of narrow heads),
    # o = sum_j p_j (1 + e_j) v_j with |e_j| <= u and v_j <= 1 + 4 u, so that delta is off by up to d u (1 + 4 u) more, and
    # P times that is at most 1 / 2 for the smaller weight and the whole for the larger
    p = 0.25
    ds_tol = d ** -0.5 * (2 * p * d * 2 * (2.0 ** -8 * u + 2.0 ** -20) + p * 4 * u * d * (2.0 ** -15 + u))
    if rows > 1 or d > 128:
        ds_tol += d ** -0.5 * d * u * (1 + 4 * u)
    room = u * ref["dq"].abs() + ds_tol * k.double().cpu().abs().sum(1, keepdim=True)
    assert ((dq.double().cpu() - ref["dq"]).abs() <= room + FLOOR[dtype]).all()


@pytest.mark.parametrize("d", [64, 136, 256])
@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("rows", [1, 130])
def test_the_low_bits_of_the_output_serve_the_gradients(rows, dtype, d):
    """Two equal weights, which are exact, and values 1 and 1 + 2 u: o = 1 + u lies between two numbers of its type, and
    dS = -+ P u d scale.  From the rounded output, 1, it would be 0 and twice that."""
    from flashdiffusion_b200.attention import attend
    g = torch.Generator("cuda").manual_seed(59)
    u = torch.finfo(dtype).eps / 2
    q = torch.zeros(1, rows, 1, d, device="cuda", dtype=dtype, requires_grad=True)
    k = torch.randn(1, 2, 1, d, device="cuda", generator=g).to(dtype)
    v = torch.ones(1, 2, 1, d, device="cuda", dtype=dtype)
    v[0, 1] += 2 * u
    do = torch.ones(1, rows, 1, d, device="cuda", dtype=dtype)
    dq, = torch.autograd.grad(attend(q, k, v), q, do)
    k64 = k.double()[0, :, 0]
    ds = 0.5 * u * d ** 0.5
    want = ds * (k64[1] - k64[0])
    # delta = d (1 + u) is kept exactly and summed in fp32 (d 2^-24 of it at most); P is off by 2^-15 and rounded once, so
    # is dS, and the output
    ds_tol = ds * (2.0 ** -15 + 2 * u) + 0.5 * d ** -0.5 * d * d * 2.0 ** -24
    room = u * want.abs() + ds_tol * k64.abs().sum(0)
    assert ((dq.double()[0, :, 0] - want).abs() <= room + FLOOR[dtype]).all()


@pytest.mark.parametrize("cap", [None, 50.0])
@pytest.mark.parametrize("dtype,d,new,h,hk", [(BF, 128, 4, 8, 2), (HF, 64, 3, 4, 1), (BF, 64, 8, 4, 1), (HF, 128, 2, 2, 2),
                                              (BF, 256, 3, 4, 2), (SF, 64, 3, 4, 2)], ids=str)
def test_keys_of_later_tokens_do_not_touch_earlier_ones(dtype, d, new, h, hk, cap):
    """Several new tokens: a key that only the last of them see may be large, and moves no bit of the others."""
    from flashdiffusion_b200.attention import attend_cached
    b, capacity = 40, 400
    q, k, v, _ = _inputs(b, new, capacity, h, hk, d, dtype, seed=99)
    n = torch.linspace(new, capacity, b, device="cuda").int()
    want = attend_cached(q, k, v, n, cap=cap)
    at = n.long()[:, None] - 1                                     # the last token's key
    k2 = k.scatter(1, at[:, :, None, None].expand(b, 1, hk, d), k.gather(1, at[:, :, None, None].expand(b, 1, hk, d)) * 24)
    got = attend_cached(q, k2, v, n, cap=cap)
    assert not torch.equal(got[:, -1], want[:, -1])
    assert torch.equal(got[:, :-1], want[:, :-1])


@pytest.mark.parametrize("cap", [None, 50.0])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,dtype", SIZES, ids=str)
def test_later_keys_do_not_touch_earlier_rows(b, sq, sk, h, hk, d, dtype, cap):
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=101)
    want = _step(q, k, v, do, causal=True, cap=cap)
    row = sq - 1 if sq < 40 else sq // 3                           # the first row that sees the keys below
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[:, max(sk - sq + row, 0):] *= 24
    got = _step(q, k2, v2, do, causal=True, cap=cap)
    assert torch.equal(got["o"][:, :row], want["o"][:, :row])
    assert torch.equal(got["lse"][:, :, :row], want["lse"][:, :, :row])
    x, y = got["dq"][:, :row], want["dq"][:, :row]
    if dtype is not HF or d > 128:
        assert torch.equal(x, y)
        return
    # fp16 gradients hold dS at a power of two that brings 2 |dO| |V|, of all rows of a sequence that take part, to 2^14 or
    # more: below fp16's normal numbers it is off by at most half of 2^-24 there, in either run, and dq with it
    v2 = v2.double().flatten(0, 2).norm(dim=1).max()
    ds = 2.0 ** -24 * 2 * float(do.double().flatten(0, 2).norm(dim=1).max() * v2) / 2.0 ** 14
    room = d ** -0.5 * ds * k.double().abs().sum(1, keepdim=True).repeat_interleave(h // hk, 2)
    assert ((x.double() - y.double()).abs() <= room + 2 * 2.0 ** -11 * y.double().abs() + FLOOR[HF]).all()


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF), (128, HF), (40, SF)], ids=str)
def test_keys_of_other_rows_do_not_touch_a_row(d, dtype):
    """Few rows with spans of their own: keys that half of them see may be large, and move no bit of the others.  So many
    sequences that a warp goes from keys that all rows see to these."""
    from flashdiffusion_b200.attention import Spans, attend
    b, sq, sk, h, hk = 400, 4, 256, 8, 2
    q, k, v, _ = _inputs(b, sq, sk, h, hk, d, dtype, seed=103)
    first = torch.tensor([72, 64, 72, 64], dtype=torch.int32, device="cuda")
    spans = Spans(first, torch.full_like(first, 230))
    want = attend(q, k, v, spans=spans)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[:, 66:72] *= 24
    got = attend(q, k2, v2, spans=spans)
    assert torch.equal(got[:, 0::2], want[:, 0::2]) and not torch.equal(got[:, 1::2], want[:, 1::2])


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
def test_very_long_rows_in_one_part(dtype):
    """131072 keys a row, and so many query tiles that the key axis is not cut: what the accumulator loses by adding up
    values of one sign, rounding toward zero, stays inside its bound."""
    from flashdiffusion_b200.attention import attend
    sq, sk, h, d = 512, 131072, 40, 64
    g = torch.Generator(device="cuda").manual_seed(105)
    q, k, v = (torch.randn(1, n, x, d, device="cuda", generator=g).to(dtype) for n, x in ((sq, h), (sk, 1), (sk, 1)))
    v = v.abs()
    o = attend(q, k, v)
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    for head in (0, h - 1):
        s = q[0, :, head].double() @ k[0, :, 0].double().T * d ** -0.5
        size = float((q[0, :, head].double().abs() @ k[0, :, 0].double().abs().T).max()) * d ** -0.5
        want = torch.softmax(s, -1) @ v[0, :, 0].double()
        es = 2 * (d + 8) * w * size + 8 * w * (float(s.abs().max()) + 1)
        # the weights' and the output's rounding; scores and exponentials; one last place for each step of 16 keys; the
        # sum of weights, tile by tile
        rel = 2 * u + 2 * es + 8e-6 + sk / 16 * 2.0 ** -23 + 2 * (sk / 128 + 64) * w
        assert ((o[0, :, head].double() - want).abs() <= rel * want).all()
