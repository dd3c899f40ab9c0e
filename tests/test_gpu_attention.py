"""attend and attend_cached against their definition in 64 bits (tests/attention_reference.py, where the bounds come from)."""
import pytest
import torch

from tests.attention_reference import check, reference, spans_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    """A bounded wait that gives up leaves its mark in the status word and its results unfinished."""
    yield
    from flashdiffusion_b200 import native
    native.check_status()

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
# fp16 holds nothing finer than 2^-25 absolute: outputs that small, and the ds values they are summed from
FLOOR = {BF: 0.0, HF: 2.0 ** -25, SF: 0.0}


def _inputs(b, sq, sk, h, hk, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return mk(b, sq, h, d), mk(b, sk, hk, d), mk(b, sk, hk, d), mk(b, sq, h, d)


def _run(q, k, v, do, grad=True, **kw):
    from flashdiffusion_b200.attention import attend
    q, k, v = (t.detach().requires_grad_(grad) for t in (q, k, v))
    o, lse = attend(q, k, v, return_lse=True, **kw)
    out = {"o": o, "lse": lse}
    if grad:
        out["dq"], out["dk"], out["dv"] = torch.autograd.grad(o, (q, k, v), do)
    return out


def _compare(out, ref, dtype):
    for name in out:
        check(name, out[name], ref, 0.0 if name == "lse" else FLOOR[dtype])


SHAPES = [
    (1, 1, 1, 1, 1, 64), (2, 77, 77, 4, 4, 64), (1, 128, 128, 2, 1, 128), (1, 129, 257, 6, 2, 128), (2, 300, 300, 4, 2, 96),
    (1, 5, 640, 8, 2, 128), (1, 260, 40, 2, 2, 64), (3, 31, 513, 3, 1, 72),
]


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, causal, dtype):
    b, sq, sk, h, hk, d = shape
    q, k, v, do = _inputs(*shape, dtype, seed=sq + sk)
    lo, hi, pos = spans_of(sq, sk, b, causal=causal)
    _compare(_run(q, k, v, do, causal=causal), reference(q, k, v, lo, hi, pos, do=do), dtype)


@pytest.mark.parametrize("dtype,d", [(SF, 64), (SF, 20), (SF, 256), (BF, 7), (HF, 160), (BF, 200)], ids=str)
def test_general_path_types_and_head_sizes(dtype, d):
    q, k, v, do = _inputs(2, 45, 70, 4, 2, d, dtype, seed=d)
    slopes = torch.tensor([0.5, 0.1, 0.0, -0.02], device="cuda")
    lo, hi, pos = spans_of(45, 70, 2, causal=True, window=33)
    out = _run(q, k, v, do, causal=True, window=33, cap=15.0, slopes=slopes)
    _compare(out, reference(q, k, v, lo, hi, pos, cap=15.0, slopes=slopes, do=do), dtype)


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [
    dict(cap=5.0), dict(cap=30.0, causal=True), dict(slopes=True), dict(slopes=True, causal=True),
    dict(cap=8.0, slopes=True, causal=True, window=50), dict(causal=True, window=1), dict(causal=True, window=130),
    dict(causal=True, window=2 ** 31 - 1), dict(scale=0.7), dict(scale=-0.3, causal=True), dict(scale=0.0),
], ids=str)
def test_scores(kw, d, dtype):
    kw = dict(kw)
    q, k, v, do = _inputs(2, 200, 333, 4, 2, d, dtype, seed=7)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.tensor([0.3, 0.05, 0.004, 0.0], device="cuda")
    lo, hi, pos = spans_of(200, 333, 2, causal=kw.get("causal", False), window=kw.get("window"))
    out = _run(q, k, v, do, **kw)
    ref = reference(q, k, v, lo, hi, pos, scale=kw.get("scale"), cap=kw.get("cap", 0.0), slopes=kw.get("slopes"), do=do)
    _compare(out, ref, dtype)


@pytest.mark.parametrize("scale", [1e-12, 1e9])
def test_cap_with_extreme_scales(scale):
    """Products that vanish under the cap, and a slope of the tanh whose powers leave fp32 (rows of zeros among them)."""
    q, k, v, do = _inputs(1, 140, 140, 2, 1, 64, BF, seed=9)
    q[:, 5], k[:, 9] = 0, 0
    lo, hi, pos = spans_of(140, 140, 1)
    out = _run(q, k, v, do, cap=2.0, scale=scale, grad=False)
    _compare(out, reference(q, k, v, lo, hi, pos, cap=2.0, scale=scale), BF)


def test_large_scores_and_cap_at_its_ends():
    """Scores of hundreds: without a cap one key takes all, with one the tanh is flat at both ends."""
    q, k, v, do = _inputs(1, 150, 150, 2, 2, 64, BF, seed=3)
    q = q * 20
    for cap in (0.0, 3.0, 50.0):
        lo, hi, pos = spans_of(150, 150, 1, causal=True)
        out = _run(q, k, v, do, causal=True, cap=cap or None)
        _compare(out, reference(q, k, v, lo, hi, pos, cap=cap, do=do), BF)


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, HF), (40, SF)], ids=str)
@pytest.mark.parametrize("causal,window,prefix", [(True, None, False), (False, None, False), (True, 20, False),
                                                  (True, None, True)])
def test_documents(causal, window, prefix, d, dtype):
    from flashdiffusion_b200.attention import document_spans
    offsets = [3, 4, 4, 140, 141, 290, 401]          # rows 0..2 and 401.. are padding; one document is empty
    rows = 430
    q, k, v, do = _inputs(1, rows, rows, 3, 1, d, dtype, seed=11)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    pre = torch.tensor([1, 9, 40, 0, 500, 16], dtype=torch.int32, device="cuda") if prefix else None
    spans = document_spans(off, rows, causal=causal, window=window, prefix=pre)
    first, end = torch.zeros(1, rows, dtype=torch.long), torch.zeros(1, rows, dtype=torch.long)
    for n, (a, z) in enumerate(zip(offsets[:-1], offsets[1:])):
        for i in range(a, z):
            first[0, i] = max(a, i - window + 1) if window else a
            end[0, i] = i + 1 if causal else z
            if prefix:
                end[0, i] = min(z, max(i + 1, a + int(pre[n])))
    empty = end[0] <= first[0]
    assert torch.equal((spans.end <= spans.first)[0].cpu(), empty)
    assert torch.equal(spans.first[0].cpu()[~empty], first[0][~empty].int())
    assert torch.equal(spans.end[0].cpu()[~empty], end[0][~empty].int())
    lo, hi, pos = spans_of(rows, rows, 1, first=first, end=end)
    out = _run(q, k, v, do, spans=spans)
    _compare(out, reference(q, k, v, lo, hi, pos, do=do), dtype)
    assert (out["o"][0, empty.cuda()] == 0).all() and (out["lse"][0][:, empty.cuda()] == float("-inf")).all()
    assert (out["dq"][0, empty.cuda()] == 0).all()
    assert (out["dk"][0, 401:] == 0).all() and (out["dv"][0, :3] == 0).all()


@pytest.mark.parametrize("sq,sk", [(200, 200), (130, 333)])
def test_prefix(sq, sk):
    from flashdiffusion_b200.attention import prefix_spans
    q, k, v, do = _inputs(4, sq, sk, 4, 2, 128, BF, seed=5)
    pre = torch.tensor([0, 1, 150, 10 ** 6], dtype=torch.int32, device="cuda")
    i = torch.arange(sq)[None] + sk - sq
    end = torch.maximum(i + 1, pre.cpu().long()[:, None])
    lo, hi, pos = spans_of(sq, sk, 4, first=torch.zeros_like(end), end=end)
    slopes = torch.tensor([0.2, 0.1, 0.05, 0.025], device="cuda")
    out = _run(q, k, v, do, spans=prefix_spans(pre, sq, sk), slopes=slopes)
    _compare(out, reference(q, k, v, lo, hi, pos, slopes=slopes, do=do), BF)


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF), (24, SF)], ids=str)
def test_any_spans(d, dtype):
    """Spans in no order, out of range, crossed and empty."""
    from flashdiffusion_b200.attention import Spans
    sq, sk = 270, 401
    q, k, v, do = _inputs(2, sq, sk, 2, 1, d, dtype, seed=13)
    g = torch.Generator().manual_seed(1)
    first = torch.randint(-50, sk + 50, (2, sq), generator=g, dtype=torch.int32)
    end = first + torch.randint(-20, 300, (2, sq), generator=g, dtype=torch.int32)
    end[0, 5], first[0, 6], end[0, 6] = -(2 ** 31), -(2 ** 31), 2 ** 31 - 1
    lo, hi, pos = spans_of(sq, sk, 2, first=first, end=end)
    out = _run(q, k, v, do, spans=Spans(first.cuda(), end.cuda()))
    _compare(out, reference(q, k, v, lo, hi, pos, do=do), dtype)
    one = Spans(first[0].cuda(), end[0].cuda())          # the same spans for every batch entry
    lo, hi, pos = spans_of(sq, sk, 2, first=first[:1], end=end[:1])
    _compare(_run(q, k, v, do, spans=one), reference(q, k, v, lo, hi, pos, do=do), dtype)


@pytest.mark.parametrize("dtype", [BF, HF, SF], ids=str)
def test_layouts_and_strides(dtype):
    """Packed qkv, head-major tensors, odd offsets, expanded keys, tensors without a batch axis: the same bits as contiguous ones."""
    from flashdiffusion_b200.attention import attend
    b, s, h, d = 2, 150, 4, 64
    q, k, v, do = _inputs(b, s, s, h, h, d, dtype, seed=17)
    want = _run(q, k, v, do, causal=True)
    qkv = torch.stack([q, k, v], 2)
    views = {
        "packed": qkv.unbind(2),
        "head-major": [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)],
        "padded": [torch.nn.functional.pad(t, (0, 8))[..., :d] for t in (q, k, v)],
        "last-major": [t.transpose(1, 3).contiguous().transpose(1, 3) for t in (q, k, v)],
    }
    for name, (a, b_, c) in views.items():
        got = _run(a, b_, c, do.transpose(1, 2).contiguous().transpose(1, 2), causal=True)
        for n in got:
            assert torch.equal(got[n], want[n]), (name, n)
    # odd element offsets take other kernels: compared by value
    odd = [torch.nn.functional.pad(t, (1, 1))[..., 1:d + 1] for t in (q, k, v)]
    lo, hi, pos = spans_of(s, s, b, causal=True)
    _compare(_run(*odd, do, causal=True), reference(q, k, v, lo, hi, pos, do=do), dtype)
    flat = attend(q[0], k[0], v[0], causal=True)
    assert torch.equal(flat, attend(q[:1], k[:1], v[:1], causal=True)[0])
    # one key sequence shared by the batch: its gradient is the sum over the batch
    ke = k[:1].expand(b, s, h, d)
    got = _run(q, ke, v, do, causal=True)
    _compare(got, reference(q, ke, v, lo, hi, pos, do=do), dtype)
    leaf = k[:1].clone().requires_grad_(True)
    o = attend(q, leaf.expand(b, s, h, d), v, causal=True)
    shared = torch.autograd.grad(o, leaf, do)[0]
    u = torch.finfo(dtype).eps / 2
    assert ((shared - got["dk"].float().sum(0, keepdim=True)).abs() <= 3 * u * got["dk"].float().abs().sum(0) + 1e-6).all()
    # an expanded gradient, as the sum of the output gives
    leaf = q.clone().requires_grad_(True)
    dq = torch.autograd.grad(attend(leaf, k, v, causal=True).sum(), leaf)[0]
    ref = reference(q, k, v, lo, hi, pos, do=torch.ones_like(do))
    check("dq", dq, ref, FLOOR[dtype])


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (SF, 48)], ids=str)
def test_masked_places_hold_anything(dtype, d):
    """NaN and infinities behind the last document, and in its padding rows of q and do, change nothing."""
    from flashdiffusion_b200.attention import document_spans
    rows, used = 300, 210
    q, k, v, do = _inputs(1, rows, rows, 2, 2, d, dtype, seed=19)
    off = torch.tensor([0, 100, used], dtype=torch.int32, device="cuda")
    spans = document_spans(off, rows)
    want = _run(q, k, v, do, spans=spans)
    for bad in (float("nan"), float("inf"), -float("inf")):
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        for t in (q2, k2, v2, do2):
            t[:, used:] = bad
        got = _run(q2, k2, v2, do2, spans=spans)
        for n in got:
            assert torch.equal(got[n], want[n]), (n, bad)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (SF, 48)], ids=str)
def test_masked_places_hold_anything_under_a_cap(dtype, d):
    """The same with capped scores, whose slope 1 - tanh^2 is a NaN in such places, and a bias."""
    from flashdiffusion_b200.attention import Spans
    s = 300
    q, k, v, do = _inputs(1, s, s, 4, 2, d, dtype, seed=63)
    first, end = torch.full((s,), 7, dtype=torch.int32), torch.arange(s).clamp(max=250).int()
    slopes = torch.tensor([0.1, 0.0, 0.01, 0.5], device="cuda")
    kw = dict(spans=Spans(first.cuda(), end.cuda()), cap=6.0, slopes=slopes)
    want = _run(q, k, v, do, **kw)
    for bad in (float("nan"), float("inf"), -float("inf")):
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        for t in (q2, do2):
            t[:, :8] = bad                                 # rows that see nothing
        for t in (k2, v2):
            t[:, :7], t[:, 250:] = bad, bad                # keys that nobody sees
        got = _run(q2, k2, v2, do2, **kw)
        for n in got:
            assert torch.equal(got[n], want[n]), (n, bad)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (SF, 48)], ids=str)
def test_causal_future_holds_anything(dtype, d):
    """A NaN or infinity in a key or value reaches the rows that see it and no other."""
    s, at = 300, 170
    q, k, v, do = _inputs(1, s, s, 2, 2, d, dtype, seed=23)
    want = _run(q, k, v, do, causal=True, grad=False)
    for bad in (float("nan"), float("inf")):
        v2 = v.clone()
        v2[:, at, :, 3] = bad
        got = _run(q, k, v2, do, causal=True, grad=False)
        assert torch.equal(got["o"][:, :at], want["o"][:, :at])
        assert not torch.isfinite(got["o"][:, at:, :, 3]).any()
        assert torch.equal(got["o"][:, at:, :, 4:], want["o"][:, at:, :, 4:])
        k2 = k.clone()
        k2[:, at] = bad
        got = _run(q, k2, v, do, causal=True, grad=False)
        assert torch.equal(got["o"][:, :at], want["o"][:, :at])
        assert not torch.isfinite(got["o"][:, at + 1:]).all(-1).any()
    want = _run(q, k, v, do, causal=True)
    # gradients: a row's NaN stays out of the keys that the row does not see
    for which in ("q", "do"):
        q2, do2 = q.clone(), do.clone()
        (q2 if which == "q" else do2)[:, at] = float("nan")
        got = _run(q2, k, v, do2, causal=True)
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:, at + 1:], want[n][:, at + 1:]), (which, n)
        assert not torch.isfinite(got["dk"][:, :at + 1]).any()
        assert torch.equal(got["dq"][:, :at], want["dq"][:, :at]) and torch.equal(got["dq"][:, at + 1:], want["dq"][:, at + 1:])
    k2 = k.clone()
    k2[:, at] = float("nan")
    got = _run(q, k2, v, do, causal=True)
    assert torch.equal(got["dq"][:, :at], want["dq"][:, :at])


def test_empty_sizes():
    from flashdiffusion_b200.attention import attend, attend_cached
    q, k, v, do = _inputs(2, 5, 0, 2, 1, 64, BF)
    out = _run(q, k, v, do)
    assert (out["o"] == 0).all() and (out["lse"] == float("-inf")).all() and (out["dq"] == 0).all()
    q, k, v, do = _inputs(2, 0, 9, 2, 1, 64, BF)
    out = _run(q, k, v, do)
    assert out["o"].shape == (2, 0, 2, 64) and (out["dk"] == 0).all() and (out["dv"] == 0).all()
    assert attend(*(torch.empty(0, 4, 2, 64, device="cuda", dtype=BF) for _ in range(3))).shape == (0, 4, 2, 64)
    q, k, v, _ = _inputs(3, 1, 16, 2, 1, 64, BF)
    o = attend_cached(q, k, v, torch.tensor([0, 1, -7], dtype=torch.int32, device="cuda"))
    assert (o[0] == 0).all() and (o[2] == 0).all() and torch.equal(o[1, 0], v[1, 0].expand(2, 64))


def test_same_bits_again():
    q, k, v, do = _inputs(2, 513, 513, 6, 2, 128, BF, seed=29)
    a = _run(q, k, v, do, causal=True, cap=20.0)
    for _ in range(3):
        b = _run(q, k, v, do, causal=True, cap=20.0)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_gradient_against_differences():
    """fp32 heads: the derivative along a random direction against central differences of the loss in 64 bits."""
    q, k, v, do = _inputs(1, 40, 55, 2, 1, 32, SF, seed=31)
    slopes = torch.tensor([0.1, 0.01], device="cuda")
    out = _run(q, k, v, do, causal=True, cap=4.0, slopes=slopes)
    g = torch.Generator(device="cuda").manual_seed(2)
    lo, hi, pos = spans_of(40, 55, 1, causal=True)
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
        e = torch.randn(t.shape, device="cuda", generator=g)
        ends = []
        for sign in (1, -1):
            moved = {"dq": q, "dk": k, "dv": v} | {n: (t.double() + sign * 1e-4 * e.double())}
            o = _exact_output(moved["dq"].double(), moved["dk"].double(), moved["dv"].double(), lo, hi, pos, 4.0, slopes)
            ends.append(float((o * do.cpu().double()).sum()))
        want = (ends[0] - ends[1]) / 2e-4
        got = float((out[n].double() * e.double()).sum())
        # differences: third derivatives of order 1 times 1e-8 per direction of 1760 coordinates; kernel: fp32 rounding
        assert abs(got - want) <= 1e-4 * (1 + float((out[n].double() * e.double()).abs().sum())), (n, got, want)


def _exact_output(q, k, v, lo, hi, pos, cap, slopes):
    return reference(q, k, v, lo, hi, pos, cap=cap, slopes=slopes)["o"]


@pytest.mark.parametrize("dtype", [BF, HF, SF], ids=str)
@pytest.mark.parametrize("new,h,hk,d,cap,window", [
    (1, 8, 2, 128, None, None), (1, 8, 8, 64, 30.0, None), (4, 8, 2, 128, None, 100), (2, 5, 1, 64, 10.0, None),
    (1, 32, 1, 128, None, None), (3, 24, 2, 96, None, 1), (1, 7, 7, 40, None, None), (17, 4, 2, 128, None, None),
])
def test_cached(new, h, hk, d, cap, window, dtype):
    from flashdiffusion_b200.attention import attend_cached
    capacity = 1100
    lengths = [1, 2, 63, 64, 65, 300, 1000, capacity, capacity + 5, 0]
    q, k, v, _ = _inputs(len(lengths), new, capacity, h, hk, d, dtype, seed=new + h)
    n = torch.tensor(lengths, dtype=torch.int32)
    for b, m in enumerate(lengths):            # the cache behind the length was never written
        k[b, m:] = float("nan")
        v[b, m:] = float("inf")
    slopes = torch.linspace(0.5, 0.001, h, device="cuda")
    lo, hi, pos = spans_of(new, capacity, len(lengths), causal=True, window=window, lengths=n)
    o, lse = attend_cached(q, k, v, n.cuda(), cap=cap, window=window, slopes=slopes, return_lse=True)
    ref = reference(q, k, v, lo, hi, pos, cap=cap or 0.0, slopes=slopes)
    check("o", o, ref, FLOOR[dtype])
    check("lse", lse, ref)


def test_cached_long_and_strided():
    """A cache longer than one split, in head-major memory, and a view of a larger cache."""
    from flashdiffusion_b200.attention import attend_cached
    q, k, v, _ = _inputs(2, 1, 20000, 8, 2, 128, BF, seed=41)
    n = torch.tensor([20000, 12345], dtype=torch.int32)
    lo, hi, pos = spans_of(1, 20000, 2, causal=True, lengths=n)
    ref = reference(q, k, v, lo, hi, pos)
    a = attend_cached(q, k, v, n.cuda())
    check("o", a, ref)
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    assert torch.equal(attend_cached(q, kt, vt, n.cuda()), a)
    big = torch.randn(2, 20000, 4, 256, device="cuda").to(BF)
    big[:, :, 1:3, 64:192] = k
    assert torch.equal(attend_cached(q, big[:, :, 1:3, 64:192], v, n.cuda()), a)


def test_from_a_thread_that_has_no_context_yet():
    """The first CUDA call of a new thread may be the operator's own (an autograd worker's is)."""
    import ctypes
    import threading

    from flashdiffusion_b200 import attention as A
    from flashdiffusion_b200 import native
    q, k, v, _ = _inputs(1, 130, 130, 2, 1, 64, BF)
    want = A.attend(q, k, v)
    o = torch.zeros_like(q)
    torch.cuda.synchronize()
    args = A._arguments(q, k, v, o, None, None, (None, False, 0, None, None, 64 ** -0.5, 0.0))
    stream = torch.cuda.current_stream().cuda_stream
    got = []

    def work():
        got.append(native.load().fd_attention_forward(args, None, 0, ctypes.c_void_p(stream)))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert got == [native.FD_OK] and torch.equal(o, want)


def test_no_second_derivative():
    from flashdiffusion_b200.attention import attend
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    q, k, v, do = _inputs(1, 8, 8, 2, 1, 64, BF)
    a = q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(attend(a, k, v), a, do, create_graph=True)
    r = apply_rotary(a, positions=torch.arange(8, device="cuda"), freqs=rotary_frequencies(64))
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(r, a, do, create_graph=True)


def test_refuses_on_the_device():
    from flashdiffusion_b200.attention import Spans, attend, attend_cached
    q, k, v, _ = _inputs(2, 8, 8, 4, 2, 64, BF)
    with pytest.raises(ValueError):
        attend_cached(q.requires_grad_(True), k, v, torch.tensor([8, 8], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        attend_cached(q.detach(), k, v, torch.tensor([8], dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        attend_cached(q.detach(), k, v, torch.tensor([8, 8], device="cuda"))
    s = torch.zeros(7, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        attend(q, k, v, spans=Spans(s, s))
    with pytest.raises(ValueError):
        attend(q, k, v, spans=Spans(s.cpu(), s.cpu()))


def test_other_stream_and_captured_graph():
    """Forward and backward on a side stream, and captured and replayed on new inputs, give the eager bits."""
    from flashdiffusion_b200.attention import attend, attend_cached
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies
    q, k, v, do = _inputs(1, 200, 200, 4, 2, 128, BF, seed=43)
    q2, k2, v2, do2 = _inputs(1, 200, 200, 4, 2, 128, BF, seed=44)
    f, pos = rotary_frequencies(128), torch.arange(200, device="cuda")
    n = torch.tensor([150], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = attend(*apply_rotary(a, b, positions=pos, freqs=f), c, causal=True, cap=20.0)
        with torch.no_grad():
            last = attend_cached(q[:, -1:], k, v, n)
        return (o.detach(), last, *torch.autograd.grad(o, (a, b, c), do))

    want = [step(q, k, v, do), step(q2, k2, v2, do2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, v, do)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    ins = [t.clone() for t in (q, k, v, do)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*ins)
    for new, w in (((q2, k2, v2, do2), want[1]), ((q, k, v, do), want[0])):
        for t, x in zip(ins, new):
            t.copy_(x)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(outs, w))


@pytest.mark.parametrize("dtype,d", [(SF, 64), (SF, 33), (SF, 128), (HF, 200), (BF, 256), (BF, 20)], ids=str)
def test_general_path_tiles(dtype, d):
    """More rows than the general path takes one by one: whole tiles, ends inside tiles, shared heads, a window, and
    keys and rows outside the spans that hold anything."""
    from flashdiffusion_b200.attention import Spans
    b, sq, sk, h, hk = 2, 300, 333, 4, 2
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=d)
    lo, hi, pos = spans_of(sq, sk, b, causal=True, window=150)
    ref = reference(q, k, v, lo, hi, pos, do=do)
    _compare(_run(q, k, v, do, causal=True, window=150), ref, dtype)
    g = torch.Generator().manual_seed(d)
    lo = torch.randint(10, 200, (b, sq), generator=g).int()
    hi = (lo + torch.randint(0, 140, (b, sq), generator=g)).clamp(max=321).int()
    for x in range(b):
        for t in (k, v):
            t[x, :10], t[x, 321:] = float("nan"), float("inf")
        q[x, hi[x] <= lo[x]] = float("nan")
        do[x, hi[x] <= lo[x]] = float("inf")
    ref = reference(q, k, v, lo, hi, pos, cap=9.0, do=do)
    _compare(_run(q, k, v, do, spans=Spans(lo.cuda(), hi.cuda()), cap=9.0), ref, dtype)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (BF, 80)], ids=str)
@pytest.mark.parametrize("b,sq,sk,h,hk,window", [
    (1, 300, 3001, 2, 1, None), (2, 130, 1100, 4, 1, 700), (1, 1500, 1500, 4, 1, None), (1, 2100, 140, 1, 1, None),
    (1, 1400, 1400, 3, 1, 300),
])
def test_split_axes(b, sq, sk, h, hk, window, dtype, d):
    """Few tiles for many SMs: keys (forward, dq) and queries (dk, dv) are cut into parts that are joined."""
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=sk)
    lo, hi, pos = spans_of(sq, sk, b, causal=True, window=window)
    out = _run(q, k, v, do, causal=True, window=window)
    _compare(out, reference(q, k, v, lo, hi, pos, do=do), dtype)
    again = _run(q, k, v, do, causal=True, window=window)
    assert all(torch.equal(out[n], again[n]) for n in out)


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
def test_split_axes_with_anything_in_masked_places(dtype):
    from flashdiffusion_b200.attention import Spans
    b, sq, sk, h, hk, d = 1, 700, 2500, 3, 1, 128
    q, k, v, do = _inputs(b, sq, sk, h, hk, d, dtype, seed=61)
    g = torch.Generator().manual_seed(61)
    lo = torch.randint(5, 1500, (b, sq), generator=g).int()
    hi = (lo + torch.randint(0, 900, (b, sq), generator=g) * torch.randint(0, 2, (b, sq), generator=g)).int()
    hi = hi.clamp(max=2390)
    empty = hi[0] <= lo[0]
    for t in (k, v):
        t[0, :5], t[0, 2390:] = float("inf"), float("nan")
    q[0, empty], do[0, empty] = float("nan"), float("inf")
    pos = spans_of(sq, sk, b)[2]
    slopes = torch.tensor([0.001, 0.0, 0.01], device="cuda")
    kw = dict(spans=Spans(lo.cuda(), hi.cuda()), cap=8.0, slopes=slopes)
    _compare(_run(q, k, v, do, **kw), reference(q, k, v, lo, hi, pos, cap=8.0, slopes=slopes, do=do), dtype)
    # a visible infinity of dO reaches dV of the keys that its row sees, and no other's
    clean = _run(q, k, v, do, **kw)
    i = int((hi[0] - lo[0]).argmax())
    do2 = do.clone()
    do2[0, i, 1, 7] = float("inf")
    got = _run(q, k, v, do2, **kw)["dv"]
    inside = torch.zeros(sk, dtype=torch.bool, device="cuda")
    inside[lo[0, i]:hi[0, i]] = True
    assert not torch.isfinite(got[0, inside, 0, 7]).any()
    assert torch.equal(got[0, ~inside], clean["dv"][0, ~inside])


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("new,h,hk,d,cap,window", [(1, 8, 2, 256, None, None), (3, 4, 4, 136, 20.0, None),
                                                   (1, 5, 1, 192, None, 90), (140, 2, 1, 256, None, None)])
def test_wide_heads_against_a_cache(new, h, hk, d, cap, window, dtype):
    from flashdiffusion_b200.attention import attend_cached
    capacity = 2000
    lengths = [1, 0, 127, 128, 129, 1000, capacity]
    q, k, v, _ = _inputs(len(lengths), new, capacity, h, hk, d, dtype, seed=d)
    n = torch.tensor(lengths, dtype=torch.int32)
    for b, m in enumerate(lengths):
        k[b, m:] = float("nan")
        v[b, m:] = float("inf")
    slopes = torch.linspace(0.5, 0.001, h, device="cuda")
    lo, hi, pos = spans_of(new, capacity, len(lengths), causal=True, window=window, lengths=n)
    o, lse = attend_cached(q, k, v, n.cuda(), cap=cap, window=window, slopes=slopes, return_lse=True)
    ref = reference(q, k, v, lo, hi, pos, cap=cap or 0.0, slopes=slopes)
    check("o", o, ref, FLOOR[dtype])
    check("lse", lse, ref)


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("d", [136, 256])
def test_wide_heads_forward(d, dtype):
    """Enough tiles not to be split; ends inside tiles, strided views, a visible infinity."""
    b, sq, sk, h, hk = 3, 700, 390, 14, 2
    q, k, v, _ = _inputs(b, sq, sk, h, hk, d, dtype, seed=65)
    v[1, 300, 0, 3] = float("inf")
    lo, hi, pos = spans_of(sq, sk, b, causal=True)
    wide = torch.randn(b, sk, 2 * hk, d, device="cuda").to(dtype)
    wide[:, :, hk:] = k
    got = _run(q, wide[:, :, hk:], v, None, grad=False, causal=True)
    vr = v.clone()
    vr[1, 300, 0, 3] = 0
    ref = reference(q, k, vr, lo, hi, pos)
    check("lse", got["lse"], ref)
    sees = (hi[1] > 300).cuda()
    spoiled = got["o"][1, :, :7, 3]
    assert (spoiled[sees] == float("inf")).all() and torch.isfinite(spoiled[~sees]).all()
    o = got["o"].clone()
    o[1, sees, :7, 3] = ref["o"][1, sees.cpu(), :7, 3].to(o)
    check("o", o, ref, FLOOR[dtype])


@pytest.mark.parametrize("dtype,d", [(BF, 64), (SF, 16)], ids=str)
def test_very_many_heads(dtype, d):
    """More (sequence, head) pairs than a grid's second axis holds."""
    from flashdiffusion_b200.attention import attend
    q, k, v, _ = _inputs(2100, 1, 3, 32, 32, d, dtype)
    o = attend(q, k, v).double()
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * d ** -0.5
    p = torch.softmax(s, -1)
    u = torch.finfo(dtype).eps / 2
    # the reference module's bound with scores of D + 8 roundings, their sum at most 8 sqrt(d) here
    rel = u + 2 * (2 * (d + 8) * 2.0 ** -24 * 8 * d ** 0.5) + 2e-5
    want, room = (torch.einsum("bhij,bjhd->bihd", p, x) for x in (v.double(), v.double().abs()))
    assert float(s.abs().max()) < 8 * d ** 0.5
    assert ((o - want).abs() <= u * want.abs() + rel * room + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF, SF], ids=str)
def test_one_tensor_in_every_place(dtype):
    """attend(x, x, x): the gradient of x is the sum of the three."""
    from flashdiffusion_b200.attention import attend
    x, _, _, do = _inputs(1, 140, 140, 2, 2, 64, dtype, seed=51)
    lo, hi, pos = spans_of(140, 140, 1, causal=True)
    ref = reference(x, x, x, lo, hi, pos, do=do)
    x.requires_grad_(True)
    o = attend(x, x, x, causal=True)
    dx, = torch.autograd.grad(o, x, do)
    total = sum(ref[n] for n in ("dq", "dk", "dv"))
    u = torch.finfo(dtype).eps / 2
    # two additions of rounded gradients, each rounded again: partial sums stay below the three sizes' sum
    size = sum(ref[n].abs() + ref[n + "_tol"] for n in ("dq", "dk", "dv"))
    check("dx", dx, {"dx": total, "dx_tol": sum(ref[n + "_tol"] for n in ("dq", "dk", "dv")) + 2 * u * size})


@pytest.mark.parametrize("d,dtype", [(64, BF), (64, SF)], ids=str)
def test_offsets_beyond_32_bits(d, dtype):
    """A cache of more than 2^31 elements: only its end is written, read and compared."""
    from flashdiffusion_b200.attention import Spans, attend, attend_cached
    rows = 2 ** 31 // d + 700
    q, k, v, _ = _inputs(1, 3, 600, 4, 1, d, dtype, seed=53)
    kc, vc = (torch.empty(1, rows, 1, d, dtype=dtype, device="cuda") for _ in "kv")
    kc[:, -600:], vc[:, -600:] = k, v
    n = torch.tensor([rows], dtype=torch.int32, device="cuda")
    lo, hi, pos = spans_of(3, 600, 1, causal=True, window=500)
    ref = reference(q, k, v, lo, hi, pos)
    check("o", attend_cached(q, kc, vc, n, window=500), ref, FLOOR[dtype])
    many = torch.randn(1, 1200, 4, d, device="cuda").to(dtype)
    at = torch.arange(1200, device="cuda", dtype=torch.int32) % 100 + (rows - 300)
    lo, hi, pos = spans_of(1200, 600, 1, first=(at - (rows - 600)).cpu(), end=(at - (rows - 600)).cpu() + 77)
    ref = reference(many, k, v, lo, hi, pos)
    check("o", attend(many, kc, vc, spans=Spans(at, at + 77)), ref, FLOOR[dtype])


@pytest.mark.parametrize("dtype", [BF, HF, SF], ids=str)
def test_two_streams_at_once(dtype):
    """Training steps and cache reads in flight on two streams together give the bits that each gives alone."""
    from flashdiffusion_b200.attention import attend, attend_cached
    sets = [_inputs(2, 500, 500, 8, 2, 64, dtype, seed=s) for s in (55, 56)]
    n = torch.tensor([500, 77], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = attend(a, b, c, causal=True)
        return (o.detach(), attend_cached(q[:, -2:], k, v, n), *torch.autograd.grad(o, (a, b, c), do))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, (stream, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(step(*s))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, y) for g in got[i] for x, y in zip(g, want[i]))


def test_two_threads_at_once():
    """Two host threads, each with its own stream, type and head size, give the bits that each gives alone."""
    import threading

    from flashdiffusion_b200.attention import attend, attend_cached
    sets = [_inputs(1, 300, 300, 4, 2, d, t, seed=d) for d, t in ((64, HF), (128, BF))]
    n = torch.tensor([280], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = attend(a, b, c, causal=True, cap=20.0)
        return (o.detach(), attend_cached(q[:, -1:], k, v, n), *torch.autograd.grad(o, (a, b, c), do))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(*sets[i])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:       # what a thread raises is lost otherwise
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", [BF, HF, SF], ids=str)
def test_two_captured_graphs_of_one_pool(dtype):
    """Two training steps captured into one memory pool and replayed in turn on changing inputs."""
    from flashdiffusion_b200.attention import attend, attend_cached
    sets = [_inputs(1, s, s, 4, 2, 128, dtype, seed=s) for s in (130, 390)]
    n = torch.tensor([100], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = attend(a, b, c, causal=True, cap=30.0)
        return (o.detach(), attend_cached(q[:, -1:], k, v, n), *torch.autograd.grad(o, (a, b, c), do))

    want = [[step(*s), step(*(t.flip(1) for t in s))] for s in sets]
    ins = [[t.clone() for t in s] for s in sets]
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(*x))
        graphs.append(g)
    for turn in (0, 1, 0):
        for i in (0, 1):
            for t, x in zip(ins[i], sets[i]):
                t.copy_(x.flip(1) if turn else x)
            graphs[i].replay()
            assert all(torch.equal(x, y) for x, y in zip(outs[i], want[i][turn]))


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
@pytest.mark.parametrize("dtype", [BF, SF], ids=str)
def test_captured_while_a_warm_up_graph_of_the_same_leaves_lives(dtype):
    """The warm-up ran on a side stream, as the documentation of capture asks, and its output is still referenced."""
    from flashdiffusion_b200.attention import attend
    q, k, v, do = _inputs(1, 200, 200, 4, 2, 128, dtype, seed=59)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = attend(*leaves, causal=True)
        warm.backward(do)
    torch.cuda.current_stream().wait_stream(side)
    want = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(*leaves, causal=True).backward(do)
    graph.replay()
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    del warm


def test_what_the_gradients_read_again_is_watched():
    """Spans, slopes and heads changed in place between the passes are refused, not used."""
    from flashdiffusion_b200.attention import Spans, attend
    q, k, v, do = _inputs(1, 20, 20, 2, 1, 64, BF)
    first, end = torch.zeros(20, dtype=torch.int32, device="cuda"), torch.full((20,), 20, dtype=torch.int32, device="cuda")
    slopes = torch.ones(2, device="cuda")
    for change in (lambda: end.fill_(3), lambda: slopes.zero_(), lambda: k.zero_()):
        o = attend(q.requires_grad_(True), k, v, spans=Spans(first, end), slopes=slopes)
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.backward(do)


def test_the_low_bits_of_the_output_serve_the_gradients():
    """Rows that cancel: dq of one query that looks at two keys whose values differ little.  dS = P (dP - delta) is then
    the small difference of large numbers; with delta from o rounded to bf16 it would be off by 2^-9 |dO . o|, with
    eight more bits by 2^-17 of it."""
    from flashdiffusion_b200.attention import attend
    d = 64
    q, k = (torch.randn(1, n, 1, d, device="cuda", generator=torch.Generator("cuda").manual_seed(57)).to(BF) for n in (1, 2))
    v = torch.ones(1, 2, 1, d, device="cuda", dtype=BF)
    v[0, 1] += 2.0 ** -6
    do = torch.ones(1, 1, 1, d, device="cuda", dtype=BF)
    lo, hi, pos = spans_of(1, 2, 1)
    ref = reference(q, k, v, lo, hi, pos, do=do)
    dq, = torch.autograd.grad(attend(q.requires_grad_(True), k, v), q, do)
    p = 0.25                                               # the largest p (1 - p)
    # ds = scale p0 p1 64 2^-6 <= p / 8; error of delta: 64 (2^-17 for the kept bits, 2^-20 for fp32 steps), of P: 2^-16
    ds_tol = d ** -0.5 * (2 * p * 64 * (2.0 ** -17 + 2.0 ** -20) + p * 2.0 ** -15) + 2.0 ** -8 * d ** -0.5 * p
    room = 2.0 ** -8 * ref["dq"].abs() + ds_tol * k.double().cpu().abs().sum(1, keepdim=True)
    assert ((dq.double().cpu() - ref["dq"]).abs() <= room).all()


def test_a_prompt_its_training_step_and_its_answers():
    """The operators together: rotate, attend over a packed prompt, gradients to the unrotated heads; then token by
    token against the cache, where each answer equals the prompt's row within both calls' rounding."""
    from flashdiffusion_b200.attention import attend, attend_cached
    from flashdiffusion_b200.rope import apply_rotary, rotary_frequencies, rotary_magnitude
    s, h, hk, d = 190, 8, 2, 128
    q, k, v, do = _inputs(1, s, s, h, hk, d, BF, seed=47)
    f = rotary_frequencies(d, scaling="parts", factor=4.0, trained=64, device="cuda")
    mag = rotary_magnitude(4.0)
    pos = torch.arange(s, device="cuda")
    a, b, c = (t.clone().requires_grad_(True) for t in (q, k, v))
    rq, rk = apply_rotary(a, b, positions=pos, freqs=f, magnitude=mag)
    o = attend(rq, rk, c, causal=True, cap=25.0)
    da, db, dc = torch.autograd.grad(o, (a, b, c), do)
    lo, hi, p = spans_of(s, s, 1, causal=True)
    ref = reference(rq, rk, v, lo, hi, p, cap=25.0, do=do)
    check("o", o, ref)
    check("dv", dc, ref)
    # the rotation's gradient: the reference's dq turned back, in fp32 on the same formula
    back = apply_rotary(ref["dq"].float().cuda(), positions=pos, freqs=f, magnitude=mag, inverse=True)
    room = apply_rotary(ref["dq_tol"].float().cuda(), positions=torch.zeros_like(pos), freqs=f, magnitude=mag)
    pair = room + room.roll(d // 2, -1)      # |cos| a + |sin| b of a pair, at most their sum
    size = ref["dq"].abs().float().cuda()
    u = 2.0 ** -8
    assert ((da.float() - back).abs() <= (pair + u * mag * (size + size.roll(d // 2, -1))) * 1.01 + 1e-6).all()
    kc = torch.full((1, 256, hk, d), float("nan"), device="cuda", dtype=BF)
    vc = torch.full_like(kc, float("nan"))
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        for t in range(s):
            tq, tk = apply_rotary(q[:, t:t + 1], k[:, t:t + 1], positions=pos[t:t + 1], freqs=f, magnitude=mag)
            kc[:, t:t + 1], vc[:, t:t + 1] = tk, v[:, t:t + 1]
            n += 1
            if t in (0, 1, 63, 64, 127, 128, s - 1):
                got = attend_cached(tq, kc, vc, n, cap=25.0)
                one = {"o": ref["o"][:, t:t + 1], "o_tol": ref["o_tol"][:, t:t + 1]}
                check("o", got, one)
