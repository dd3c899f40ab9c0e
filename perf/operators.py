"""Workloads of the rotary and attention operators: inputs, plain forms, exact values and the calls a program makes.

``run`` computes each operator in plain torch operations where ``own`` is false and through
``flashdiffusion_b200`` where it is true.  Three operators:

rotary   rotation of query and key heads by their positions (``rope.apply_rotary``), with gradients in training
attend   softmax attention over key spans with a tanh cap on the scores or a bias by distance
         (``attention.attend``), forward, and with gradients in training
cached   the same for the newest tokens of each sequence against a key/value cache (``attention.attend_cached``)
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotary(name, **kw):
    case = {"name": name, "op": "rotary", "batch": 1, "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 128, "rot": 128,
            "layout": "half", "dtype": "bf16", "scaling": "none", "factor": 1.0, "reach": 4096, "fractional": False,
            "grad": False}
    case.update(kw)
    return case


def _attend(name, **kw):
    case = {"name": name, "op": "attend", "batch": 1, "q_len": 1, "k_len": 1, "heads": 8, "kv_heads": 8, "dim": 128,
            "dtype": "bf16", "mask": "causal", "window": 0, "documents": 0, "cap": 0.0, "bias": False, "grad": False}
    case.update(kw)
    return case


def _cached(name, **kw):
    case = {"name": name, "op": "cached", "batch": 1, "new": 1, "shortest": 1, "longest": 1, "heads": 8, "kv_heads": 8,
            "dim": 128, "dtype": "bf16", "window": 0, "cap": 0.0, "bias": False}
    case.update(kw)
    return case


def listed():
    return [
        # one decoding step of a batch: the call is all latency; positions far beyond the trained length
        _rotary("rotary_step", batch=16, heads=32, kv_heads=8, scaling="parts", factor=8.0, reach=131072),
        # prompts of two sequences, grouped key heads
        _rotary("rotary_prompt", batch=2, tokens=4096, heads=32, kv_heads=8),
        # a training step that rotates part of each head, adjacent pairs, odd length
        _rotary("rotary_train_part", batch=3, tokens=1777, heads=16, kv_heads=16, dim=96, rot=64, layout="interleaved",
                dtype="fp16", scaling="linear", factor=4.0, grad=True),
        # samples of a time series at fractional positions, one vector per sample, as the series encoder has them
        _rotary("rotary_series", tokens=100001, heads=1, kv_heads=0, dim=64, rot=64, layout="interleaved",
                dtype="fp32", reach=100001, fractional=True),
        # a short sequence, every pair visible, forward and backward: launches and latency count
        _attend("attend_short", q_len=77, k_len=77, heads=4, kv_heads=4, dim=64, dtype="fp16", mask="full", grad=True),
        # the ordinary training step: causal, grouped heads
        _attend("attend_causal", batch=2, q_len=4096, k_len=4096, heads=16, kv_heads=4, grad=True),
        # a packed batch of ragged documents with capped scores; some padding rows behind the last one
        _attend("attend_documents", q_len=7001, k_len=7001, heads=12, kv_heads=12, dim=64, mask="documents",
                documents=9, cap=30.0, grad=True),
        # prefixes that every row sees, causal behind them, a bias that falls with distance
        _attend("attend_prefix", batch=4, q_len=1531, k_len=1531, heads=8, kv_heads=2, mask="prefix", bias=True,
                grad=True),
        # a long prompt with a sliding window and capped scores, forward only
        _attend("attend_long", q_len=16384, k_len=16384, heads=8, kv_heads=2, dtype="fp16", mask="window", window=4096,
                cap=50.0),
        # one token of one sequence: latency
        _cached("cached_one", shortest=2049, longest=2049, heads=32, kv_heads=8),
        # one token for each of a ragged batch
        _cached("cached_ragged", batch=48, longest=8192, heads=32, kv_heads=8, cap=50.0),
        # four tokens at once against very long caches
        _cached("cached_long", batch=3, new=4, shortest=40000, longest=131072, heads=16, kv_heads=2, dim=64,
                dtype="fp16", bias=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "cached"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rotary":
        kv = rng.choice([0, 1, 2, 4, 8])
        heads = max(1, kv) * rng.choice([1, 2, 4])
        dim = 8 * rng.randint(4, 16)
        rot = rng.choice([dim, dim, 16 * rng.randint(1, dim // 16)])
        layout = rng.choice(["half", "interleaved"])
        if layout == "half":
            rot -= rot % 16
        batch = _log_int(rng, 1, 16)
        tokens = _log_int(rng, 1, max(1, 20_000_000 // (batch * (heads + kv) * dim)))
        scaling = rng.choice(["none", "linear", "parts"])
        case = _rotary("", batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, rot=rot, layout=layout,
                       dtype=rng.choice(["bf16", "fp16", "fp32"]), scaling=scaling,
                       factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                       reach=_log_int(rng, tokens, 1 << 20), fractional=rng.random() < 0.2, grad=rng.random() < 0.4)
    elif op == "attend":
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2, 3, 4])
        batch = rng.choice([1, 1, 2, 3])
        mask = rng.choice(["full", "causal", "window", "documents", "prefix"])
        if mask == "documents":
            batch = 1
        k_len = _log_int(rng, 16, int(math.sqrt(2.5e8 / (batch * heads))))
        q_len = k_len if mask in ("documents", "prefix") or rng.random() < 0.6 else _log_int(rng, 1, k_len)
        case = _attend("", batch=batch, q_len=q_len, k_len=k_len, heads=heads, kv_heads=kv,
                       dim=rng.choice([64, 80, 96, 128, 128]), dtype=dtype, mask=mask,
                       window=rng.randint(1, k_len) if mask == "window" else 0,
                       documents=rng.randint(1, min(12, k_len // 8)) if mask == "documents" else 0,
                       cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3, grad=rng.random() < 0.6)
    else:
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        batch = _log_int(rng, 1, 48)
        longest = _log_int(rng, 1, min(131072, 100_000_000 // (batch * kv * 128)))
        new = rng.choice([1, 1, 1, 2, 4])
        longest = max(longest, new)
        case = _cached("", batch=batch, new=new, shortest=rng.randint(new, longest), longest=longest, heads=heads,
                       kv_heads=kv, dim=rng.choice([64, 96, 128]), dtype=dtype,
                       window=rng.randint(1, longest) if rng.random() < 0.3 else 0,
                       cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.3)
    del case["name"]
    return case


# ---- what the cases say ---------------------------------------------------------------------------------------------

def _frequencies(case):
    """Angle per position of each pair, fp64; "linear" divides all by the factor, "parts" only the slow ones."""
    half = case["rot"] // 2
    f = [10000.0 ** (-p / half) for p in range(half)]
    if case["scaling"] == "linear":
        f = [x / case["factor"] for x in f]
    if case["scaling"] == "parts":
        for p, x in enumerate(f):
            turns = 4096 * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            f[p] = x * (keep + (1 - keep) / case["factor"])
    return f


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0


def _document_lengths(case):
    """Ragged lengths, the same for every seed but for their order; the last 1/64 of the rows is padding."""
    n, tokens = case["documents"], case["q_len"] - case["q_len"] // 64
    share = [1.0 + 3.0 * ((5 * d + 2) % n) / n for d in range(n)]
    lengths = [int(tokens * s / sum(share)) for s in share]
    lengths[0] += tokens - sum(lengths)
    return lengths


def _prefix_lengths(case):
    return [case["k_len"] * (2 * b + 1) // (4 * case["batch"]) for b in range(case["batch"])]


def _cache_lengths(case):
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [min(hi, max(lo, round(lo * (hi / lo) ** ((b + 1) / n)))) for b in range(n)]


def _slopes(case):
    return [2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])]


def _pairs(case):
    """Visible (query, key) pairs of all sequences, for one head."""
    if case["op"] == "cached":
        return sum(_row_sum(n, case["new"], case["window"]) for n in _cache_lengths(case))
    q, k = case["q_len"], case["k_len"]
    if case["mask"] == "full":
        return case["batch"] * q * k
    if case["mask"] == "documents":
        return sum(n * (n + 1) // 2 for n in _document_lengths(case))
    if case["mask"] == "prefix":
        return sum(p * p + (k * (k + 1) - p * (p + 1)) // 2 for p in _prefix_lengths(case))
    return case["batch"] * _row_sum(k, q, case["window"])


def _row_sum(keys, rows, window):
    """Keys seen by the last `rows` positions of `keys`, each sees itself and those before it, within the window."""
    seen = range(keys - rows + 1, keys + 1)
    return sum(min(n, window) for n in seen) if window else sum(seen)


def work(case):
    item = ITEM[case["dtype"]]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * item + 8 * tokens), "flops": passes * 3 * n}
    if case["op"] == "cached":
        rows = case["batch"] * case["new"] * case["heads"] * case["dim"]
        seen = sum(min(n, case["window"] + case["new"] - 1) if case["window"] else n for n in _cache_lengths(case))
        cache = 2 * seen * case["kv_heads"] * case["dim"]
        return {"bytes": (2 * rows + cache) * item, "flops": 4 * case["dim"] * case["heads"] * _pairs(case)}
    rows = case["batch"] * case["q_len"] * case["heads"] * case["dim"]
    keys = 2 * case["batch"] * case["k_len"] * case["kv_heads"] * case["dim"]
    # two products forward; backward the scores again and four more (the scores of all pairs are not kept)
    per_pair = (14 if case["grad"] else 4) * case["dim"]
    moved = 2 * rows + keys + (2 * rows + keys if case["grad"] else 0)
    return {"bytes": moved * item, "flops": per_pair * case["heads"] * _pairs(case)}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=gen).to(dtype)

    def device(values, kind):
        return torch.tensor(values, device="cuda", dtype=kind)

    state = {"case": case}
    if case["op"] == "rotary":
        b, s, h, hk, d = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
        state["q"] = normal(b, s, h, d)
        state["k"] = normal(b, s, hk, d) if hk else None
        first = torch.randint(0, max(1, case["reach"] - s + 1), (b, 1), device="cuda", generator=gen)
        positions = first + torch.arange(s, device="cuda")[None, :]
        if case["fractional"]:
            positions = positions.double() + torch.rand(b, s, device="cuda", dtype=torch.float64, generator=gen)
        state["positions"] = positions
        state["freqs"] = device(_frequencies(case), torch.float64)
        state["magnitude"] = _magnitude(case)
        if case["grad"]:
            state["dq"] = normal(b, s, h, d)
            state["dk"] = normal(b, s, hk, d) if hk else None
    elif case["op"] == "attend":
        b, sq, sk, h, hk, d = (case[n] for n in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
        state["q"], state["k"], state["v"] = normal(b, sq, h, d), normal(b, sk, hk, d), normal(b, sk, hk, d)
        if case["grad"]:
            state["do"] = normal(b, sq, h, d)
        state["slopes"] = device(_slopes(case), torch.float32) if case["bias"] else None
        if case["mask"] == "documents":
            lengths = device(_document_lengths(case), torch.int32)
            lengths = lengths[torch.randperm(len(lengths), device="cuda", generator=gen)]
            state["offsets"] = torch.cat([lengths.new_zeros(1), lengths.cumsum(0, dtype=torch.int32)])
        if case["mask"] == "prefix":
            prefix = device(_prefix_lengths(case), torch.int32)
            state["prefix"] = prefix[torch.randperm(b, device="cuda", generator=gen)]
    else:
        b, new, h, hk, d = (case[n] for n in ("batch", "new", "heads", "kv_heads", "dim"))
        capacity = case["longest"]
        state["q"] = normal(b, new, h, d)
        state["k"], state["v"] = normal(b, capacity, hk, d), normal(b, capacity, hk, d)
        lengths = device(_cache_lengths(case), torch.int32)
        state["lengths"] = lengths[torch.randperm(b, device="cuda", generator=gen)]
        state["slopes"] = device(_slopes(case), torch.float32) if case["bias"] else None
    if case.get("grad"):
        for name in ("q", "k", "v"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return _run_rotary(state, case)
    if case["op"] == "attend":
        return _run_attend(state, case)
    return _run_cached(state, case)


def _run_rotary(state, case):
    q, k = state["q"], state["k"]
    if own:
        from flashdiffusion_b200 import rope
        turned = rope.apply_rotary(q, k, positions=state["positions"], freqs=state["freqs"], layout=case["layout"],
                                   magnitude=state["magnitude"])
        turned = [turned] if k is None else list(turned)
        if not case["grad"]:
            return turned
        leaves, grads = ([q], [state["dq"]]) if k is None else ([q, k], [state["dq"], state["dk"]])
        return turned + list(torch.autograd.grad(turned, leaves, grads))
    angle = state["positions"].double()[..., None] * state["freqs"]
    cos, sin = torch.cos(angle).float()[:, :, None, :], torch.sin(angle).float()[:, :, None, :]
    out = [_turn(q, cos, sin, case, state["magnitude"])]
    if k is not None:
        out.append(_turn(k, cos, sin, case, state["magnitude"]))
    if case["grad"]:
        out.append(_turn(state["dq"], cos, -sin, case, state["magnitude"]))
        if k is not None:
            out.append(_turn(state["dk"], cos, -sin, case, state["magnitude"]))
    return out


def _turn(x, cos, sin, case, magnitude):
    rot, half = case["rot"], case["rot"] // 2
    y = x.detach().float().clone()
    if case["layout"] == "half":
        a, b = y[..., :half].clone(), y[..., half:rot].clone()
        y[..., :half], y[..., half:rot] = magnitude * (a * cos - b * sin), magnitude * (a * sin + b * cos)
    else:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = magnitude * (a * cos - b * sin), magnitude * (a * sin + b * cos)
    return y.to(x.dtype)


def _run_attend(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    cap = case["cap"] or None
    if own:
        from flashdiffusion_b200 import attention
        how = {"causal": case["mask"] in ("causal", "window"), "window": case["window"] or None}
        if case["mask"] == "documents":
            how = {"spans": attention.document_spans(state["offsets"], case["q_len"])}
        if case["mask"] == "prefix":
            how = {"spans": attention.prefix_spans(state["prefix"], case["q_len"])}
        out = attention.attend(q, k, v, cap=cap, slopes=state["slopes"], **how)
        if not case["grad"]:
            return [out]
        return [out] + list(torch.autograd.grad(out, (q, k, v), state["do"]))
    if not case["grad"]:
        with torch.no_grad():
            return [_plain_attention(q.float(), k.float(), v.float(), _visible(state, case), case, state["slopes"]).to(q.dtype)]
    leaves = [x.detach().float().requires_grad_(True) for x in (q, k, v)]
    out = _plain_attention(*leaves, _visible(state, case), case, state["slopes"])
    grads = torch.autograd.grad(out, leaves, state["do"].float())
    return [out.detach().to(q.dtype)] + [g.to(q.dtype) for g in grads]


def _visible(state, case):
    """(batch or 1, 1, 1, q_len, k_len) truth values."""
    sq, sk = case["q_len"], case["k_len"]
    j = torch.arange(sk, device="cuda")[None, None, :]
    i = torch.arange(sk - sq, sk, device="cuda")[None, :, None]
    if case["mask"] == "full":
        see = (j >= 0) & (i >= i)
    elif case["mask"] == "documents":
        document = torch.bucketize(torch.arange(sk, device="cuda"), state["offsets"][1:], right=True)
        inside = torch.arange(sk, device="cuda") < state["offsets"][-1]
        see = (j <= i) & (document[None, :, None] == document[None, None, :]) & inside[None, :, None]
    elif case["mask"] == "prefix":
        see = (j <= i) | (j < state["prefix"][:, None, None])
    else:
        see = j <= i
        if case["window"]:
            see = see & (j > i - case["window"])
    return see[:, None, None, :, :]


def _plain_attention(q, k, v, see, case, slopes):
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    g = h // hk
    qh = q.permute(0, 2, 1, 3).reshape(b, hk, g * sq, d)
    s = (qh @ k.permute(0, 2, 3, 1)).reshape(b, hk, g, sq, sk) * (1.0 / math.sqrt(d))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if slopes is not None:
        s = s - slopes.reshape(1, hk, g, 1, 1) * _distance(sq, sk)
    s = torch.where(see, s, float("-inf"))
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = p.reshape(b, hk, g * sq, sk) @ v.permute(0, 2, 1, 3)
    return o.reshape(b, h, sq, d).permute(0, 2, 1, 3)


def _distance(sq, sk):
    i = torch.arange(sk - sq, sk, device="cuda", dtype=torch.float32)
    return (i[:, None] - torch.arange(sk, device="cuda", dtype=torch.float32)[None, :]).abs()


def _run_cached(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    if own:
        from flashdiffusion_b200 import attention
        return [attention.attend_cached(q, k, v, state["lengths"], window=case["window"] or None,
                                        cap=case["cap"] or None, slopes=state["slopes"])]
    b, new, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    g = h // hk
    qh = q.float().permute(0, 2, 1, 3).reshape(b, hk, g * new, d)
    s = (qh @ k.float().permute(0, 2, 3, 1)).reshape(b, hk, g, new, n) * (1.0 / math.sqrt(d))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    j = torch.arange(n, device="cuda")[None, None, :]
    i = state["lengths"][:, None, None] - new + torch.arange(new, device="cuda")[None, :, None]
    if state["slopes"] is not None:
        s = s - state["slopes"].reshape(1, hk, g, 1, 1) * (i - j).abs().float()[:, None, None]
    see = j <= i
    if case["window"]:
        see = see & (j > i - case["window"])
    s = torch.where(see[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = p.reshape(b, hk, g * new, n) @ v.float().permute(0, 2, 1, 3)
    return [o.reshape(b, h, new, d).permute(0, 2, 1, 3).to(q.dtype)]


# ---- the definitions in 64 bits, one head of one sequence at a time -------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(state, case)
    with torch.no_grad():
        return _exact_attention(state, case)


def _exact_rotary(state, case):
    rot, half = case["rot"], case["rot"] // 2
    phase = torch.polar(torch.full_like(state["freqs"], state["magnitude"]).expand(*state["positions"].shape, half),
                        state["positions"].double().unsqueeze(-1) * state["freqs"]).unsqueeze(2)

    def spin(x, factor):
        x = x.detach().double()
        head = x[..., :rot]
        pairs = head.unflatten(-1, (2, half)).transpose(-1, -2) if case["layout"] == "half" else head.unflatten(-1, (half, 2))
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * factor)
        turned = turned.transpose(-1, -2) if case["layout"] == "half" else turned
        return torch.cat([turned.flatten(-2), x[..., rot:]], -1)

    back = [("dq", "q"), ("dk", "k")] if case["grad"] else []
    return [spin(state[n], phase) for n in ("q", "k") if state[n] is not None] + [
        spin(state[n], phase.conj()) for n, x in back if state[x] is not None]


def _exact_attention(state, case):
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    group, scale, cap = h // hk, d ** -0.5, case["cap"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v)] if case.get("grad") else []
    keys = torch.arange(sk, device="cuda").unsqueeze(0)
    for n in range(b):
        first, end, place = _exact_spans(state, case, n)
        hidden = (keys < first.unsqueeze(1)) | (keys >= end.unsqueeze(1))
        empty = (end <= first).unsqueeze(1)
        for m in range(h):
            qm, km, vm = q[n, :, m].double(), k[n, :, m // group].double(), v[n, :, m // group].double()
            score = scale * (qm @ km.T)
            bend = None
            if cap:
                bend = torch.tanh(score / cap)
                score = cap * bend
            if state["slopes"] is not None:
                score -= float(state["slopes"][m]) * (place.unsqueeze(1) - keys).abs()
            p = torch.softmax(score.masked_fill_(hidden, -1e300), -1).masked_fill_(hidden | empty, 0.0)
            del score
            out[n, :, m] = p @ vm
            if grads:
                dom = state["do"][n, :, m].double()
                grads[2][n, :, m // group] += p.T @ dom
                slope = dom @ vm.T
                slope -= (dom * out[n, :, m]).sum(-1, keepdim=True)
                slope *= p * scale
                if bend is not None:
                    slope *= 1 - bend * bend
                grads[0][n, :, m] = slope @ km
                grads[1][n, :, m // group] += slope.T @ qm
    return [out] + grads


def _exact_spans(state, case, n):
    """(first key, end of keys, position) of each query row of sequence n."""
    if case["op"] == "cached":
        place = int(state["lengths"][n]) - case["new"] + torch.arange(case["new"], device="cuda")
        first = (place - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(place)
        return first, place + 1, place
    place = torch.arange(case["q_len"], device="cuda") + case["k_len"] - case["q_len"]
    first, end = torch.zeros_like(place), place + 1
    if case["mask"] == "full":
        end = torch.full_like(place, case["k_len"])
    if case["mask"] == "window":
        first = (place - case["window"] + 1).clamp(min=0)
    if case["mask"] == "documents":
        ends = state["offsets"].tolist()
        first, end = torch.zeros_like(place), torch.zeros_like(place)
        for lo, hi in zip(ends[:-1], ends[1:]):
            first[lo:hi] = lo
            end[lo:hi] = place[lo:hi] + 1
    if case["mask"] == "prefix":
        end = torch.maximum(end, state["prefix"][n].long())
    return first, end, place
