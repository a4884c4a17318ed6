"""What a decoder layer computes between its Monarch projections, as cases to time and to compare.

* ``op="norm"``: ``rms_norm`` of hidden states after the residual's addition, alone or with the gradients of both
  (``train``); ``op="norm8"``: ``rms_norm_fp8``, the same with an output in 8 bits (float8_e4m3fn) and a scale
  for each ``group``.
* ``op="rotary"``: ``rotary`` of queries and keys, alone or with their gradients.
* ``op="attention"``: ``differential_attention``: of one new token for each sequence of a cache (``queries`` 1), of a
  prompt, or with all gradients (``train``).

Widths are those of the benchmark configurations (toy 512, 257M 1024, 1.3B 2048, 6.89B 4096:
``monarch_muon_amd/workloads.py``) and of a 124M model (768); 1024 tokens are one training sequence.  A differential
head has two query and two key heads of ``dim`` columns and values of twice as many: width = 2 x dim x heads.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_E4M3_MAX = 448.0
#: Elements of the largest norm and rotary cases, and visible pairs x columns of the largest attention, forward products.
MOST_ELEMENTS = 16384 * 4096
MOST_PAIRS = 16 * 128 * 8192 * 8192 // 2
MOST_CACHE = 131072 * 8 * 128


def _norm(name, op, tokens, width, train=False, dtype="bf16", residual=True, group=0):
    """``group``: columns of a scale of the 8-bit output; 0: one for the row."""
    return dict(name=name, op=op, tokens=tokens, width=width, train=train, dtype=dtype, residual=residual, group=group)


def _rotary(name, batch, tokens, qheads, kheads, dim, part, train, interleaved=False, dtype="bf16", table=2048, far=False,
            scaling="none"):
    """``part``: columns of a head that are rotated; ``far``: each sequence stands at a position of its own, up to
    ``table``; ``scaling``: of the table for contexts longer than those trained."""
    return dict(name=name, op="rotary", batch=batch, tokens=tokens, qheads=qheads, kheads=kheads, dim=dim, part=part,
                train=train, interleaved=interleaved, dtype=dtype, table=table, far=far, scaling=scaling)


def _attention(name, batch, queries, keys, heads, kvheads, dim, train, causal=True, ragged=False):
    """``ragged``: ``keys`` is what a cache holds at most, the sequences have lengths of their own."""
    return dict(name=name, op="attention", batch=batch, queries=queries, keys=keys, heads=heads, kvheads=kvheads, dim=dim,
                train=train, causal=causal, ragged=ragged)


def listed():
    return [
        # generation: one token's hidden state through a 6.89B layer's norm
        _norm("norm-1-6.89b", "norm", 1, 4096),
        # prompt processing: a micro-batch (4 x 1024) of the 6.89B model on its way into an 8-bit projection
        _norm("norm8-6.89b", "norm8", 4096, 4096, group=128),
        # training the 6.89B model: 16 sequences of 1024
        _norm("norm-train-6.89b", "norm", 16384, 4096, True),
        # generation: one token of each of eight sequences, at positions of their own, tables scaled for long contexts
        _rotary("rotary-8-6.89b", 8, 1, 32, 8, 128, 128, False, table=32768, far=True, scaling="yarn"),
        # training a 124M model in fp32: half of each head rotated, neighbouring columns as pairs, a ragged micro-batch
        _rotary("rotary-train-124m-odd", 1, 2047, 12, 12, 64, 32, True, True, "f32"),
        # training the 6.89B model: 16 sequences of 1024
        _rotary("rotary-train-6.89b", 16, 1024, 32, 32, 128, 128, True),
        # generation: eight sequences of up to 4096 tokens in the cache of a 6.89B layer, four query heads to a key head
        _attention("decode-8-6.89b", 8, 1, 4096, 16, 4, 128, False, ragged=True),
        # generation: one long document in the cache of a 1.3B layer
        _attention("decode-long-1.3b", 1, 1, 131072, 8, 8, 128, False, ragged=True),
        # prompt processing: one long ragged prompt through a 6.89B layer
        _attention("prefill-6.89b", 1, 8191, 8191, 16, 16, 128, False),
        # training a 124M model: three ragged sequences, three query heads to a key head
        _attention("train-124m-odd", 3, 1001, 1001, 6, 2, 64, True),
        # training the 257M model: 16 sequences of 1024
        _attention("train-257m", 16, 1024, 1024, 8, 8, 64, True),
        # training the 6.89B model at the benchmark's micro-batch (4 x 1024)
        _attention("train-6.89b", 4, 1024, 1024, 16, 16, 128, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.3:
        width = rng.choice([8 * _log(rng, 16, 1024), 8 * _log(rng, 16, 1024), _log(rng, 100, 8192)])
        op, dtype = rng.choice([("norm", "bf16"), ("norm", "bf16"), ("norm", "f32"), ("norm8", "bf16")])
        train = op == "norm" and rng.random() < 0.6
        tokens = _log(rng, 1, min(131072, MOST_ELEMENTS // width // (1 if dtype == "bf16" else 2)))
        c = _norm("", op, tokens, width, train, dtype, rng.random() < 0.7, rng.choice([0, 128]) if op == "norm8" else 0)
    elif kind < 0.5:
        dim = rng.choice([32, 64, 128, 8 * rng.randint(2, 32), 2 * rng.randint(8, 100)])
        kheads = rng.choice([1, 2, 4, 8, 12, 16])
        qheads = kheads * rng.choice([1, 1, 2, 3, 4])
        part = rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
        far, dtype = rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"])
        most = MOST_ELEMENTS // ((qheads + kheads) * dim) // (1 if dtype == "bf16" else 2)
        tokens = _log(rng, 1, min(8192, most))
        batch = _log(rng, 1, min(64, max(1, most // tokens)))
        c = _rotary("", batch, tokens, qheads, kheads, dim, part, rng.random() < 0.5, rng.random() < 0.5, dtype,
                    32768 if far else 8192, far, rng.choice(["none", "linear", "ntk", "yarn", "llama"]))
    else:
        dim = rng.choice([32, 64, 64, 128, 128, 8 * rng.randint(2, 16)])
        kvheads = rng.choice([1, 2, 4, 6, 8])
        heads = kvheads * rng.choice([1, 1, 2, 3, 4])
        if rng.random() < 0.4:                           # new tokens of a cache
            batch = _log(rng, 1, 64)
            keys = _log(rng, 16, min(131072, max(16, MOST_CACHE // (batch * kvheads * dim))))
            c = _attention("", batch, rng.choice([1, 1, 1, rng.randint(2, 8)]), keys, heads, kvheads, dim, False,
                           ragged=rng.random() < 0.8)
        else:
            train, causal = rng.random() < 0.6, rng.random() < 0.8
            # visible pairs x dim x heads x batch, three times as much with the gradients
            most = MOST_PAIRS // (max(dim, 64) * heads * (3 if train else 1))
            keys = _log(rng, 16, min(8192, int((most * (2 if causal else 1)) ** 0.5)))
            queries = keys if rng.random() < 0.7 else _log(rng, 1, keys)
            batch = _log(rng, 1, max(1, min(16, most * (2 if causal else 1) // keys ** 2)))
            c = _attention("", batch, queries, keys, heads, kvheads, dim, train, causal, rng.random() < 0.3)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _frequencies(part, scaling):
    """(angle of a position for each pair, in 64 bits; factor of the rotated columns) of 2048 positions trained and the
    scaling for 32768 of them."""
    f = 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / part)
    trained, factor = 2048, 16.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return f * factor ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / max(part - 2, 1)), 1.0
    turns = trained * f / (2 * math.pi)
    if scaling == "yarn":      # pairs of over 32 turns within the trained positions as they are, of under 1 slowed
        at = lambda n: part * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), part - 1)
        slow = ((torch.arange(part // 2, dtype=torch.float64, device=DEV) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / factor * slow + f * (1 - slow), 0.1 * math.log(factor) + 1.0
    if scaling == "llama":     # pairs of over 4 turns as they are, of under 1 slowed
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    return f, 1.0


def _positions(case, g):
    B, T = case["batch"], case["tokens"]
    t = torch.arange(T, device=DEV).expand(B, T)
    if not case["far"]:
        return t
    return t + torch.randint(0, case["table"] - T + 1, (B, 1), generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["op"] in ("norm", "norm8"):
        T, D, dt, grad = case["tokens"], case["width"], _DT[case["dtype"]], case["train"]
        # a residual stream whose columns differ in size, and what a block adds to it
        size = torch.exp(0.5 * _randn(g, D))
        s["x"] = (0.5 * _randn(g, T, D) * size).to(dt).requires_grad_(grad)
        s["r"] = (2 * _randn(g, T, D) * size).to(dt).requires_grad_(grad) if case["residual"] else None
        s["w"] = (1 + 0.2 * _randn(g, D)).to(dt).requires_grad_(grad)
        if grad:
            s["dy"] = (1e-3 * _randn(g, T, D)).to(dt)
            s["dh"] = (1e-3 * _randn(g, T, D)).to(dt) if case["residual"] else None
    elif case["op"] == "rotary":
        B, T, d, dt, grad = case["batch"], case["tokens"], case["dim"], _DT[case["dtype"]], case["train"]
        s["pos"] = _positions(case, g)
        f, factor = _frequencies(case["part"], case["scaling"])
        a = torch.arange(case["table"], dtype=torch.float64, device=DEV).unsqueeze(1) * f
        s["table"] = (torch.cat([a.cos(), a.sin()], 1) * factor).float()
        s["q"] = _randn(g, B, T, case["qheads"], d).to(dt).requires_grad_(grad)
        s["k"] = _randn(g, B, T, case["kheads"], d).to(dt).requires_grad_(grad)
        if grad:
            s["dq"] = (1e-3 * _randn(g, B, T, case["qheads"], d)).to(dt)
            s["dk"] = (1e-3 * _randn(g, B, T, case["kheads"], d)).to(dt)
    else:
        B, Tq, Tk, d, grad = case["batch"], case["queries"], case["keys"], case["dim"], case["train"]
        H, K = case["heads"], case["kvheads"]
        s["q"] = (1.5 * _randn(g, B, Tq, 2 * H, d)).bfloat16().requires_grad_(grad)
        s["k"] = _randn(g, B, Tk, 2 * K, d).bfloat16().requires_grad_(grad)
        s["v"] = _randn(g, B, Tk, K, 2 * d).bfloat16().requires_grad_(grad)
        s["lam"] = (0.2 + 0.6 * torch.rand(H, generator=g, device=DEV)).requires_grad_(grad)
        s["n"] = None
        if case["ragged"]:
            s["n"] = torch.randint(max(1, Tk // 2), Tk + 1, (B,), generator=g, device=DEV)
            s["n"][0] = Tk
        if grad:
            s["do"] = (1e-3 * _randn(g, B, Tq, H, 2 * d)).bfloat16()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s["case"], s)


def _own_norm(c, s):
    from monarch_muon_amd import rms_norm
    out = rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
    if not c["train"]:
        return out
    if not c["residual"]:
        return out.detach(), *torch.autograd.grad(out, (s["x"], s["w"]), s["dy"])
    grads = torch.autograd.grad(out, (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
    return out[0].detach(), out[1].detach(), *grads


def _own_norm8(c, s):
    from monarch_muon_amd import rms_norm_fp8
    return rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=EPS, group=c["group"] or None)


def _own_rotary(c, s):
    from monarch_muon_amd import rotary
    out = rotary(s["q"], s["k"], s["table"], s["pos"] if c["far"] else None, interleaved=c["interleaved"])
    if not c["train"]:
        return out
    return out[0].detach(), out[1].detach(), *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))


def _own_attention(c, s):
    from monarch_muon_amd import differential_attention
    out = differential_attention(s["q"], s["k"], s["v"], s["lam"], causal=c["causal"], lengths=s["n"])
    if not c["train"]:
        return out
    return out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["lam"]), s["do"])


@torch.no_grad()
def _plain_norm(c, s):
    x, r, w = s["x"], s["r"], s["w"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)      # the residual stream is kept in its own type
    hf, wf = h.float(), w.float()
    inv = (hf.square().mean(1, keepdim=True) + EPS).rsqrt()
    n = hf * inv
    y = (n * wf).to(x.dtype)
    if not c["train"]:
        return y if r is None else (y, h)
    dy = s["dy"].float()
    dw = (dy * n).sum(0).to(w.dtype)
    dn = dy * wf
    dx = inv * (dn - n * (dn * n).mean(1, keepdim=True))
    if r is None:
        return y, dx.to(x.dtype), dw
    dx = (dx + s["dh"].float()).to(x.dtype)
    return y, h, dx, dx, dw


@torch.no_grad()
def _plain_norm8(c, s):
    x, r = s["x"], s["r"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    hf = h.double()                                      # a value beside a border goes to one side of it or the other
    y = hf * (hf.square().mean(1, keepdim=True) + EPS).rsqrt() * s["w"].double()
    T, D = y.shape
    G = c["group"] or D
    most = torch.nn.functional.pad(y, (0, -D % G)).view(T, -1, G).abs().amax(2)
    scale = torch.where(most > 0, most / _E4M3_MAX, 1.0)
    codes = (y / scale.repeat_interleave(G, 1)[:, :D]).float().to(torch.float8_e4m3fn)
    return codes, scale.float(), *([] if r is None else [h])


def _turned(x, cos, sin, part, interleaved):
    """``x`` (B, T, H, d) with its first ``part`` columns rotated."""
    a, b = (x[..., 0:part:2], x[..., 1:part:2]) if interleaved else (x[..., :part // 2], x[..., part // 2:part])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., part:]], -1)


@torch.no_grad()
def _plain_rotary(c, s):
    at = s["table"][s["pos"]].unsqueeze(2)
    half, args = c["part"] // 2, (c["part"], c["interleaved"])
    cos, sin = at[..., :half], at[..., half:]
    out = [_turned(t.float(), cos, sin, *args).to(t.dtype) for t in (s["q"], s["k"])]
    if c["train"]:
        out += [_turned(t.float(), cos, -sin, *args).to(t.dtype) for t in (s["dq"], s["dk"])]
    return tuple(out)


def _visible(c, s):
    """(B, queries, keys): the keys that each query sees."""
    B, Tq, Tk = c["batch"], c["queries"], c["keys"]
    n = torch.full((B,), Tk, device=DEV) if s["n"] is None else s["n"]
    j = torch.arange(Tk, device=DEV)
    see = (j < n[:, None])[:, None, :].expand(B, Tq, Tk)
    if c["causal"]:
        at = n[:, None] - Tq + torch.arange(Tq, device=DEV)
        see = see & (j <= at[:, :, None])
    return see


@torch.no_grad()
def _plain_attention(c, s):
    B, Tq, Tk, d = c["batch"], c["queries"], c["keys"], c["dim"]
    H, K = c["heads"], c["kvheads"]
    G = H // K
    # (B, K, G, 2, T, d), and (B, K, 1, T, 2 d) for the values
    q = s["q"].float().view(B, Tq, K, G, 2, d).permute(0, 2, 3, 4, 1, 5)
    k = s["k"].float().view(B, Tk, K, 1, 2, d).permute(0, 2, 3, 4, 1, 5)
    v = s["v"].float().view(B, Tk, K, 1, 2 * d).permute(0, 2, 3, 1, 4)
    lam = s["lam"].float().view(K, G, 1, 1)
    see = _visible(c, s)[:, None, None, None]
    x = (q @ k.transpose(-1, -2) * d ** -0.5).masked_fill_(~see, -math.inf)
    x = (x - x.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    p = x.div_(x.sum(-1, keepdim=True).clamp_min(1e-30))
    p1, p2 = p[:, :, :, 0], p[:, :, :, 1]
    both = p1 - lam * p2
    merged = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, Tq, H, 2 * d).bfloat16()  # noqa: E731
    if not c["train"]:
        return merged(both @ v)
    do = s["do"].float().view(B, Tq, K, G, 2 * d).permute(0, 2, 3, 1, 4)
    dp = do @ v.transpose(-1, -2)
    along = (p * dp.unsqueeze(3)).sum(-1, keepdim=True)
    dlam = -along[:, :, :, 1].double().sum((0, 3, 4)).view(H).float()
    ds = p * (dp.unsqueeze(3) - along)
    ds[:, :, :, 1] *= -lam
    ds *= d ** -0.5
    dq = (ds @ k).permute(0, 4, 1, 2, 3, 5).reshape(B, Tq, 2 * H, d).bfloat16()
    dk = (ds.transpose(-1, -2) @ q).sum(2).permute(0, 3, 1, 2, 4).reshape(B, Tk, 2 * K, d).bfloat16()
    dv = (both.transpose(-1, -2) @ do).sum(2).permute(0, 2, 1, 3).reshape(B, Tk, K, 2 * d).bfloat16()
    return merged(both @ v), dq, dk, dv, dlam


_own = dict(norm=_own_norm, norm8=_own_norm8, rotary=_own_rotary, attention=_own_attention)
_plain = dict(norm=_plain_norm, norm8=_plain_norm8, rotary=_plain_rotary, attention=_plain_attention)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] in ("norm", "norm8"):
        T, D, b = case["tokens"], case["width"], 2 if case["dtype"] == "bf16" else 4
        r = case["residual"]
        if case["op"] == "norm8":
            groups = -(-D // case["group"]) if case["group"] else 1
            return {"bytes": T * (D * (b * (3 if r else 1) + 1) + 4 * groups) + b * D, "flops": 0}
        forward, backward = b * T * D * (4 if r else 2), b * T * D * (3 if r else 2)
        return {"bytes": forward + b * D + (backward + b * D if case["train"] else 0), "flops": 0}
    if case["op"] == "rotary":
        B, T, b = case["batch"], case["tokens"], 2 if case["dtype"] == "bf16" else 4
        each = 2 * b * B * T * (case["qheads"] + case["kheads"]) * case["dim"]
        rows = min(B * T, case["table"]) if case["far"] else T
        return {"bytes": each * (2 if case["train"] else 1) + 4 * rows * case["part"] + (8 * B * T if case["far"] else 0),
                "flops": 0}
    B, Tq, Tk, d, H, K = (case[n] for n in ("batch", "queries", "keys", "dim", "heads", "kvheads"))
    # lengths are from half of the cache to all of it, the first one all
    seen = [Tk] + [0.75 * Tk] * (B - 1) if case["ragged"] else [Tk] * B

    def pairs_of(n):
        if not case["causal"]:
            return Tq * n
        rows = min(Tq, n)                                # query i sees n - Tq + i + 1 keys
        return rows * n - rows * (rows - 1) / 2

    pairs = H * sum(pairs_of(n) for n in seen)
    qo, kv = 2 * B * Tq * H * 2 * d, 2 * sum(seen) * K * 4 * d
    train = case["train"]
    return {"bytes": int((4 if train else 2) * qo + (2 if train else 1) * kv), "flops": int((24 if train else 8) * d * pairs)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact[case["op"]](case, {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v
                                         for k, v in s.items()}, s)


def _exact_norm(c, s, given):
    w = s["w"]
    h = s["x"]
    if s["r"] is not None:                               # the sum as it is kept
        h = (s["x"] + s["r"]).to(given["x"].dtype).double()
    rms = (h.pow(2).sum(1) / c["width"] + EPS).sqrt().unsqueeze(1)
    y = h / rms * w
    if c["op"] == "norm8":
        T, D = y.shape
        G = c["group"] or D
        out, steps = torch.empty_like(y), []
        for i in range(0, D, G):
            part = y[:, i:i + G]
            step = part.abs().amax(1, keepdim=True) / _E4M3_MAX
            step[step == 0] = 1
            z = part / step
            # to 3 bits behind the leading one, the smallest normal number being 2^-6
            unit = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
            out[:, i:i + G] = torch.round(z / unit) * unit
            steps.append(step)
        return out, torch.cat(steps, 1), *([] if s["r"] is None else [h])
    if not c["train"]:
        return y if s["r"] is None else (y, h)
    dy = s["dy"]
    g = dy * w / rms
    dx = g - h * (g * h).sum(1, keepdim=True) / (c["width"] * rms.pow(2))
    dw = (dy * h / rms).sum(0)
    if s["r"] is None:
        return y, dx, dw
    dx = dx + s["dh"]
    return y, h, dx, dx, dw


def _exact_rotary(c, s, given):
    f, factor = _frequencies(c["part"], c["scaling"])
    a = given["pos"].double()[:, :, None, None] * f
    spin = torch.polar(torch.full_like(a, factor), a)
    half = c["part"] // 2
    first = torch.arange(half, device=DEV) * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)

    def turn(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out
    out = [turn(s["q"], spin), turn(s["k"], spin)]
    if c["train"]:
        out += [turn(s["dq"], spin.conj()), turn(s["dk"], spin.conj())]
    return tuple(out)


def _exact_attention(c, s, given):
    B, Tq, Tk, d, H, K = (c[n] for n in ("batch", "queries", "keys", "dim", "heads", "kvheads"))
    train, scale = c["train"], 1 / math.sqrt(d)
    o = torch.zeros(B, Tq, H, 2 * d, dtype=torch.float64, device=DEV)
    dq, dk, dv, dlam = (torch.zeros_like(s[n]) for n in ("q", "k", "v", "lam"))
    for b in range(B):
        n = Tk if given["n"] is None else int(given["n"][b])
        rows = torch.arange(Tq, device=DEV) + (n - Tq)
        hidden = torch.arange(n, device=DEV)[None, :] > rows[:, None] if c["causal"] else None
        for h in range(H):
            g, lam = h // (H // K), s["lam"][h]
            v = s["v"][b, :n, g]
            maps = []
            for m in (0, 1):
                z = s["q"][b, :, 2 * h + m] @ s["k"][b, :n, 2 * g + m].T * scale
                if hidden is not None:
                    z[hidden] = -math.inf
                maps.append(torch.nan_to_num(torch.softmax(z, 1), nan=0.0))
            o[b, :, h] = maps[0] @ v - lam * (maps[1] @ v)
            if not train:
                continue
            do = s["do"][b, :, h]
            dv[b, :n, g] += (maps[0] - lam * maps[1]).T @ do
            dp = do @ v.T
            for m, sign in ((0, 1.0), (1, -lam)):
                mean = (maps[m] * dp).sum(1, keepdim=True)
                if m == 1:
                    dlam[h] -= mean.sum()
                dz = maps[m] * (dp - mean) * (sign * scale)
                dq[b, :, 2 * h + m] = dz @ s["k"][b, :n, 2 * g + m]
                dk[b, :n, 2 * g + m] += dz.T @ s["q"][b, :, 2 * h + m]
    return (o, dq, dk, dv, dlam) if train else o


_exact = dict(norm=_exact_norm, norm8=_exact_norm, rotary=_exact_rotary, attention=_exact_attention)
