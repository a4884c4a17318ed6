"""The operators between a layer's projections on the GPU at the ends of what their documentation allows: sequences of more
elements than 31 bits count, and more threads than one launch holds."""
import pytest
import torch

from monarch_muon_amd import differential_attention, rms_norm, rms_norm_fp8, rotary, rotary_table
from oracle import butterfly
from oracle import layer as oracle
from test_gpu_attention import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def randn(*shape, seed=0, size=1.0, dtype=torch.bfloat16):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(DEV).to(dtype)


def room_for(gigabytes):
    if torch.cuda.get_device_properties(0).total_memory < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


# ----- rotary ----------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_a_sequence_of_more_than_31_bits(interleaved):
    """2^31 + 10240 elements of one sequence: the bits of its two halves, and the exact values at its ends."""
    room_for(60)
    T, H, K, D, part = (1 << 20) + 5, 15, 1, 128, 64
    q, k = randn(1, 997, H, D, seed=1).repeat(1, T // 997 + 1, 1, 1)[:, :T], randn(1, 1, K, D, seed=2).expand(1, T, K, D)
    table, at = rotary_table(part, T, device=DEV), torch.arange(T, device=DEV)
    out = rotary(q, k, table, interleaved=interleaved)
    for half in (slice(0, T // 2), slice(T // 2, T)):
        for x, y in zip(out, rotary(q[:, half], k[:, half], table, at[half], interleaved=interleaved)):
            assert torch.equal(x[:, half], y)
    ends = torch.tensor([0, 1, T // 2, T - 1], device=DEV)
    angles = ends.double()[None, :, None] * 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / part)
    for x, y in zip((q, k), out):
        ref, tol = oracle.rotary(x[:, ends], angles, interleaved=interleaved)
        assert ((y[:, ends].double() - ref).abs() <= tol).all()


def test_rotary_of_a_sequence_of_more_threads_than_a_launch():
    """2^31 + 70 tokens of one chunk: a launch holds 2^31 of them."""
    room_for(90)
    T, cycle = (1 << 31) + 70, 1000
    q, table = randn(1, 1, 1, 2, seed=3), rotary_table(2, cycle, device=DEV)
    at = torch.arange(T, device=DEV).remainder_(cycle)
    out, _ = rotary(q.expand(1, T, 1, 2), q[:, :, :0].expand(1, T, 0, 2), table, at)
    ref, _ = rotary(q.expand(1, cycle, 1, 2), q[:, :, :0].expand(1, cycle, 0, 2), table)
    out, ref = out.view(torch.int32).flatten(), ref.view(torch.int32).flatten()
    whole = T // cycle * cycle
    assert torch.equal(out[:whole].view(-1, cycle), ref.expand(T // cycle, cycle))
    assert torch.equal(out[whole:], ref[:T - whole])


# ----- attention: rows and keys that nothing reaches ---------------------------------
BAD = (float("nan"), float("inf"), float("-inf"))


def attend(q, k, v, lam, dout, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    out = differential_attention(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def inputs(B, Tq, Tk, H, K, d, seed):
    return (randn(B, Tq, 2 * H, d, seed=seed, size=1.5), randn(B, Tk, 2 * K, d, seed=seed + 1), randn(B, Tk, K, 2 * d, seed=seed + 2),
            torch.linspace(0.2, 0.8, H, device=DEV), randn(B, Tq, H, 2 * d, seed=seed + 3))


# (of one tile; of several; keys in parts; queries and keys in parts; many sequences, eight waves)
SIZES = [(2, 40, 40, 2, 1), (1, 150, 150, 2, 2), (1, 3, 2000, 2, 1), (1, 700, 700, 1, 1), (12, 300, 300, 8, 8)]


@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("B, Tq, Tk, H, K", SIZES)
def test_queries_that_see_nothing_reach_nothing(B, Tq, Tk, H, K, d):
    """Whatever the queries before the first key hold, and their output's gradients: the others have the same bits, they zeros."""
    q, k, v, lam, dout = inputs(B, Tq, Tk, H, K, d, 31)
    for none in (1, Tq // 2, Tq):            # so many queries see no key
        starts = torch.full((B,), -none, device=DEV)
        ref = attend(q, k, v, lam, dout, starts=starts)
        assert not ref[0][:, :none].any() and not ref[1][:, :none].any()
        for bad in BAD:
            q[:, :none], dout[:, :none] = bad, bad
            for x, y in zip(attend(q, k, v, lam, dout, starts=starts), ref):
                assert torch.equal(x, y)
        q[:, :none], dout[:, :none] = 0.5, 0.25


@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("B, Tq, Tk, H, K", SIZES)
def test_queries_that_see_nothing_are_zero_beside_any_key(B, Tq, Tk, H, K, d):
    """A key that is no number reaches the queries that see it; those before every key have zeros all the same."""
    q, k, v, lam, dout = inputs(B, Tq, Tk, H, K, d, 41)
    none = (Tq + 1) // 2
    for bad in BAD:
        k[:, 0], v[:, 0] = bad, bad
        o, dq, *_ = attend(q, k, v, lam, dout, starts=torch.full((B,), -none, device=DEV))
        assert not o[:, :none].any() and not dq[:, :none].any()
        assert none == Tq or o[:, none:].isnan().any(-1).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("B, Tq, Tk, H, K", SIZES)
def test_keys_that_nobody_sees_have_zeros_beside_any_query(B, Tq, Tk, H, K, d, causal):
    """Behind a sequence's length, and behind the last query's place: zeros, whatever the queries hold."""
    q, k, v, lam, dout = inputs(B, Tq, Tk, H, K, d, 51)
    n = Tk - 5
    for bad in BAD:
        q[:, -1], dout[:, -1] = bad, bad
        cases = [dict(lengths=torch.full((B,), n, device=DEV))]
        if causal and n >= Tq:
            cases.append(dict(starts=torch.full((B,), n - Tq, device=DEV)))
        for kw in cases:
            _, _, dk, dv, _ = attend(q, k, v, lam, dout, causal=causal, **kw)
            assert not dk[:, n:].any() and not dv[:, n:].any()
            assert dv[:, n - 1].isnan().all()


# ----- the example -------------------------------------------------------------------
def tiny_model(seed=3):
    from monarch_muon_amd import example
    torch.manual_seed(seed)
    return example, example.TinyMonarchLM().to(DEV)


def test_the_example_goes_beyond_a_training_sequence():
    """Tokens one by one and sequences in one call, longer than those that it is trained on."""
    example, model = tiny_model()
    count = 2 * example.SEQ + 5
    tokens, scores = example.generate(model, 7, count)
    assert len(tokens) == count and all(0 <= t < example.VOCAB for t in tokens)
    assert all(-50 < s <= 0 for s in scores)             # log-probabilities of a fresh model: about -ln 509 at most
    assert example.generate(model, 7, 20)[0] == tokens[:20]
    ids = torch.tensor([[7, *tokens[:-1]]], device=DEV)
    with torch.no_grad():
        fresh = tiny_model()[1]
        whole = fresh.hidden(ids)
        assert whole.isfinite().all() and torch.equal(whole, model.hidden(ids))
        # one call or one by one: the sums of the projections and of attention's parts are of other orders
        caches = fresh.caches(1, count)
        last = [fresh.hidden(ids[:, t:t + 1], caches, t) for t in range(count)][-1]
    assert float((last - whole[:, -1:]).float().norm() / whole[:, -1:].float().norm()) < 12 * 2 ** -9
    assert model.loss(ids[:, :-1], ids[:, 1:]).isfinite()


def test_the_example_takes_ids_of_any_shape():
    example, model = tiny_model()
    ids, targets = example.text(torch.Generator().manual_seed(4), DEV)
    with torch.no_grad():
        h = model.hidden(ids)
        assert h.shape == (*ids.shape, example.WIDTH)
        assert torch.equal(model.hidden(ids.view(2, 4, -1)), h.view(2, 4, *h.shape[1:]))
        for none in (ids[:, :0], ids[:0], ids[0, :0]):
            assert model.hidden(none).shape == (*none.shape, example.WIDTH)
        one = model.hidden(ids[0])
        assert one.shape == h[0].shape
        # (one sequence's products are split otherwise than eight's)
        assert float((one - h[0]).float().norm() / h[0].float().norm()) < 12 * 2 ** -9
        assert abs(float(model.loss(ids[0], targets[0])) - float(model.loss(ids[:1], targets[:1]))) == 0


class Rounded(torch.autograd.Function):
    """To bf16's values and back, the gradient too."""

    @staticmethod
    def forward(ctx, x):
        return x.bfloat16().to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.bfloat16().to(g.dtype)


def plain_model(example, p, ids, targets, r):
    """The example's loss in 64 bits, its results through ``r``."""
    p = {n: r(t) for n, t in p.items()}
    H, D, W = example.HEADS, example.DIM, example.WIDTH
    B, T = ids.shape
    angle = torch.arange(T, dtype=torch.float64)[:, None, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    hidden = torch.ones(T, T, dtype=torch.bool).triu(1)

    def norm(h, w):
        return r(h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w)

    def monarch(x, w1, w2):
        x2 = x.reshape(B * T, -1)
        y = r(x2.view(B * T, w1.shape[0], -1).transpose(0, 1) @ w1.transpose(1, 2))
        y = r(butterfly.riffle(y, w2.shape[0]) @ w2.transpose(1, 2))
        return y.permute(1, 2, 0).reshape(B, T, -1)

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return r(torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1))

    x, stream = r(p["wte"][ids] * W ** 0.5), None
    x = torch.where((ids == example.PAD)[..., None], x.detach(), x)   # the padding's row takes no gradient
    for i in range(example.LAYERS):
        at = lambda n: p[f"blocks.{i}.{n}"]  # noqa: E731
        stream = x if stream is None else r(x + stream)
        y = norm(stream, at("norms.0"))
        q, k, v = (monarch(y, at(f"attention.w.{j}"), at(f"attention.w.{j + 1}")) for j in (0, 2, 4))
        q, k, v = turn(q.view(B, T, 2 * H, D)).view(B, T, H, 2, D), turn(k.view(B, T, 2 * H, D)).view(B, T, H, 2, D), v.view(B, T, H, 2 * D)
        s = torch.einsum("bthmd,bshmd->bhmts", q, k) * D ** -0.5
        s = r(s.masked_fill(hidden, -float("inf")).softmax(-1))
        o = r(torch.einsum("bhts,bshd->bthd", s[:, :, 0] - at("attention.lam")[:, None, None] * s[:, :, 1], v))
        x = monarch(norm(o, at("attention.norm")), at("attention.w.6"), at("attention.w.7"))
        stream = r(x + stream)
        y = monarch(norm(stream, at("norms.1")), at("w.0"), at("w.1"))
        x = monarch(r(y * y.sigmoid()), at("w.2"), at("w.3"))
    logits = norm(r(x + stream), p["ln_f"]) @ p["lm_head"].t()
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=example.PAD)


def test_the_examples_gradients_against_differences():
    """Each parameter's gradient against that of the model in 64 bits, which differences of its loss confirm.  The same
    model with its results and their gradients rounded to bf16 says how far those roundings take each gradient: the
    kernels' are as many or fewer and independent of these, so four times as far is beyond what they explain."""
    from monarch_muon_amd import example
    torch.manual_seed(3)
    model = example.TinyMonarchLM()
    ids, targets = example.text(torch.Generator().manual_seed(4), "cpu")
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    loss = plain_model(example, p, ids, targets, lambda t: t)
    exact = dict(zip(p, torch.autograd.grad(loss, list(p.values()))))
    rounded = dict(zip(p, torch.autograd.grad(plain_model(example, p, ids, targets, Rounded.apply), list(p.values()))))
    g = torch.Generator().manual_seed(5)
    along = {n: torch.randn(t.shape, generator=g, dtype=torch.float64) * t.detach().norm() / t.numel() ** 0.5 for n, t in p.items()}
    e = 1e-5
    with torch.no_grad():
        ends = [plain_model(example, {n: t + s * e * along[n] for n, t in p.items()}, ids, targets, lambda t: t) for s in (1, -1)]
    slope = sum(float((exact[n] * along[n]).sum()) for n in p)
    # the differences' own error: the third derivative's e^2, and 64 bits' rounding of the loss over e
    size = sum(float((exact[n] * along[n]).norm()) for n in p)
    assert abs(float(ends[0] - ends[1]) / (2 * e) - slope) <= 1e-6 * size
    model.to(DEV)
    got = model.loss(ids.to(DEV), targets.to(DEV))
    assert abs(float(got.detach()) - float(loss.detach())) <= 0.01 * float(loss.detach())
    for (name, _), grad in zip(model.named_parameters(), torch.autograd.grad(got, list(model.parameters()))):
        off, room = (float((t.double().cpu() - exact[name]).norm()) for t in (grad, rounded[name]))
        assert off <= 4 * room, (name, off / float(exact[name].norm()), room / float(exact[name].norm()))


# ----- attention: scores far from zero -----------------------------------------------
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_gradients_of_large_scores(d, causal):
    """Scores of up to some thousands, within the bounds of fp32 scores: a row's log-sum-exp is rounded like they are."""
    q, k, v, lam, dout = inputs(2, 150, 150, 2, 2, d, 61)
    k = (k.float() * torch.linspace(0.01, 6, 150, device=DEV)[None, :, None, None]).bfloat16()
    q = (q.float() * 30).bfloat16()
    refs, bounds = oracle.attention(q, k, v, lam, causal=causal, dout=dout)
    # A probability or a dS below fp32's 2^-126 is lost, where the form in 64 bits has it: in each of the 300 terms of an
    # element (150 rows or keys, two heads at most) under 2^-126 of P, times |dP| + |D| <= 2 max |dO| . |v|, or 2^-126 of dS
    # itself; times an element of q, k, dO or v.
    largest = max(float(t.abs().max()) for t in (q, k, v, dout))
    lost = 300 * 2.0 ** -126 * (1 + 2 * 2 * d * float(dout.abs().max()) * float(v.abs().max())) * largest
    for name, x, ref, bound in zip(("o", "dq", "dk", "dv", "dlam"), attend(q, k, v, lam, dout, causal=causal), refs, bounds):
        worst, bad = float(((x.double() - ref).abs() - bound).max()), bool(x.isnan().any())
        assert not bad and worst <= lost, (name, worst)


# ----- attention: far offsets, exactly -----------------------------------------------
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("apart", [(1 << 21) + 8, (1 << 22) - 8, 1 << 22])
def test_tokens_far_apart(apart, d):
    """Queries, keys and values of one buffer whose tokens stand up to the kernels' largest stride apart, and beyond it, where
    they are copied: offsets of over 2^32 bytes, and each output and gradient within the bounds of near ones."""
    room_for(60)
    T, H, K = (5 << 30) // (2 * apart) + 40, 4, 2
    buffer = torch.empty(1, T, apart, device=DEV, dtype=torch.bfloat16)
    sizes = (2 * H * d, 2 * K * d, 2 * K * d)
    parts = buffer[..., -sum(sizes):].split(sizes, -1)
    for i, part in enumerate(parts):
        part.copy_(randn(*part.shape, seed=71 + i))
    q, k, v = (part.unflatten(-1, (-1, w)) for part, w in zip(parts, (d, d, 2 * d)))
    lam = torch.linspace(0.1, 0.9, H, device=DEV)
    check(q, k, v, lam)
    check(q[:, -3:], k, v, lam, lengths=torch.tensor([T - 1]), grads=False)


# ----- norm: the ends of float32 -----------------------------------------------------
def test_norm_where_squares_leave_float32():
    """Sums of squares beyond float32: zeros, and beside them what there is; below it, eps alone counts."""
    x, w = randn(4, 200, seed=81, dtype=torch.float32), randn(200, seed=82, dtype=torch.float32)
    x[1] *= 1e20
    x[2] *= 1e-30
    y = rms_norm(x, w)
    assert not y[1].any()
    keep = [0, 2, 3]
    ref, _, _, tol = oracle.norm(x[keep], w)
    assert ((y[keep].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("group", [128, None])
def test_scales_below_the_normal_numbers(group, fmt):
    most = torch.finfo(fmt).max * 2.0 ** -126              # the least of a group's largest that has a scale
    x = torch.zeros(3, 256, device=DEV)
    x[:, 0], x[:, 128] = 1.0, -1.0
    inv = (128 ** -1 + 1e-6) ** -0.5                        # two ones of 256
    for size, seen in ((4.0, True), (0.25, False)):
        codes, scale = rms_norm_fp8(x, torch.full((256,), size * most / inv, device=DEV), dtype=fmt, group=group)
        assert bool((codes.float() != 0).any()) == seen
        assert (scale == 1).all() if not seen else (scale < 1e-36).all() and (codes.float()[:, 0] == torch.finfo(fmt).max).all()
