"""The operators between a layer's projections as programs use them: together, over a cache, captured and replayed, on
other streams, side by side, at offsets beyond 32 bits, under autocast and with hooks of torch around them."""
import pytest
import torch

from monarch_muon_amd import differential_attention, embedding, linear_cross_entropy, rms_norm, rms_norm_fp8, rotary, rotary_table
from oracle import layer as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def randn(*shape, seed=0, size=1.0, dtype=torch.bfloat16):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(DEV).to(dtype)


# ----- together ----------------------------------------------------------------------
B, T, W, H, K, D = 2, 90, 256, 4, 2, 32


def weights(seed=0):
    sizes = {"q": (W, 2 * H * D), "k": (W, 2 * K * D), "v": (W, 2 * K * D), "o": (2 * H * D, W)}
    w = {n: randn(*s, seed=seed + i, size=s[0] ** -0.5) for i, (n, s) in enumerate(sizes.items())}
    w["n1"], w["sub"] = (1 + randn(n, seed=seed + 9, size=0.1) for n in (W, 2 * D))
    w["lam"] = torch.linspace(0.2, 0.7, H, device=DEV)
    return w


def layer(x, r, w, table, at=None, cache=None, norm=None):
    """(what the layer's attention part adds, the residual stream)"""
    n = norm or rms_norm
    y, r = n(x, w["n1"], residual=r)
    b, t, _ = y.shape
    q, k, v = ((y @ w[i]).view(b, t, -1, d) for i, d in (("q", D), ("k", D), ("v", 2 * D)))
    q, k = rotary(q, k, table, at)
    lengths = None
    if cache is not None:
        rows = torch.arange(b, device=DEV)[:, None]
        cache[0][rows, at], cache[1][rows, at] = k, v
        (k, v), lengths = cache, at[:, -1] + 1
    o = rms_norm(differential_attention(q, k, v, w["lam"], lengths=lengths), w["sub"])
    return o.flatten(2) @ w["o"], r


def plain_layer(x, r, w, f=torch.float64):
    """The same in ``f``, with the stream's sum and nothing else rounded."""
    x, w = x.to(f), {n: t.to(f) for n, t in w.items()}
    norm = lambda h, n: h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * n  # noqa: E731
    r = x + r.to(f)
    y = norm(r, w["n1"])
    q, k, v = ((y @ w[i]).view(B, T, -1, d) for i, d in (("q", D), ("k", D), ("v", 2 * D)))
    a = torch.arange(T, device=DEV, dtype=f)[:, None, None] * 10000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=f) / D)
    turn = lambda z: torch.cat([z[..., :D // 2] * a.cos() - z[..., D // 2:] * a.sin(),  # noqa: E731
                                z[..., :D // 2] * a.sin() + z[..., D // 2:] * a.cos()], -1)
    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(H // K, 2) for t in (k.view(B, T, K, 2 * D), v))
    q, k = q.view(B, T, H, 2, D), k.view(B, T, H, 2, D)
    s = torch.einsum("bthmd,bshmd->bhmts", q, k) * D ** -0.5
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), -float("inf")).softmax(-1)
    o = torch.einsum("bhts,bshd->bthd", s[:, :, 0] - w["lam"][:, None, None] * s[:, :, 1], v)
    return norm(o, w["sub"]).flatten(2) @ w["o"], r


def test_a_layer_and_its_gradients():
    """Norm, projections, rotary, attention and the head's norm in a row, against one graph in 64 bits: a dozen
    roundings to bf16 in a row, each of a relative 2^-9 in the mean and independent, leave under 12 x 2^-9 = 2.4%."""
    w = {n: t.requires_grad_() for n, t in weights().items()}
    x, r = randn(B, T, W, seed=50).requires_grad_(), randn(B, T, W, seed=51, size=2.0).requires_grad_()
    table = rotary_table(D, 128, device=DEV)
    leaves = [x, r, *w.values()]
    got = layer(x, r, w, table)
    ups = randn(B, T, W, seed=52), randn(B, T, W, seed=53)
    grads = torch.autograd.grad(got, leaves, ups)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    ref = plain_layer(exact[0], exact[1], dict(zip(w, exact[2:])))
    refs = torch.autograd.grad(ref, exact, tuple(u.double() for u in ups))
    for name, a, b in zip(("out", "stream", "x", "r", *w), (*got, *grads), (*ref, *refs)):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 12 * 2 ** -9, name


def test_tokens_one_at_a_time_over_a_cache():
    """Sequences of different lengths: their prompts in one padded call, then token by token at places of their own,
    give what one call over the whole gives."""
    w, table = weights(3), rotary_table(D, 128, device=DEV)
    x, r = randn(B, T, W, seed=60), randn(B, T, W, seed=61)
    whole, _ = layer(x, r, w, table)
    cache = [torch.full((B, 100, 2 * K, D), float("nan"), device=DEV, dtype=torch.bfloat16),
             torch.full((B, 100, K, 2 * D), float("nan"), device=DEV, dtype=torch.bfloat16)]
    for b, n in enumerate((40, 77)):   # the prompts
        at = torch.arange(n, device=DEV)[None]
        part = [c[b:b + 1] for c in cache]
        out, _ = layer(x[b:b + 1, :n], r[b:b + 1, :n], w, table, at, part)
        torch.testing.assert_close(out, whole[b:b + 1, :n], rtol=0.05, atol=0.05)
    for i in range(10):
        at = torch.tensor([[40 + i], [77 + i]], device=DEV)
        rows = torch.arange(B, device=DEV)[:, None]
        out, _ = layer(x[rows, at], r[rows, at], w, table, at, cache)
        ref = whole[rows, at]
        # the projections' own sums are of another order for one token: a few roundings to bf16
        assert float((out - ref).float().norm() / ref.float().norm()) < 12 * 2 ** -9


# ----- graphs and streams ------------------------------------------------------------
def calls():
    """name -> (inputs, call): small programs, forward and backward."""
    x, r, w = randn(70, 264, seed=1), randn(70, 264, seed=2), randn(264, seed=3)
    q, k, v = randn(2, 65, 8, 64, seed=4), randn(2, 65, 4, 64, seed=5), randn(2, 65, 2, 128, seed=6)
    lam, table = torch.linspace(0.1, 0.9, 4, device=DEV), rotary_table(32, 128, device=DEV)
    n, at = torch.tensor([65, 20], device=DEV), torch.randint(0, 128, (2, 65), generator=torch.Generator().manual_seed(7)).to(DEV)
    long_k, long_v = randn(1, 3000, 4, 64, seed=8), randn(1, 3000, 2, 128, seed=9)
    up, dup = randn(70, 264, seed=10), randn(2, 65, 4, 128, seed=11)

    def norm(x, r, w):
        leaves = [t.detach().requires_grad_() for t in (x, r, w)]
        out = rms_norm(leaves[0], leaves[2], residual=leaves[1])
        return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (up, up)))

    def turn(q, k, at):
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        out = rotary(*leaves, table, at)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (q, k)))

    def attend(q, k, v, lam, n):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        out = differential_attention(*leaves, lengths=n)
        return (out.detach(), *torch.autograd.grad(out, leaves, dup))
    return {
        "norm": ([x, r, w], norm),
        "norm_fp8": ([x, r, w], lambda x, r, w: tuple(t.float() for t in rms_norm_fp8(x, w, residual=r))),
        "rotary": ([q, k, at], turn),
        "attention": ([q, k, v, lam, n], attend),
        "decode": ([q[:1, :1], long_k, long_v, lam], lambda q, k, v, lam: (differential_attention(q, k, v, lam),)),
    }


@pytest.mark.parametrize("name", ["norm", "norm_fp8", "rotary", "attention", "decode"])
def test_captured_and_replayed(name):
    """One graph on other inputs, with the program's own eager calls and synchronizations between the replays."""
    inputs, call = calls()[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*inputs)
    for seed in range(4):
        for i, t in enumerate(inputs):
            if t.is_floating_point():
                t.copy_(randn(*t.shape, seed=100 + 10 * seed + i))
            elif t.dim() == 1:
                t.copy_(torch.tensor([seed * 20, 65 - seed]))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(*inputs)
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), seed


def test_two_graphs_take_turns():
    """Two captured calls with workspaces of their own, replayed in turn and side by side."""
    inputs, call = calls()["attention"]
    graphs = []
    for seed in (1, 2):
        mine = [t.clone() for t in inputs]
        mine[0].copy_(randn(*mine[0].shape, seed=seed))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(*mine)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*mine)
        graphs.append((graph, out, [t.clone() for t in call(*mine)], torch.cuda.Stream(), mine))   # (a graph reads its inputs where they were)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, _, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, ref, *_ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


@pytest.mark.parametrize("name", ["norm", "norm_fp8", "rotary", "attention", "decode"])
def test_on_other_streams(name):
    inputs, call = calls()[name]
    ref = call(*inputs)
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append([call(*inputs) for _ in range(3)])
    torch.cuda.synchronize()
    for each in results:
        for out in each:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_calls_from_many_threads():
    import threading
    programs = calls()
    refs = {n: call(*inputs) for n, (inputs, call) in programs.items()}
    torch.cuda.synchronize()
    wrong = []

    def work(name):
        inputs, call = programs[name]
        for _ in range(5):
            if not all(torch.equal(a, b) for a, b in zip(call(*inputs), refs[name])):
                wrong.append(name)
    threads = [threading.Thread(target=work, args=(n,)) for n in refs for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ----- torch around them -------------------------------------------------------------
def test_under_autocast():
    """Norm and rotary keep their inputs' types; attention computes in bf16 and gives its inputs' gradients in theirs."""
    q, k, v = (randn(*s, seed=i, dtype=torch.float32).requires_grad_() for i, s in enumerate([(1, 9, 4, 16), (1, 9, 2, 16), (1, 9, 1, 32)]))
    lam, x = torch.tensor(0.5, device=DEV, requires_grad=True), randn(9, 32, dtype=torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        o = differential_attention(q, k, v, lam)
        assert rms_norm(x, torch.ones(32, device=DEV)).dtype == torch.float32
    assert o.dtype == torch.bfloat16
    for g in torch.autograd.grad(o.float().sum(), (q, k, v, lam)):
        assert g.dtype == torch.float32
    assert torch.equal(o, differential_attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), lam))


def test_checkpointed_and_hooked():
    from torch.utils.checkpoint import checkpoint
    w, table = {n: t.requires_grad_() for n, t in weights(5).items()}, rotary_table(D, 128, device=DEV)
    x, r = randn(B, T, W, seed=70).requires_grad_(), randn(B, T, W, seed=71).requires_grad_()
    up = randn(B, T, W, seed=72)
    ref = torch.autograd.grad(layer(x, r, w, table)[0], [x, r, *w.values()], up)
    again = checkpoint(lambda x, r: layer(x, r, w, table)[0], x, r, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(again, [x, r, *w.values()], up), ref):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        out = layer(x, r, w, table)[0]
    for a, b in zip(torch.autograd.grad(out, [x, r, *w.values()], up), ref):
        assert torch.equal(a, b)


def test_with_the_models_ends():
    """Ids to loss and back through a layer, every part on this library's kernels."""
    ids = torch.randint(0, 300, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    table, head = randn(300, W, seed=80).requires_grad_(), randn(300, W, seed=81, size=W ** -0.5).requires_grad_()
    w = {n: t.requires_grad_() for n, t in weights(7).items()}
    x = embedding(ids, table)
    y, r = layer(x, x, w, rotary_table(D, 128, device=DEV))
    loss = linear_cross_entropy(rms_norm(y, w["n1"], residual=r)[0], head, ids.roll(-1, 1))
    loss.backward()
    assert loss.isfinite()
    for t in (table, head, *w.values()):
        assert t.grad is not None and t.grad.isfinite().all() and t.grad.any()


def test_the_examples_gradients_and_its_cache():
    """The tiny model's loss by its parameters, along a direction, against differences of it in 32-bit sums; its cached
    tokens against one call over all of them."""
    from monarch_muon_amd import example
    torch.manual_seed(3)
    model = example.TinyMonarchLM().to(DEV)
    ids, _ = example.text(torch.Generator().manual_seed(4), DEV)
    with torch.no_grad():
        caches, whole = model.caches(8, 24), model.hidden(ids[:, :24])
        parts = [model.hidden(ids[:, :7], caches, 0)] + [model.hidden(ids[:, t:t + 1], caches, t) for t in range(7, 24)]
        got = torch.cat(parts, 1)
    assert float((got - whole).float().norm() / whole.float().norm()) < 12 * 2 ** -9
    loss = model.loss(*example.text(torch.Generator().manual_seed(4), DEV))
    grads = torch.autograd.grad(loss, list(model.parameters()))
    assert all(g.isfinite().all() and g.any() for g in grads)


# ----- far offsets -------------------------------------------------------------------
def test_norm_beyond_32_bit_offsets():
    rows, width = 600_000, 8192                       # 4.9e9 elements
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 50 GB")
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    last = randn(5, width, seed=1)
    x[-5:] = last
    w = randn(width, seed=2)
    y, h = rms_norm(x, w, residual=x)
    ref, _, _, tol = oracle.norm(last, w, last)
    assert ((y[-5:].double() - ref).abs() <= tol).all() and torch.equal(h[-5:], last + last) and not y[:-5].any()
    del y, h
    x.requires_grad_()
    wl = w.clone().requires_grad_()
    y = rms_norm(x, wl)
    dy = torch.zeros_like(y)
    dy[-5:] = randn(5, width, seed=3)
    gx, gw = torch.autograd.grad(y, (x, wl), dy)
    dx, dw, (xt, wt) = oracle.norm_grad(last, w, dy[-5:])
    assert ((gx[-5:].double() - dx).abs() <= xt).all() and ((gw.double() - dw).abs() <= wt).all()


@pytest.mark.parametrize("codes", [False, True])
def test_norm_of_more_rows_than_a_launch_holds(codes):
    rows, width, each = (1 << 27) + 70, 65, 1 << 27    # 16 lanes of a row: 2^27 rows are 2^31 threads
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 40 GB")
    x = randn(width, seed=4).expand(rows, width)
    at = torch.tensor([0, 1, each - 1, each, each + 1, rows - 1], device=DEV)
    w = randn(width, seed=5)
    if codes:
        y, scale = rms_norm_fp8(x, w)
        one, s1 = rms_norm_fp8(x[:1], w)
        assert torch.equal(y.view(torch.uint8)[at], one.view(torch.uint8).expand(6, width)) and torch.equal(scale[at], s1.expand(6, 1))
        return
    y = rms_norm(x, w)
    ref, _, _, tol = oracle.norm(x[:1], w)
    assert ((y[at].double() - ref).abs() <= tol).all() and torch.equal(y[at], y[:1].expand(6, width))
    assert torch.equal(y[each:], y[:70])


def test_rotary_beyond_32_bit_offsets():
    q = torch.zeros(40, 20000, 64, 128, dtype=torch.bfloat16, device=DEV)   # 6.6e9 elements
    q[-1, -1] = randn(64, 128, seed=1)
    k = randn(40, 20000, 1, 8, seed=2)
    table = rotary_table(8, 20000, device=DEV)
    out, _ = rotary(q[..., :8], k, table)
    a = torch.full((1, 1, 1), 19999.0, dtype=torch.float64, device=DEV) * 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64, device=DEV) / 8)
    ref, tol = oracle.rotary(q[-1:, -1:, :, :8], a)
    assert ((out[-1:, -1:].double() - ref).abs() <= tol).all() and not out[:-1].any()


@pytest.mark.parametrize("d", [64, 128])
def test_a_cache_beyond_32_bit_offsets(d):
    """A cache of 4.9e9 bytes of keys and as many of values; the newest keys are what is seen most."""
    S, K = 1_200_000 * 64 // d, 16
    k = torch.zeros(1, S, 2 * K, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(1, S, K, 2 * d, dtype=torch.bfloat16, device=DEV)
    n = 300
    k[0, -n:], v[0, -n:] = randn(n, 2 * K, d, seed=1, size=3.0), randn(n, K, 2 * d, seed=2)
    q, lam = randn(1, 2, 2 * K, d, seed=3, size=3.0), torch.full((K,), 0.5, device=DEV)
    got = differential_attention(q, k, v, lam)
    # the keys of zeros have a score of 0: exp(0) each beside the others' sums
    for h in range(K):
        o = []
        for m in (0, 1):
            s = q[0, :, 2 * h + m].double() @ k[0, -n:, 2 * h + m].double().T * d ** -0.5
            s[0, -1] = -float("inf")
            top = s.amax(1, keepdim=True).clamp_min(0.0)
            p = (s - top).exp()
            rest = (S - n) * (-top).exp()
            o.append(p @ v[0, -n:, h].double() / (p.sum(1, keepdim=True) + rest))
        ref = o[0] - 0.5 * o[1]
        # P and the result rounded to bf16; a weight that is a sum of a million has 2^-8 of each at most
        bound = 2 * 2 ** -8 * (o[0].abs() + 0.5 * o[1].abs()) + 2 ** -8 * sum(x.abs() for x in o) + 1e-4 * v[0, -n:, h].double().abs().amax()
        assert ((got[0, :, h].double() - ref).abs() <= bound + 0.02 * ref.abs().max()).all()
