"""The language-model ends on the GPU against their plain float64 forms, within bounds derived from their roundings
(oracle/lm.py): sizes around the kernels' tiles and waves, ragged and odd vocabularies, strides, masks, and values
that could leak from masked places."""
import pytest
import torch

from monarch_muon_amd import embedding, linear_cross_entropy
from oracle import lm as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def head(T, D, V, seed=0, ignored=0.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) / D ** 0.5).bfloat16()
    y = torch.randint(0, V, (T,), generator=g)
    x = (spread * torch.randn(T, D, generator=g) + 4 * torch.rand(T, 1, generator=g) * w[y].float()).bfloat16()
    y[torch.rand(T, generator=g) < ignored] = -100
    return x, w, y


def within(got, ref, bound, what):
    got = got.detach().double().to(ref.device)
    assert got.shape == ref.shape, what
    assert torch.equal(got.isnan(), ref.isnan()), what
    off = (got - ref).abs()[~ref.isnan()] - torch.as_tensor(bound, device=ref.device).expand_as(ref)[~ref.isnan()]
    assert not off.numel() or float(off.max()) <= 0, (what, float(off.max()))


def check_head(x, w, y, reduction="mean", up=None, **kw):
    """x, w: device tensors (any strides); the loss alone, and with gradients."""
    loss, dx, dw, (lt, xt, wt) = oracle.cross_entropy(x, w, y, kw.get("ignore_index", -100), reduction, up)
    alone = linear_cross_entropy(x.detach(), w.detach(), y, reduction=reduction, **kw)
    within(alone, loss, lt, "loss alone")
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = linear_cross_entropy(x, w, y, reduction=reduction, **kw)
    within(out, loss, lt, "loss")
    gx, gw = torch.autograd.grad(out, (x, w), None if up is None else up.to(DEV))
    assert gx.dtype == gw.dtype == torch.bfloat16
    within(gx, dx, xt, "dx")
    within(gw, dw, wt, "dw")


@pytest.mark.parametrize("T, D, V", [(1, 8, 1), (1, 64, 50257), (2, 40, 2), (15, 32, 255), (16, 264, 256), (17, 512, 257),
                                     (33, 96, 1000), (63, 24, 4097), (64, 128, 333), (65, 200, 513), (127, 72, 129),
                                     (129, 256, 1023), (255, 32, 31), (257, 520, 8191), (600, 776, 2500)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_head_sizes(T, D, V, reduction):
    x, w, y = head(T, D, V, seed=T + V)
    check_head(x.to(DEV), w.to(DEV), y.to(DEV), reduction)


@pytest.mark.parametrize("T", [1, 32, 64])
@pytest.mark.parametrize("V", [31, 33, 127, 128, 129, 161, 98400])
def test_head_small_tiles(T, V):
    """The loss alone of up to 64 tokens, in tiles of 128 of the vocabulary: its edges, its parts of 32, and more tiles
    than are resident at a time (769 of them)."""
    x, w, y = head(T, 40, V, seed=T + V)
    y[0], y[-1] = 0, V - 1
    for reduction in ("mean", "none"):
        ref, _, _, (bound, _, _) = oracle.cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), -100, reduction)
        within(linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), reduction=reduction), ref, bound, reduction)


@pytest.mark.parametrize("T, D, V", [(1, 32, 100), (70, 64, 1000), (300, 72, 515)])
def test_head_per_token(T, D, V):
    x, w, y = head(T, D, V, seed=5, ignored=0.2)
    up = torch.randn(T, generator=torch.Generator().manual_seed(6))
    up[T // 2] = 0
    check_head(x.to(DEV), w.to(DEV), y.to(DEV), "none", up)


@pytest.mark.parametrize("ignored", [0.02, 0.5, 0.98, 1.0])
@pytest.mark.parametrize("T, piece", [(30, None), (300, None), (700, 256), (700, 100), (513, 1), (700, 699)])
def test_head_masks_and_pieces(T, piece, ignored):
    if piece == 1:
        T = 5
    x, w, y = head(T, 64, 777, seed=T, ignored=ignored)
    for reduction in ("mean", "sum"):
        check_head(x.to(DEV), w.to(DEV), y.to(DEV), reduction, piece_tokens=piece)


@pytest.mark.parametrize("T, D, V, piece", [
    (1000, 2048, 16640, None),   # 260 tiles of logits: the last four split over the width, the last tiles of dw too
    (1100, 1032, 16500, None),   # the same, with edges in every direction
    (200, 520, 70000, None),     # dx of a few tiles: all split over the vocabulary
    (128, 2048, 45000, None),    # dw beyond the Infinity Cache's share: stored past it
    (900, 264, 33000, 400),      # pieces, the last one shorter, dw carried from one to the next
])
@pytest.mark.parametrize("ignored", [0.0, 0.4])
def test_head_splits(T, D, V, piece, ignored):
    x, w, y = (t.to(DEV) for t in head(T, D, V, seed=T + D, ignored=ignored))
    check_head(x, w, y, piece_tokens=piece)


def test_head_pieces_agree_where_no_sum_crosses_them():
    x, w, y = head(1000, 128, 3000, ignored=0.3)
    x, w, y = x.to(DEV), w.to(DEV), y.to(DEV)
    whole = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.equal(whole, linear_cross_entropy(x, w, y, reduction="none"))
    grads = []
    for piece in (None, 256, 500):
        a = x.clone().requires_grad_()
        grads.append(torch.autograd.grad(linear_cross_entropy(a, w, y, reduction="sum", piece_tokens=piece), a)[0])
    for g in grads[1:]:
        assert float((g - grads[0]).float().norm()) <= 2.0 ** -7 * float(grads[0].float().norm())


def test_head_offsets_beyond_32_bits():
    """A piece of 2.4e9 logits against small pieces, and rows of it against the plain form."""
    x, w, y = (t.to(DEV) for t in head(48000, 8, 50304, seed=30, ignored=0.01))
    nll = linear_cross_entropy(x, w, y, reduction="none", piece_tokens=48000)
    assert torch.equal(nll, linear_cross_entropy(x, w, y, reduction="none", piece_tokens=4096))
    whole = x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(whole, w, y, reduction="sum", piece_tokens=48000), whole)
    rows = torch.cat([torch.arange(3), torch.arange(47997, 48000)]).to(DEV)
    loss, rx, _, (lt, xt, _) = oracle.cross_entropy(x[rows], w, y[rows], reduction="none", grad=torch.ones(6))
    within(nll[rows], loss, lt, "loss")
    within(dx[rows], rx, xt, "dx")


def test_head_empty():
    w = torch.ones(40, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = torch.empty(0, device=DEV, dtype=torch.long)
    assert linear_cross_entropy(x, w, y, reduction="none").shape == (0,)
    assert linear_cross_entropy(x, w, y).isnan()
    loss = linear_cross_entropy(x, w, y, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert float(loss.detach()) == 0 and dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("layout", ["rows", "transposed", "odd start", "expanded", "batch", "int32"])
def test_head_layouts(layout):
    x, w, y = head(50, 64, 300, seed=9, ignored=0.1)
    x, w, y = x.to(DEV), w.to(DEV), y.to(DEV)
    if layout == "rows":
        x = torch.cat([x, x + 1, x], 1)[:, 64:128] - 1
        wide = torch.zeros(300, 200, device=DEV, dtype=torch.bfloat16)
        wide[:, 8:72] = w
        wide_x = torch.full((50, 136), float("nan"), device=DEV, dtype=torch.bfloat16)
        wide_x[:, 16:80] = x
        x, w = wide_x[:, 16:80], wide[:, 8:72]
    elif layout == "transposed":
        x, w = x.T.contiguous().T, w.T.contiguous().T
    elif layout == "odd start":
        x = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(50, 64)
        w = torch.cat([w.new_zeros(3), w.reshape(-1)])[3:].view(300, 64)
    elif layout == "expanded":
        x = x[:1].expand(50, 64)
    elif layout == "int32":
        y = y.int()
    if layout == "batch":
        a, b = x.view(5, 10, 64).requires_grad_(), w.requires_grad_()
        out = linear_cross_entropy(a, b, y.view(5, 10), reduction="none")
        flat = linear_cross_entropy(x, w, y, reduction="none")
        assert out.shape == (5, 10) and torch.equal(out.view(-1), flat)
        assert torch.autograd.grad(out.sum(), a)[0].shape == a.shape
    else:
        check_head(x, w, y)


def test_head_ignored_rows_reach_nothing():
    """NaN and infinities in the hidden states of ignored tokens; another ignore_index, one that is a token."""
    x, w, y = head(400, 64, 500, seed=11, ignored=0.3)
    y[y == -100] = 7
    x, w, y = x.to(DEV), w.to(DEV), y.to(DEV)
    bad = x.clone()
    bad[y == 7] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 16, device=DEV).bfloat16()
    outs = []
    for a in (x, bad):
        a, b = a.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, y, ignore_index=7)
        outs.append((loss, *torch.autograd.grad(loss, (a, b))))
    assert all(torch.equal(p, q) and not p.isnan().any() for p, q in zip(*outs))
    assert float(outs[0][1][y == 7].abs().sum()) == 0
    check_head(x, w, y, ignore_index=7)


def test_head_extreme_logits():
    """Logits of thousands, a certain target, and a vocabulary part that lies far below the others."""
    x, w, y = head(130, 64, 1000, seed=12)
    x[:64] *= 200
    x[64:100] = 8 * w[y[64:100]] * 64
    w[300:800] -= (x[5].float().sign() * 50).bfloat16()
    check_head(x.to(DEV), w.to(DEV), y.to(DEV))


def test_head_bad_values_show():
    """NaN in a token's hidden state and a target that is no token give NaN for that token, and only there."""
    x, w, y = head(90, 32, 400, seed=13)
    x[3, 5] = float("nan")
    y[10], y[20], y[21] = 400, -1, 2 ** 40
    out = linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), reduction="none").cpu()
    expect = torch.zeros(90, dtype=torch.bool)
    expect[[3, 10, 20, 21]] = True
    assert torch.equal(out.isnan(), expect)
    a = x.to(DEV).requires_grad_()
    g, = torch.autograd.grad(linear_cross_entropy(a, w.to(DEV), y.to(DEV), reduction="sum"), a)
    assert torch.equal(g.isnan().any(1).cpu(), expect)


def test_head_gradient_against_differences():
    x, w, y = head(20, 32, 60, seed=14)
    xd, wd, yd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
    dx, dw = torch.autograd.grad(linear_cross_entropy(xd, wd, yd, reduction="sum"), (xd, wd))
    for t, d, which in ((x, dx, 0), (w, dw, 1)):
        for i in range(0, t.numel(), 61):
            ends, h = [], 0.0
            for step in (-0.25, 0.25):
                u = t.clone()
                u.view(-1)[i] += step
                h += float(u.view(-1)[i] - t.view(-1)[i]) * (1 if step > 0 else -1)
                a = [x, w]
                a[which] = u
                ends.append(float(linear_cross_entropy(a[0].to(DEV), a[1].to(DEV), yd, reduction="sum")))
            # third derivatives of the loss are below 20 max(|x|, |w|)^3, the loss is exact to 1e-4
            slope = (ends[1] - ends[0]) / h
            got = float(d.view(-1)[i])
            assert abs(slope - got) <= 0.05 * (1 + abs(got)) + 0.25 * abs(got), (which, i, slope, got)


def test_head_upstream_factor_and_one_backward():
    x, w, y = head(100, 64, 500, seed=15, ignored=0.1)
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
    one = torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    quarter = torch.autograd.grad(linear_cross_entropy(x, w, y) / 4, (x, w))
    assert all(torch.equal(a / 4, b) for a, b in zip(one, quarter))
    loss = linear_cross_entropy(x, w, y)
    torch.autograd.grad(loss, (x, w), retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss, (x, w))
    only, = torch.autograd.grad(linear_cross_entropy(x, w.detach(), y), x)
    assert torch.equal(only, one[0])
    only, = torch.autograd.grad(linear_cross_entropy(x.detach(), w, y), w)
    assert torch.equal(only, one[1])


def test_head_repeats_itself_and_follows_the_stream():
    x, w, y = head(500, 128, 5000, seed=16, ignored=0.2)
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
    ref = torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, again))


def test_head_in_a_graph():
    """Captured once and replayed on other inputs, with eager work between the replays."""
    x, w, y = (t.to(DEV) for t in head(300, 64, 1000, seed=17, ignored=0.2))
    x.requires_grad_()
    w.requires_grad_()

    def step():
        loss = linear_cross_entropy(x, w, y)
        return (loss, *torch.autograd.grad(loss, (x, w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (18, 19, 20):
        nx, _, ny = head(300, 64, 1000, seed=seed, ignored=0.1 * (seed - 17))
        with torch.no_grad():
            x.copy_(nx)
            y.copy_(ny)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), seed


def test_head_under_autocast():
    x, w, y = head(40, 64, 200, seed=21)
    x, w, y = x.float().to(DEV).requires_grad_(), w.float().to(DEV).requires_grad_(), y.to(DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.dtype == dw.dtype == torch.float32
    ref, ox, ow, (lt, xt, wt) = oracle.cross_entropy(x.detach(), w.detach(), y)
    within(loss, ref, lt, "loss")
    within(dx, ox, xt, "dx")
    within(dw, ow, wt, "dw")


# ----- embedding -----------------------------------------------------------------
def ids(n, vocab, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), vocab // 2)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return ((vocab + 1) ** u - 1).long().clamp_(0, vocab - 1) if kind == "zipf" else torch.randint(0, vocab, (n,), generator=g)


def check_embedding(i, w, dy, scale=1.0, pad=None):
    wd = w.detach().requires_grad_()
    out = embedding(i, wd, scale=scale, padding_idx=pad)
    assert torch.equal(out, (w[i].float() * scale).to(w.dtype))
    dw, = torch.autograd.grad(out, wd, dy)
    ref, bound = oracle.embedding_grad(dy, i, w.shape[0], scale, pad)
    u = 2.0 ** -24 if w.dtype == torch.float32 else 2.0 ** -8
    within(dw, ref, bound + 1.01 * u * ref.abs(), "dw")
    again, = torch.autograd.grad(embedding(i, wd, scale=scale, padding_idx=pad), wd, dy)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T, D, V", [(1, 1, 1), (1, 4096, 300), (3, 7, 2), (63, 8, 255), (64, 65, 257), (65, 512, 1000),
                                     (1000, 768, 5000), (1023, 100, 50257), (1025, 264, 31), (5000, 24, 131072),
                                     (4097, 1032, 90)])
def test_embedding_sizes(T, D, V, dtype):
    g = torch.Generator().manual_seed(T)
    w, dy = torch.randn(V, D, generator=g).to(dtype).to(DEV), torch.randn(T, D, generator=g).to(dtype).to(DEV)
    check_embedding(ids(T, V, T).to(DEV), w, dy)
    check_embedding(ids(T, V, T, "even").to(DEV), w, dy, scale=D ** 0.5, pad=V - 1)


@pytest.mark.parametrize("T", [40, 2000, 20000])
def test_embedding_of_one_word(T):
    g = torch.Generator().manual_seed(T)
    for D, dtype in ((64, torch.bfloat16), (33, torch.float32), (1024, torch.bfloat16)):
        w, dy = torch.randn(700, D, generator=g).to(dtype).to(DEV), torch.randn(T, D, generator=g).to(dtype).to(DEV)
        i = ids(T, 700, 0, "one").to(DEV)
        check_embedding(i, w, dy)
        i[::3] = 5
        i[1::7] = 699
        check_embedding(i, w, dy, scale=0.5, pad=5)


def test_embedding_shapes_layouts_and_empty():
    g = torch.Generator().manual_seed(4)
    w = torch.randn(50, 48, generator=g).bfloat16().to(DEV)
    i = ids(24, 50, 4).to(DEV).view(2, 3, 4)
    assert embedding(i, w).shape == (2, 3, 4, 48)
    assert torch.equal(embedding(i.int().permute(2, 0, 1), w), w[i.permute(2, 0, 1)])
    assert torch.equal(embedding(i[0, 0, 0], w), w[i[0, 0, 0]])
    wide = torch.full((50, 101), float("nan"), device=DEV, dtype=torch.bfloat16)
    for lo in (0, 1, 8):
        wide[:, lo:lo + 48] = w
        assert torch.equal(embedding(i, wide[:, lo:lo + 48]), w[i])
    assert torch.equal(embedding(i, w.T.contiguous().T), w[i])
    wd = w.clone().requires_grad_()
    none = embedding(torch.empty(0, 3, dtype=torch.long, device=DEV), wd)
    assert none.shape == (0, 3, 48) and torch.equal(torch.autograd.grad(none.sum(), wd)[0], torch.zeros_like(w))
    # a gradient with other strides, at an odd element, and one that is broadcast
    i = i.view(-1)
    dy = torch.randn(24, 48, generator=g).bfloat16().to(DEV)
    ref, = torch.autograd.grad(embedding(i, wd), wd, dy)
    for other in (dy.T.contiguous().T, torch.cat([dy, dy], 1)[:, :48], torch.cat([dy.new_zeros(1), dy.reshape(-1)])[1:].view(24, 48)):
        assert torch.equal(torch.autograd.grad(embedding(i, wd), wd, other)[0], ref)
    check_embedding(i, w, dy[:1].expand(24, 48))


def test_embedding_offsets_beyond_32_bits():
    V, D = 1100000, 2048
    w = torch.zeros(V, D, device=DEV, dtype=torch.bfloat16)
    i = torch.tensor([0, V - 1, 1048576, V - 1], device=DEV)
    w[i[:3]] = torch.randn(3, D, device=DEV).bfloat16()
    assert torch.equal(embedding(i, w), w[i])
    dy = torch.randn(4, D, device=DEV).bfloat16()
    wd = w.requires_grad_()
    dw, = torch.autograd.grad(embedding(i, wd), wd, dy)
    assert torch.equal(dw[V - 1], (dy[1].float() + dy[3].float()).bfloat16())
    assert torch.equal(dw[0], dy[0]) and torch.equal(dw[1048576], dy[2]) and int(dw.any(1).sum()) == 3


def test_embedding_ids_that_are_no_token():
    g = torch.Generator().manual_seed(7)
    w, dy = torch.randn(30, 16, generator=g).to(DEV), torch.randn(6, 16, generator=g).to(DEV)
    i = torch.tensor([3, -1, 30, 2 ** 40, 3, -2 ** 40], device=DEV)
    wd = w.clone().requires_grad_()
    out = embedding(i, wd)
    good = (i >= 0) & (i < 30)
    assert torch.equal(out.isnan().all(1), ~good) and torch.equal(out[good], w[i[good]])
    dy[~good] = float("nan")
    dw, = torch.autograd.grad(out, wd, dy)
    ref = torch.zeros_like(w)
    ref[3] = dy[0] + dy[4]
    assert torch.equal(dw, ref)


def test_embedding_padding_takes_nothing():
    """NaN in the gradient of padding tokens reaches no row; a padding row counted from the end."""
    g = torch.Generator().manual_seed(8)
    w, dy = torch.randn(30, 16, generator=g).bfloat16().to(DEV), torch.randn(200, 16, generator=g).bfloat16().to(DEV)
    i = ids(200, 30, 8, "even").to(DEV)
    dy[i == 29] = float("nan")
    wd = w.clone().requires_grad_()
    a, = torch.autograd.grad(embedding(i, wd, padding_idx=29), wd, dy)
    b, = torch.autograd.grad(embedding(i, wd, padding_idx=-1), wd, dy)
    assert torch.equal(a, b) and not a.isnan().any() and float(a[29].abs().sum()) == 0
    check_embedding(i, w, torch.nan_to_num(dy), pad=29)


def test_embedding_in_a_graph_and_on_another_stream():
    g = torch.Generator().manual_seed(9)
    w, dy = torch.randn(300, 64, generator=g).to(DEV).requires_grad_(), torch.randn(500, 64, generator=g).to(DEV)
    i = ids(500, 300, 1).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(embedding(i, w), w, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, = torch.autograd.grad(embedding(i, w), w, dy)
    for seed in (2, 3, 4):
        i.copy_(ids(500, 300, seed, "zipf" if seed < 4 else "one"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, torch.autograd.grad(embedding(i, w), w, dy)[0]), seed


# ----- together --------------------------------------------------------------------
def test_example_learns_and_scores():
    """Embedding, Monarch layers, loss, backward, optimizer, generation of single tokens."""
    from monarch_muon_amd import example
    model, losses = example.train(steps=60)
    assert losses.isfinite().all() and float(losses[0]) > 5.5 and float(losses[-5:].mean()) < 3.0, losses
    tokens, scores = example.generate(model, 7, 4)
    assert all(0 <= t < example.VOCAB for t in tokens) and all(-6.3 < s <= 0 for s in scores)
    # the loss of the example's own calls against the plain form on the same hidden states
    ids, targets = example.text(torch.Generator().manual_seed(5), DEV)
    with torch.no_grad():
        h = model.hidden(ids).reshape(-1, example.WIDTH)
        got = model.loss(ids, targets)
    ref, _, _, (bound, _, _) = oracle.cross_entropy(h, model.lm_head.detach(), targets.reshape(-1), ignore_index=example.PAD)
    within(got, ref, bound, "loss")
