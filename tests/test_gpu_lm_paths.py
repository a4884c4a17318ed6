"""More of the language-model operators on the GPU against their plain float64 forms: what ordinary calls reach beside
the sizes and layouts of test_gpu_lm.py."""
import pytest
import torch
import torch.utils.checkpoint

from monarch_muon_amd import embedding, linear_cross_entropy

from lm_paths import HEAD_PATHS
from oracle import lm as oracle
from test_gpu_lm import check_embedding, check_head, head, ids, within

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


# ----- derivatives of gradients ------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_embedding_gradient_derivative(dtype):
    """The derivative of the table's gradient by the gradient that arrived: scale * up[i], one rounding, and nothing for
    padding and for ids that are no token, whatever ``up`` holds there."""
    g = torch.Generator().manual_seed(1)
    i = torch.tensor([3, 0, 29, -1, 30, 2 ** 40, 3, 7], device=DEV).view(2, 4)
    w, up = (torch.randn(30, 24, generator=g).to(dtype).to(DEV) for _ in range(2))
    dout = torch.randn(2, 4, 24, generator=g).to(dtype).to(DEV).requires_grad_()
    up[7] = float("nan")
    dw, = torch.autograd.grad(embedding(i, w.requires_grad_(), scale=1.5, padding_idx=7), w, dout, create_graph=True)
    plain, = torch.autograd.grad(embedding(i, w, scale=1.5, padding_idx=7), w, dout.detach())
    assert torch.equal(dw, plain)
    d, = torch.autograd.grad(dw, dout, up)
    ref = torch.zeros(2, 4, 24, device=DEV)
    for r, c, v in ((0, 0, 3), (0, 1, 0), (0, 2, 29), (1, 2, 3)):
        ref[r, c] = up[v].float() * 1.5
    assert d.dtype == dtype and torch.equal(d, ref.to(dtype))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_gradient_of_a_kept_graph(reduction):
    """create_graph changes no value; a derivative of the gradients is refused."""
    g = torch.Generator().manual_seed(2)
    x, w = (torch.randn(n, 64, generator=g).bfloat16().to(DEV).requires_grad_() for n in (70, 300))
    y = torch.randint(0, 300, (70,), generator=g).to(DEV)
    want = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction).sum() / 4, (x, w))
    got = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction).sum() / 4, (x, w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(RuntimeError, match="no autograd formula"):
        (got[0].float().square().sum() + w.float().sum()).backward()


# ----- tilings of the products -------------------------------------------------------
@pytest.mark.parametrize("ignored", [0.0, 0.4])
@pytest.mark.parametrize("size, path", HEAD_PATHS, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
def test_head_paths(size, path, ignored):
    """Each tile and split over K that a product can take, the loss alone and with gradients."""
    T, D, V, piece = size
    x, w, y = (t.to(DEV) for t in head(T, D, V, seed=T + V, ignored=ignored))
    check_head(x, w, y, piece_tokens=piece)


# ----- what bf16 takes from dl at the target -----------------------------------------
@pytest.mark.parametrize("reduction, ignored", [("mean", 0.0), ("sum", 0.4), ("none", 0.4)])
@pytest.mark.parametrize("size", [(129, 256, 1023, None), (600, 776, 2500, None), (200, 520, 70000, None),
                                  (900, 264, 33000, 400)] + [s for s, _ in HEAD_PATHS],
                         ids=lambda s: "x".join(map(str, s)))
def test_dx_has_the_targets_term(size, reduction, ignored):
    """dx within the bounds that leave no rounding to dl at the target, unsplit, split, masked and in pieces."""
    T, D, V, piece = size
    x, w, y = (t.to(DEV) for t in head(T, D, V, seed=T + V, ignored=ignored))
    up = torch.randn(T, generator=torch.Generator().manual_seed(1)).to(DEV) if reduction == "none" else None
    dx, bound, norm = oracle.head_dx(x, w, y, reduction=reduction, grad=up)
    x.requires_grad_()
    got, = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction, piece_tokens=piece), x, up)
    within(got, dx, bound, "dx")
    off = float((got.double() - dx).norm())
    assert off <= float(norm), (off / float(norm), off / float(dx.norm()))


# ----- memory ------------------------------------------------------------------------
def peak(x, w, y, wrt, **kw):
    """Bytes beyond what stood before, with the gradients."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(linear_cross_entropy(x, w, y, **kw), wrt)
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, grads


def test_default_piece_counts_the_sums_that_pieces_keep():
    """6000 tokens of 131072 x 4096: their codes are 1.46 GiB, two pieces' 0.75 and 2 GiB of fp32 sums of dw.  All are
    one piece where the head is trained; a frozen one takes two, and no sums."""
    T, D, V = 6000, 4096, 131072
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(T, D, generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_()
    w = (torch.randn(V, D, generator=g, device=DEV) / 64).bfloat16().requires_grad_()
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    outputs, slack = 2 * D * (T + V), 512 << 20
    whole, (dx, dw) = peak(x, w, y, (x, w))
    assert whole <= 2 * T * V + outputs + slack, whole
    pieces, (px, pw) = peak(x, w, y, (x, w), piece_tokens=3072)
    assert whole < pieces
    frozen, (fx,) = peak(x, w.detach(), y, (x,))
    assert frozen <= (1 << 30) + 2 * D * T + slack, frozen
    only, (ow,) = peak(x.detach(), w, y, (w,))
    assert only <= whole
    # the pieces' sums are of the same terms
    for a, b in ((px, dx), (fx, dx), (pw, dw), (ow, dw)):
        assert float((a.float() - b.float()).norm()) <= 2.0 ** -8 * float(b.float().norm())


# ----- rows of whole 16-byte chunks ----------------------------------------------------
@pytest.mark.parametrize("T, D, V", [(1, 4, 3), (70, 12, 50), (5000, 1028, 300), (300, 516, 1000)])
def test_float_tables_of_whole_chunks(T, D, V):
    """float32 rows of 4 mod 8 columns, whole 16-byte chunks: against the plain form, and column by column the same bits
    as the wider table's, as the same chunks are summed the same way."""
    g = torch.Generator().manual_seed(T)
    w, dy = torch.randn(V, D + 4, generator=g).to(DEV), torch.randn(T, D + 4, generator=g).to(DEV)
    i = ids(T, V, T).to(DEV)
    check_embedding(i, w[:, :D].contiguous(), dy[:, :D].contiguous(), scale=0.5, pad=V - 1)
    check_embedding(i, w[:, :D], dy[:, :D])           # rows 4 mod 8 apart where D + 4 is
    wide, = torch.autograd.grad(embedding(i, w.requires_grad_()), w, dy)
    table = w.detach()[:, :D].contiguous().requires_grad_()
    narrow, = torch.autograd.grad(embedding(i, table), table, dy[:, :D].contiguous())
    assert torch.equal(narrow, wide[:, :D])


# ----- the gradient that arrives -------------------------------------------------------
@pytest.mark.parametrize("factor", [1 / 3, 0.7, -5.0, 2.0 ** -20, 0.0])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_head_upstream_factor(factor, reduction):
    """Gradients made by the forward, times a factor that arrives later: a second rounding, none for a power of two.
    With a loss per token the factor is in dl, and the result is rounded once."""
    x, w, y = (t.to(DEV) for t in head(300, 264, 1000, seed=31, ignored=0.2))
    _, dx, dw, (_, xt, wt) = oracle.cross_entropy(x, w, y, reduction=reduction)
    x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction) * factor, (x, w))
    one = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction), (x, w))
    f = float(torch.tensor(factor))
    for a, b, ref, bound in zip(got, one, (dx, dw), (xt, wt)):
        assert torch.equal(a, (b.float() * f).bfloat16())
        within(a, f * ref, abs(f) * bound + 1.01 * oracle.UBF * (f * ref).abs() + 1e-37, "twice rounded")
    if reduction == "sum":
        up = torch.full((300,), factor, device=DEV)
        _, dx, dw, (_, xt, wt) = oracle.cross_entropy(x.detach(), w.detach(), y, reduction="none", grad=up)
        got = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction="none"), (x, w), up)
        within(got[0], dx, xt, "dx, rounded once")
        within(got[1], dw, wt, "dw, rounded once")


# ----- values beyond the numbers ---------------------------------------------------------
@pytest.mark.parametrize("where", ["x inf", "x -inf", "x nan", "w inf", "all -inf"])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_a_token_without_a_softmax_has_no_number_in_its_gradients(where, reduction):
    """Infinities and NaN among the logits of a token that counts: loss and gradients are NaN where torch's are, in every
    place, also where a logit is -inf or lies far below an infinite one."""
    x, w, y = head(70, 64, 300, seed=8)
    y[y == 9] = 10
    if where == "all -inf":
        w[:, 5] = -w[:, 5].abs() - 1
        x[3, 5] = float("inf")
    else:
        (x if where[0] == "x" else w)[(3, 5) if where[0] == "x" else (9, 2)] = float(where[2:])
    x64, w64 = (t.double().requires_grad_() for t in (x, w))
    ref = torch.nn.functional.cross_entropy(x64 @ w64.T, y, reduction=reduction)
    want = torch.autograd.grad(ref.sum(), (x64, w64))
    x, w = (t.to(DEV).requires_grad_() for t in (x, w))
    out = linear_cross_entropy(x, w, y.to(DEV), reduction=reduction)
    got = torch.autograd.grad(out.sum(), (x, w))
    alone = linear_cross_entropy(x.detach(), w.detach(), y.to(DEV), reduction=reduction)
    for name, a, b in (("loss", out, ref), ("alone", alone, ref), ("dx", got[0], want[0]), ("dw", got[1], want[1])):
        assert torch.equal(a.isnan().cpu(), b.isnan()), (name, int(a.isnan().sum()), int(b.isnan().sum()))


@pytest.mark.parametrize("T", [3, 70, 300])
def test_logits_whose_powers_overflow_show(T):
    """A logit of 2.99e38 is a float32, 1 / ln 2 of it is not: the token's loss and gradients are NaN, not those of a
    softmax without that word."""
    x, w, y = head(T, 64, 300, seed=9)
    w[:, 0], w[200, 0], x[:, 0], x[1, 0] = 0, 2.0 ** 63, 0, 1.7578125 * 2.0 ** 64
    y[1] = 5
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
    row = torch.arange(T, device=DEV) == 1
    assert torch.equal(linear_cross_entropy(x.detach(), w.detach(), y, reduction="none").isnan(), row)
    out = linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert torch.equal(out.isnan(), row) and torch.equal(dx.isnan().any(1), row) and dw.isnan().all()


def test_words_whose_powers_underflow_have_none():
    """A part of the vocabulary whose logits are all -2.99e38 counts for nothing, as one whose logits are -inf does."""
    for low in (2.0 ** 63, float("inf")):
        x, w, y = head(70, 64, 300, seed=10)
        x[:, 0], w[:, 0] = 0, 0
        x[1, 0], w[256:, 0], y[1] = -1.7578125 * 2.0 ** 64, low, 5
        if low == float("inf"):
            x[:, 0] = -1        # (0 * inf is no number)
            y[y >= 256] = 6
        loss, dx, dw, (lt, xt, wt) = oracle.cross_entropy(x[1:2], w[:256], y[1:2], reduction="none")
        x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
        alone = linear_cross_entropy(x.detach(), w.detach(), y, reduction="none")
        out = linear_cross_entropy(x, w, y, reduction="none")
        got, = torch.autograd.grad(out, x, (torch.arange(70, device=DEV) == 1).float())
        within(alone[1], loss[0], lt[0], "alone")
        within(out[1], loss[0], lt[0], "loss")
        within(got[1, 1:], dx[0, 1:], xt[0, 1:], "dx")


# ----- under torch -------------------------------------------------------------------
@pytest.mark.parametrize("how", ["compile", "compile_dynamic", "saved_hooks", "checkpoint", "expanded_grad"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_operators_under_torch(reduction, how):
    """Embedding and loss traced by torch.compile, with saved-tensor hooks, recomputed by checkpointing and with a
    gradient that is no dense tensor: the bits of the plain call, with a factor that the backward multiplies in."""
    g = torch.Generator().manual_seed(4)
    t, w = ((torch.randn(300, 64, generator=g) / s).bfloat16().to(DEV).requires_grad_() for s in (1, 8))
    i, y = (torch.randint(0, 300, (90,), generator=g).to(DEV) for _ in range(2))
    i[5], y[7] = 1, -100

    def step(i, t, w, y):
        return linear_cross_entropy(embedding(i, t, scale=2.0, padding_idx=1), w, y, reduction=reduction) * 0.3
    loss = step(i, t, w, y)
    want = torch.autograd.grad(loss.sum(), (t, w))
    again = step
    if how.startswith("compile"):
        torch._dynamo.reset()
        again = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=how.endswith("dynamic"))
    elif how == "checkpoint":
        def again(*a):
            return torch.utils.checkpoint.checkpoint(step, *a, use_reentrant=False)
    with torch.autograd.graph.saved_tensors_hooks(*((lambda s: s.cpu(), lambda s: s.to(DEV)) if how == "saved_hooks" else
                                                    (lambda s: s, lambda s: s))):
        out = again(i, t, w, y)
    got = torch.autograd.grad(out.sum() if how != "expanded_grad" else out, (t, w),
                              None if how != "expanded_grad" else torch.ones((), device=DEV).expand(out.shape))
    assert torch.equal(out, loss) and all(torch.equal(a, b) for a, b in zip(got, want))
    torch._dynamo.reset()


# ----- more than one launch holds ------------------------------------------------------
def test_lookup_of_more_threads_than_a_launch_holds():
    """2^24 tokens and some of 1025 columns, 256 threads each: 2^32 and more threads."""
    T, D = (1 << 24) + 5, 1025
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randn(1000, D, generator=g, device=DEV).bfloat16()
    i = torch.randint(0, 1000, (T,), generator=g, device=DEV)
    out = embedding(i, w)
    for t in range(0, T, 1 << 21):
        assert torch.equal(out[t:t + (1 << 21)], w[i[t:t + (1 << 21)]]), t


def test_gradient_of_more_threads_than_a_launch_holds():
    """2^26 - 1 tokens of 1025 columns, the most there may be: the sums and their join in several launches.  Small whole
    numbers, so that every order of the sums is exact."""
    T, D, V = (1 << 26) - 1, 1025, 1000
    g = torch.Generator(device=DEV).manual_seed(6)
    i = torch.randint(0, V, (T,), generator=g, device=DEV)
    row = torch.randint(-2, 3, (D,), generator=g, device=DEV)
    count = torch.bincount(i, minlength=V)
    dw = torch.ops.mmuon.embedding_grad(row.bfloat16().expand(T, D), i, V, 1.0, -1)
    assert torch.equal(dw, (count[:, None] * row).float().bfloat16())
