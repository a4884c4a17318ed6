"""Differential attention on the GPU against its plain float64 form, within bounds derived from its roundings
(oracle/layer.py): lengths around the kernels' tiles, head sizes between them, shared heads, masks that leave a query
nothing, caches longer than their sequences, strides, values behind the last key that must not show."""
import pytest
import torch

from monarch_muon_amd import differential_attention
from oracle import layer as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAMES = ("o", "dq", "dk", "dv", "dlam")


def randn(*shape, seed=0, size=1.0):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).bfloat16().to(DEV)


def inputs(B, Tq, Tk, H, K, d, seed=0):
    lam = 0.2 + 0.6 * torch.rand(H, generator=torch.Generator().manual_seed(seed + 9))
    return (randn(B, Tq, 2 * H, d, seed=seed, size=1.5), randn(B, Tk, 2 * K, d, seed=seed + 1),
            randn(B, Tk, K, 2 * d, seed=seed + 2), lam.to(DEV))


def within(got, ref, bound, what):
    got = got.detach().double()
    assert got.shape == ref.shape, what
    assert not got.isnan().any(), what
    off = (got - ref).abs() - bound
    assert not off.numel() or float(off.max()) <= 0, (what, float(off.max()))
    # roundings to bf16 are independent of one another: their sum stays well below the sum of their bounds
    if ref.numel() > 1000 and float(ref.norm()) > 0:
        assert float((got - ref).norm() / ref.norm()) <= 2 ** -8, what


def check(q, k, v, lam, grads=True, **kw):
    dout = randn(q.shape[0], q.shape[1], q.shape[2] // 2, 2 * q.shape[3], seed=77) if grads else None
    refs, bounds = oracle.attention(q, k, v, lam, dout=dout, **kw)
    kw = {n: torch.as_tensor(t, device=DEV) if n in ("lengths", "starts") and t is not None else t for n, t in kw.items()}
    out = differential_attention(q, k, v, lam, **kw)
    assert out.dtype == torch.bfloat16 and out.is_contiguous()
    within(out, refs[0], bounds[0], "alone")
    if not grads:
        return
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    out = differential_attention(*leaves, **kw)
    got = torch.autograd.grad(out, leaves, dout)
    for name, x, ref, bound in zip(NAMES, (out, *got), refs, bounds):
        within(x, ref, bound, name)


@pytest.mark.parametrize("d", [8, 24, 32, 40, 64, 96, 128])
@pytest.mark.parametrize("Tq, Tk", [(1, 1), (2, 2), (31, 31), (32, 32), (33, 33), (65, 65), (130, 130)])
def test_causal(Tq, Tk, d):
    check(*inputs(2, Tq, Tk, 2, 2, d, seed=Tq + d))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Tq, Tk", [(1, 40), (5, 300), (40, 5), (100, 33), (64, 257), (300, 7)])
def test_queries_and_keys_of_different_numbers(Tq, Tk, causal, d):
    """More queries than keys: the first ones see none."""
    check(*inputs(1, Tq, Tk, 2, 1, d, seed=Tq + Tk), causal=causal)


@pytest.mark.parametrize("d", [64, 128, 32])
@pytest.mark.parametrize("H, K", [(6, 2), (8, 1), (5, 5), (12, 3)])
@pytest.mark.parametrize("Tq", [1, 45, 129])
def test_shared_heads(Tq, H, K, d):
    check(*inputs(2, Tq, 150, H, K, d, seed=H))


@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_rows(d):
    """Workgroups of eight waves: enough sequences and heads, rows that end inside a tile and inside a wave."""
    check(*inputs(12, 300, 300, 8, 8, d, seed=3))
    check(*inputs(24, 70, 333, 16, 8, d, seed=4), causal=False)


@pytest.mark.parametrize("d", [24, 32, 40, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_many_workgroups_of_both_maps(d, causal):
    """Workgroups whose waves have both maps: 256 of them, rows that end inside a wave, keys that end inside a tile."""
    check(*inputs(16, 300, 333, 8, 8, d, seed=13), causal=causal)


@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("B, T, H, K", [(1, 700, 1, 1), (2, 517, 4, 2), (1, 1100, 6, 1)])
def test_gradients_in_parts(d, B, T, H, K):
    """Few tiles of queries and of keys: both are split, parts of a triangle among them."""
    q, k, v, lam = inputs(B, T, T, H, K, d, seed=14)
    check(q, k, v, lam)
    check(q, k, v, lam, lengths=torch.tensor([T - 40, 0])[:B])


@pytest.mark.parametrize("B, T", [(700, 1), (300, 3), (90, 17), (9, 257)])
def test_many_short_sequences(B, T):
    check(*inputs(B, T, T, 4, 2, 64, seed=15))


@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("Tq, lengths", [(1, [0, 1, 31, 32, 33, 200]), (7, [5, 7, 8, 64, 199, 200]), (200, [0, 3, 150, 199, 200, 64])])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(Tq, lengths, causal, d):
    """What stands behind the last key reaches nothing, and gets zeros for its gradient."""
    q, k, v, lam = inputs(6, Tq, 200, 4, 2, d, seed=5)
    clean = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    n = torch.tensor(lengths)
    check(q, k, v, lam, causal=causal, lengths=n, grads=False)
    for b, m in enumerate(lengths):     # the same bits whatever stands there
        k[b, m:], v[b, m:] = clean[0][b, m:], clean[1][b, m:]
    poisoned = [t.clone() for t in (k, v)]
    for b, m in enumerate(lengths):
        poisoned[0][b, m:], poisoned[1][b, m:] = float("-inf"), float("nan")
    dout = randn(6, Tq, 4, 2 * d, seed=8)
    results = []
    for kk, vv in ((k, v), poisoned):
        leaves = [t.detach().requires_grad_() for t in (q, kk, vv, lam)]
        results.append(torch.autograd.grad(differential_attention(*leaves, causal=causal, lengths=n.to(DEV)), leaves, dout))
    for x, y in zip(*results):
        assert torch.equal(x, y)
    for b, m in enumerate(lengths):
        assert not results[0][1][b, m:].any() and not results[0][2][b, m:].any()
    check(q, k, v, lam, causal=causal, lengths=n)


@pytest.mark.parametrize("d", [64, 128])
def test_lengths_beyond_what_there_is(d):
    q, k, v, lam = inputs(3, 4, 50, 2, 2, d)
    check(q, k, v, lam, lengths=torch.tensor([-5, 50, 1 << 40]))
    check(q, k, v, lam, lengths=torch.tensor([7, 50, 90], dtype=torch.int32), starts=torch.tensor([0, -(1 << 62), 1 << 62]))


@pytest.mark.parametrize("d", [64, 128])
def test_starts(d):
    """A piece of each sequence's prompt, at a place of its own, over a cache."""
    q, k, v, lam = inputs(4, 37, 180, 4, 2, d, seed=2)
    check(q, k, v, lam, lengths=torch.tensor([37, 100, 180, 64]), starts=torch.tensor([0, 63, 100, 40]))
    check(q, k, v, lam, starts=torch.tensor([0, -10, 143, 500]))
    check(q, k, v, lam, starts=torch.tensor([0, -100, 10, 30]), lengths=torch.tensor([0, 20, 30, 30]))


@pytest.mark.parametrize("d, B, H, K, Tk, Tq", [(64, 1, 8, 2, 16384, 300), (32, 1, 8, 2, 9001, 300), (128, 3, 12, 6, 5102, 208),
                                                (104, 1, 4, 4, 4099, 1023), (48, 2, 2, 2, 3333, 3333), (128, 1, 1, 1, 4200, 4200)])
def test_split_keys_of_many_rows(d, B, H, K, Tk, Tq):
    """A prompt of few heads: workgroups of eight waves over parts of the keys."""
    q, k, v, lam = inputs(B, Tq, Tk, H, K, d, seed=16)
    check(q, k, v, lam)
    check(q, k, v, lam, causal=False, grads=False)
    lengths = torch.tensor([Tk - 700, 0, 3000])[:B]
    check(q, k, v, lam, lengths=lengths, grads=False)
    check(q, k, v, lam, lengths=lengths, starts=torch.tensor([3, 0, -100])[:B], grads=False)


@pytest.mark.parametrize("d, B, H, K, Tk, Tq", [(64, 1, 1, 1, 5000, 1), (128, 1, 2, 1, 3001, 1), (128, 3, 8, 2, 777, 1), (32, 2, 4, 4, 4097, 2),
                                                (64, 2, 6, 2, 1025, 5), (128, 1, 4, 1, 600, 33), (96, 1, 1, 1, 20000, 1), (64, 5, 2, 2, 129, 1)])
def test_split_keys(d, B, H, K, Tk, Tq):
    """Few rows: the keys in parts that are joined, some of them empty."""
    q, k, v, lam = inputs(B, Tq, Tk, H, K, d, seed=6)
    check(q, k, v, lam)
    lengths = torch.tensor([Tk, 3, Tk // 2, 0, 130])[:B]
    check(q, k, v, lam, lengths=lengths, grads=False)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_large_scores(d):
    """Scores far apart: references that move, maps that are one key's, and values that cancel."""
    q, k, v, lam = inputs(2, 150, 150, 2, 2, d, seed=11)
    k = (k.float() * torch.linspace(0.01, 6, 150, device=DEV)[None, :, None, None]).bfloat16()
    check(q, k, v, lam)
    check(q, k.flip(1).contiguous(), v, lam, causal=False)
    check((q.float() * 30).bfloat16(), k, v, lam, grads=False)
    check(q[:, :, [0, 0, 2, 2]], k[:, :, [0, 0, 2, 2]], v, torch.ones(2, device=DEV), grads=False)


def test_lam():
    """One value for all heads, none, negative, large; the gradient of one value is the sum of the heads'."""
    q, k, v, _ = inputs(2, 50, 50, 4, 2, 64, seed=12)
    for value in (0.0, -0.7, 1.0, 30.0):
        check(q, k, v, torch.full((4,), value, device=DEV))
    dout = randn(2, 50, 4, 128, seed=13)
    one, each = torch.tensor(0.4, device=DEV, requires_grad=True), torch.full((4,), 0.4, device=DEV, requires_grad=True)
    a, b = (differential_attention(q, k, v, t) for t in (one, each))
    assert torch.equal(a, b)
    (ga,), (gb,) = torch.autograd.grad(a, one, dout), torch.autograd.grad(b, each, dout)
    assert ga.shape == () and abs(float(ga - gb.sum())) <= 1e-5 * float(gb.abs().sum())
    half = torch.tensor([0.4], device=DEV, dtype=torch.bfloat16, requires_grad=True)
    (gh,) = torch.autograd.grad(differential_attention(q, k, v, half), half, dout)
    assert gh.dtype == torch.bfloat16 and gh.shape == (1,)


def test_scale():
    q, k, v, lam = inputs(1, 40, 40, 2, 2, 64, seed=14)
    for scale in (1e-3, 0.3, 2.0):
        check(q, k, v, lam, scale=scale)


def test_strides():
    """Heads of one fused projection, heads before tokens, a view that begins at an odd element, a broadcast batch."""
    B, T, H, K, d = 2, 70, 4, 2, 64
    fused = randn(B, T, (2 * H + 2 * K + 2 * K) * d, seed=15)
    q, k, v = (t.reshape(B, T, -1, w) for t, w in zip(fused.split([2 * H * d, 2 * K * d, 2 * K * d], -1), (d, d, 2 * d)))
    assert not q.is_contiguous() and not v.is_contiguous()
    lam = torch.linspace(0.1, 0.9, 2 * H, device=DEV)
    check(q, k, v, lam[::2])
    check(randn(B, 2 * H, T, d).transpose(1, 2), k, randn(B, K, T, 2 * d, seed=1).transpose(1, 2), lam[:H])
    check(randn(B, T, 2 * H * d + 1)[..., 1:].view(B, T, 2 * H, d), k, v, lam[:H])
    check(q, randn(1, T, 2 * K, d).expand(B, T, 2 * K, d), v, lam[:H])
    check(q[:1, :1], k[:1, 3:4], v[:1, 3:4], lam[:H])


@pytest.mark.parametrize("B, Tq, Tk, H, K", [(0, 3, 3, 2, 1), (2, 0, 3, 2, 1), (2, 3, 0, 2, 1), (2, 3, 3, 0, 1)])
def test_nothing(B, Tq, Tk, H, K):
    check(*inputs(B, Tq, Tk, H, K, 64))


def test_gradients_that_are_wanted():
    q, k, v, lam = inputs(1, 60, 60, 2, 1, 128, seed=16)
    dout = randn(1, 60, 2, 256, seed=17)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    every = torch.autograd.grad(differential_attention(*leaves), leaves, dout)
    for i in range(4):
        args = [t if i == j else t.detach() for j, t in enumerate(leaves)]
        (one,) = torch.autograd.grad(differential_attention(*args), args[i], dout)
        assert torch.equal(one, every[i])
    wide = torch.zeros(1, 60, 2, 257, device=DEV, dtype=torch.bfloat16)
    wide[..., 1:] = dout
    for x, y in zip(torch.autograd.grad(differential_attention(*leaves), leaves, wide[..., 1:]), every):
        assert torch.equal(x, y)


@pytest.mark.parametrize("d, B, T, H, K", [(16, 5, 531, 6, 6), (32, 1, 1431, 4, 4), (64, 2, 300, 24, 6), (128, 4, 229, 4, 4)])
def test_queries_gradient_is_rounded_once(d, B, T, H, K):
    """dq is its rounding away from the exact one, and little else: a uniform rounding to bf16 has 2^-8 / sqrt(3) at most."""
    q, k, v, lam = inputs(B, T, T, H, K, d, seed=17)
    dout = randn(B, T, H, 2 * d, seed=18)
    refs, _ = oracle.attention(q, k, v, lam, dout=dout)
    q.requires_grad_()
    dq, = torch.autograd.grad(differential_attention(q, k, v, lam), q, dout)
    assert float((dq.double() - refs[1]).norm() / refs[1].norm()) <= 2 ** -8 / 3 ** 0.5


@pytest.mark.parametrize("d", [32, 128])
def test_gradients_against_differences(d):
    """The directional derivative by differences of the float64 form; bf16 leaves its roundings."""
    q, k, v, lam = inputs(1, 40, 40, 2, 1, d, seed=18)
    dout = randn(1, 40, 2, 2 * d, seed=19)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    grads = torch.autograd.grad(differential_attention(*leaves), leaves, dout)
    along = [randn(*t.shape, seed=20 + i).double() for i, t in enumerate(leaves)]
    def loss(e):
        (o, *_), _ = oracle.attention(*(t.detach().double() + e * a for t, a in zip(leaves, along)))
        return float((o * dout.double()).sum())
    e = 1e-4
    for i, (g, a) in enumerate(zip(grads, along)):
        kept = along
        along = [a if i == j else torch.zeros_like(t) for j, t in enumerate(kept)]
        slope = (loss(e) - loss(-e)) / (2 * e)
        along = kept
        got, size = float((g.double() * a).sum()), float((g.double() * a).norm())
        # independent relative errors of up to 2^-8 at each of the gradient's elements: ten of their norm
        assert abs(got - slope) <= 10 * 2 ** -8 * size + 1e-5 * abs(slope), NAMES[i + 1]


def test_the_same_bits():
    q, k, v, lam = inputs(3, 200, 200, 6, 2, 64, seed=21)
    dout = randn(3, 200, 6, 128, seed=22)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    first = torch.autograd.grad(differential_attention(*leaves), leaves, dout)
    for _ in range(3):
        for x, y in zip(torch.autograd.grad(differential_attention(*leaves), leaves, dout), first):
            assert torch.equal(x, y)
