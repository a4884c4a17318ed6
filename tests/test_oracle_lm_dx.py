"""That the bounds for dx of the head's loss can see the term which adds back what bf16 took from dl at the target: the
kernel's arithmetic in torch on the CPU, right, and with that term wrong in the ways an index or a sign can be."""
import pytest
import torch

from oracle import lm as oracle

SHAPES = [(600, 776, 2500), (200, 520, 7000), (300, 264, 1000), (129, 256, 1023)]


def inputs(T, D, V, ignored):
    g = torch.Generator().manual_seed(T + V)
    w = (torch.randn(V, D, generator=g) / D ** 0.5).bfloat16()
    y = torch.randint(0, V, (T,), generator=g)
    x = (torch.randn(T, D, generator=g) + 4 * torch.rand(T, 1, generator=g) * w[y].float()).bfloat16()
    y[torch.rand(T, generator=g) < ignored] = -100
    return x, w, y


def emulate(x, w, y, reduction, grad, resid):
    """``resid``: what becomes of the term (r, targets) -> (r, targets)."""
    keep = y != -100
    yk = y[keep]
    l = x[keep].float() @ w.float().T
    lse = l.logsumexp(1)
    part = torch.nn.functional.pad(l, (0, -l.shape[1] % 64), value=-float("inf")).unflatten(1, (-1, 64)).amax(2)
    top = part.repeat_interleave(64, 1)[:, :l.shape[1]]
    code = ((top - l) * (1.4426950408889634 * 65535 / 64)).round().clamp(0, 65535)
    p = torch.where(code == 65535, 0.0, torch.exp2(-code * (64 / 65535) + (top - lse[:, None]) * 1.4426950408889634))
    g = torch.ones(len(yk)) if grad is None else grad[keep]
    term = g * torch.expm1(l.gather(1, yk[:, None])[:, 0] - lse)
    dl = (p * g[:, None]).bfloat16()
    rows = torch.arange(len(yk))
    dl[rows, yk] = term.bfloat16()
    r, at = resid(term - term.bfloat16().float(), yk)
    dx = torch.zeros_like(x)
    factor = 1 / len(yk) if reduction == "mean" else 1.0
    dx[keep] = ((dl.float() @ w.float() + r[:, None] * w[at].float()) * factor).bfloat16()
    return dx


def off(got, dx, bound, norm):
    """How far beyond the bounds: (elementwise, norm), at most 1 where within."""
    d = (got.double() - dx).abs()
    return float((d / bound).max()), float(d.norm() / norm)


@pytest.mark.parametrize("T, D, V", SHAPES)
@pytest.mark.parametrize("reduction, ignored", [("mean", 0.0), ("sum", 0.3), ("none", 0.3)])
def test_bounds_hold_and_see_the_targets_term(T, D, V, reduction, ignored):
    x, w, y = inputs(T, D, V, ignored)
    grad = torch.randn(T, generator=torch.Generator().manual_seed(1)) if reduction == "none" else None
    ref = oracle.head_dx(x, w, y, reduction=reduction, grad=grad)
    elementwise, norm = off(emulate(x, w, y, reduction, grad, lambda r, at: (r, at)), *ref)
    assert elementwise <= 1 and norm <= 1, (elementwise, norm)
    for what, wrong in (("left out", lambda r, at: (0 * r, at)), ("of the wrong sign", lambda r, at: (-r, at)),
                        ("of the token before", lambda r, at: (r.roll(1), at)),
                        ("at the target of the token before", lambda r, at: (r, at.roll(1))),
                        ("at the next word", lambda r, at: (r, (at + 1) % V)),
                        ("of every other token left out", lambda r, at: (r * (torch.arange(len(r)) % 2), at))):
        assert off(emulate(x, w, y, reduction, grad, wrong), *ref)[1] > 1, what
