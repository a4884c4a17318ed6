"""Plain float64 forms of the language-model ends (test infrastructure): the head's cross entropy with its gradients
and the embedding with its gradient, and how far a kernel that computes them with the stated roundings may be off.

Roundings of ``linear_cross_entropy``: bf16 products summed in fp32 (unit roundoff 2^-24 per step), p from a 16-bit
code (relative 2^-11 ln 2 at most, zero below 2^-64 of a part's maximum), dl and the results rounded to bf16 (2^-8)."""
from __future__ import annotations

import torch

U32, UBF = 2.0 ** -24, 2.0 ** -8
UCODE = 2.0 ** -11 * 0.6932


def cross_entropy(x, w, target, ignore_index=-100, reduction="mean", grad=None):
    """(loss, dx, dw, bounds): float64, where x is; ``bounds`` = (of loss, dx, dw) elementwise."""
    dev, f64 = x.device, torch.float64
    x, w = x.double(), w.double().to(dev)
    target = target.to(dev).long()
    T, D = x.shape
    V = w.shape[0]
    keep = target != ignore_index
    xk, yk = x[keep], target[keep]
    n = len(yk)
    l = xk @ w.T
    lse = torch.logsumexp(l, 1)
    nll = torch.zeros(T, dtype=f64, device=dev)
    ly = l.gather(1, yk[:, None])[:, 0]
    nll[keep] = lse - ly
    # a logit: D fp32 roundings of partial sums no larger than sum |x w|; log2 e, its power, the sum over V in
    # parts, the logarithm
    size = (xk.abs() @ w.abs().T).amax(1) if n else torch.zeros(0, dtype=f64, device=dev)
    err = U32 * (2 * (D + 4) * size + 4 * lse.abs() + V ** 0.5 + 40)
    tol = torch.zeros(T, dtype=f64, device=dev)
    tol[keep] = err
    if grad is not None:
        g = grad.double().to(dev)[keep]
    elif reduction == "mean":
        g = torch.full((n,), 1.0 / n if n else 0.0, dtype=f64, device=dev)
    else:
        g = torch.ones(n, dtype=f64, device=dev)
    p = (l - lse[:, None]).exp()
    dl = p.clone()
    dl[torch.arange(n, device=dev), yk] -= 1
    dl = dl * g[:, None]
    # p: its logit and lse, its code, bf16; the target's entry p - 1 has the error of p by nll
    rel = UCODE + UBF + 2 * err[:, None] + 2.0 ** -18
    off = dl.abs() * rel + (p * g.abs()[:, None]) * (2 * err[:, None] + 4 * U32) + g.abs()[:, None] * 1e-19
    dx, dxt = torch.zeros_like(x), torch.zeros_like(x)
    dx[keep] = dl @ w
    dxt[keep] = off @ w.abs() + 2 * V * U32 * (dl.abs() @ w.abs())
    dw = dl.T @ xk
    dwt = off.T @ xk.abs() + 2 * (n + 1) * U32 * (dl.abs().T @ xk.abs())
    loss, lt = {"none": (nll, tol),
                "sum": (nll.sum(), tol.sum() + 2 * (T + 20) * U32 * nll.abs().sum()),
                "mean": (nll.sum() / n if n else nll.sum() * float("nan"),
                         (tol.sum() + 2 * (T + 20) * U32 * nll.abs().sum()) / max(n, 1))}[reduction]
    return loss, dx, dw, (lt, dxt + 1.01 * UBF * dx.abs() + 1e-37, dwt + 1.01 * UBF * dw.abs() + 1e-37)


def embedding_grad(dout, index, vocab, scale=1.0, padding_idx=None):
    """(dw, bound of an fp32 sum in any order before the last rounding), float64 on the CPU."""
    dout, index = dout.double().cpu().reshape(index.numel(), -1), index.cpu().long().reshape(-1)
    keep = (index >= 0) & (index < vocab)
    if padding_idx is not None:
        keep &= index != padding_idx
    dw = torch.zeros(vocab, dout.shape[1], dtype=torch.float64)
    dw.index_add_(0, index[keep], dout[keep])
    size = torch.zeros_like(dw).index_add_(0, index[keep], dout[keep].abs())
    count = torch.bincount(index[keep], minlength=vocab).double()
    return dw * scale, (count + 2)[:, None] * U32 * size * abs(scale)


def head_dx(x, w, target, ignore_index=-100, reduction="mean", grad=None):
    """(dx, elementwise bound, bound of the norm of the difference) where the target's entry p - 1 of dl reaches dx in
    fp32: bf16's rounding of it is added back, so it has the error of p by nll alone.  The other entries' roundings
    differ from one another; the norm of their sum is that of independent errors of at most their size, and with the
    rounding of the result (its norm known) the two add in squares.  5% for what sums of many thousands may stray."""
    dev = x.device
    x64, w64, target = x.double(), w.double().to(dev), target.to(dev).long()
    _, dx, _, (_, bound, _) = cross_entropy(x, w, target, ignore_index, reduction, grad)
    keep = target != ignore_index
    xk, yk = x64[keep], target[keep]
    n, rows = len(yk), torch.arange(len(yk), device=dev)
    p = torch.softmax(xk @ w64.T, 1)
    g = grad.double().to(dev)[keep] if grad is not None else torch.full((n,), 1.0 / max(n, 1) if reduction == "mean" else 1.0,
                                                                        dtype=torch.float64, device=dev)
    at_target = (g * (1 - p[rows, yk])).abs()
    bound[keep] -= (at_target * (UCODE + UBF))[:, None] * w64[yk].abs()
    dl = p * g[:, None]
    dl[rows, yk] = 0
    others = (dl.square() @ w64.square()).sum() * (UBF + UCODE) ** 2
    rounding = (dx.bfloat16().double() - dx).square().sum()
    return dx, bound, 1.05 * (others + rounding).sqrt()
