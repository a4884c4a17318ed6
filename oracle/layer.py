"""Plain float64 forms of what stands between a layer's projections (test infrastructure), and how far a kernel that
computes them with the stated roundings may be off, elementwise.

Roundings: sums and products in fp32 (2^-24 each), results rounded once to their type (half of its eps)."""
from __future__ import annotations

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest magnitude's step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ----- norm ------------------------------------------------------------------------
# A lane sums at most 64 squares one after another and joins its sum with 511 others in a tree, or in eight waves' order:
# 64 + 6 + 8 roundings of a sum of positive numbers; the division, eps, the root and its reciprocal 4 more.
_SUM = 64 + 6 + 8


def norm(x, w, residual=None, eps=1e-6):
    """(y, h, inv, bound of y): h in x's type, the others float64."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    hd, wd = h.double(), w.double()
    inv = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    y = hd * inv * wd
    return y, h, inv, y.abs() * (half_step(x.dtype) + (_SUM / 2 + 6) * U32) + tiny(x.dtype)


def norm_grad(h, w, dy, dh=None, eps=1e-6):
    """(dx, dw, bounds): of y's gradient dy and h's dh."""
    hd, wd, g = h.double(), w.double(), dy.double()
    D = h.shape[-1]
    inv = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    n = g * wd
    dot = (n * hd).sum(-1, keepdim=True)
    dx = inv * n - hd * inv ** 3 * dot / D
    rel = (3 * (_SUM / 2 + 4) + _SUM + 10) * U32
    tol = rel * ((inv * n).abs() + hd.abs() * inv ** 3 * (n * hd).abs().sum(-1, keepdim=True) / D)
    if dh is not None:
        dx = dx + dh.double()
        tol = tol + U32 * dx.abs()
    each = (g * hd * inv).reshape(-1, D)
    dw = each.sum(0)
    dw_tol = each.abs().sum(0) * (each.shape[0] + 60) * U32 + half_step(w.dtype) * dw.abs() + tiny(w.dtype)
    return dx, dw, (tol + half_step(h.dtype) * dx.abs() + tiny(h.dtype), dw_tol)


def norm_scale(y, dtype, group):
    """The float64 scale of each 128 columns, or the row's."""
    D = y.shape[-1]
    G = group or D
    most = torch.nn.functional.pad(y, (0, -D % G)).unflatten(-1, (-1, G)).abs().amax(-1) / torch.finfo(dtype).max
    return torch.where(most > 0, most, 1.0)


def code_step(z, dtype):
    """The distance between codes around z."""
    f = torch.finfo(dtype)
    e = torch.floor(torch.log2(z.abs().clamp_min(f.smallest_normal)))
    return torch.exp2(e) * f.eps


# ----- rotary ----------------------------------------------------------------------
def rotary(x, angles, size=1.0, interleaved=False, back=False):
    """(B, T, H, D) turned by float64 angles (B, T, part / 2), and the bound: cos and sin rounded to fp32, two products
    and a sum, one rounding."""
    part = 2 * angles.shape[-1]
    first = torch.arange(part // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else part // 2)
    c, s = angles.cos().unsqueeze(2) * size, angles.sin().unsqueeze(2) * size * (-1 if back else 1)
    xd = x.double()
    a, b = xd[..., first], xd[..., second]
    out, tol = xd.clone(), torch.zeros_like(xd)
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    tol[..., first] = ((a * c).abs() + (b * s).abs()) * 4 * U32
    tol[..., second] = ((a * s).abs() + (b * c).abs()) * 4 * U32
    tol[..., first] += half_step(x.dtype) * out[..., first].abs() + tiny(x.dtype)
    tol[..., second] += half_step(x.dtype) * out[..., second].abs() + tiny(x.dtype)
    return out, tol
