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


# ----- differential attention ------------------------------------------------------
UBF = 2.0 ** -8


def visible(Tq, Tk, causal, length=None, start=None):
    """(queries, keys): which keys each query sees."""
    n = Tk if length is None else min(max(int(length), 0), Tk)
    j, t = torch.arange(Tk), torch.arange(Tq)
    see = (j < n).expand(Tq, Tk)
    if causal:
        see = see & (j <= (n - Tq if start is None else int(start)) + t[:, None])
    return see


def attention(q, k, v, lam, causal=True, scale=None, lengths=None, starts=None, dout=None):
    """((o, dq, dk, dv, dlam), bounds), float64; the gradients where ``dout`` is given.

    Roundings: scores, their statistics and all sums in fp32; P, dS and P_1 - lam P_2 to bf16 before their products; results
    once.  o_m, of which D_m = dO . o_m is made, has weights w = P (1 + e) / sum of P (1 + e) with |e| up to 2^-8 and stays in
    fp32: o_m is off by sum of P e (v - o_m), D_m by sum of P e (dP - D_m)."""
    B, Tq, H2, d = q.shape
    H, Tk, K = H2 // 2, k.shape[1], v.shape[2]
    scale = d ** -0.5 if scale is None else scale
    f = torch.float64
    dev = q.device
    q, k, v, lam = q.double(), k.double(), v.double(), lam.double().to(dev).expand(H)
    zero = lambda *s: torch.zeros(s, dtype=f, device=dev)  # noqa: E731
    o, ot = zero(B, Tq, H, 2 * d), zero(B, Tq, H, 2 * d)
    dq, dk, dv, dl = zero(*q.shape), zero(*k.shape), zero(*v.shape), zero(H)
    qt, kt, vt, lt = zero(*q.shape), zero(*k.shape), zero(*v.shape), zero(H)
    for b in range(B):
        see = visible(Tq, Tk, causal, None if lengths is None else lengths[b], None if starts is None else starts[b]).to(dev)
        kept = see.any(0)
        for h in range(H):
            g, L = h // (H // K), lam[h]
            V = torch.where(kept[:, None], v[b, :, g], 0.0)
            P, err, O, Ot = [], [], [], []
            for m in (0, 1):
                Q, Km = q[b, :, 2 * h + m], torch.where(kept[:, None], k[b, :, 2 * g + m], 0.0)
                s = (Q @ Km.T * scale).masked_fill(~see, -float("inf"))
                p = torch.softmax(s, 1).nan_to_num(0.0)
                size = (Q.abs() @ Km.abs().T * scale).masked_fill(~see, 0.0)
                top = size.amax(1, keepdim=True) if Tk else zero(Tq, 1)
                # a probability's relative error: its score's, the reference's and the sum's; exp2 is good to 2^-22
                e = U32 * (2 * (d + 6) * (size + top) + Tk + 40)
                P.append(p)
                err.append(e)
                O.append(p @ V)
                Ot.append(((1.01 * UBF + e + 2 * Tk * U32) * p) @ V.abs() + 1.01 * UBF * O[m].abs())
            o[b, :, h] = O[0] - L * O[1]
            ot[b, :, h] = Ot[0] + L.abs() * Ot[1] + half_step(torch.bfloat16) * o[b, :, h].abs() + 1e-37
            if dout is None:
                continue
            G = dout[b, :, h].double()
            both = P[0] - L * P[1]
            dv[b, :, g] += both.T @ G
            off = P[0] * err[0] + L.abs() * P[1] * err[1]
            vt[b, :, g] += (off + UBF * both.abs() + 2 * H * Tq * U32 * (P[0] + L.abs() * P[1])).T @ G.abs()
            dp = G @ V.T
            dpt = 2 * (2 * d + 2) * U32 * (G.abs() @ V.abs().T)
            for m, sign in ((0, 1.0), (1, -L)):
                D = (P[m] * dp).sum(1, keepdim=True)
                Dt = (P[m] * (dp - D).abs() * (1.01 * UBF + err[m])).sum(1, keepdim=True) + \
                    (2 * Tk + 4 * d) * U32 * (P[m] * (G.abs() @ V.abs().T)).sum(1, keepdim=True)
                ds = P[m] * (dp - D)
                dst = P[m] * (dpt + Dt + 4 * U32 * (dp.abs() + D.abs())) + ds.abs() * (err[m] + UBF)
                ds, dst = ds * sign * scale, dst * abs(sign) * scale
                Q, Km = q[b, :, 2 * h + m], torch.where(kept[:, None], k[b, :, 2 * g + m], 0.0)
                dq[b, :, 2 * h + m] = ds @ Km
                qt[b, :, 2 * h + m] = (dst + 2 * Tk * U32 * ds.abs()) @ Km.abs()
                dk[b, :, 2 * g + m] += ds.T @ Q
                kt[b, :, 2 * g + m] += (dst + 2 * H * Tq * U32 * ds.abs()).T @ Q.abs()
                if m:
                    dl[h] -= D.sum()
                    lt[h] += (P[1] * (dpt + dp.abs() * (err[1] + (Tk + B * Tq) * U32))).sum()
    r = half_step(torch.bfloat16)
    bounds = [ot, qt + r * dq.abs() + 1e-37, kt + r * dk.abs() + 1e-37, vt + r * dv.abs() + 1e-37, lt + U32 * dl.abs() + 1e-37]
    return (o, dq, dk, dv, dl), bounds
