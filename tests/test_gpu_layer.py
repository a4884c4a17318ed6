"""The norm and the rotary positions on the GPU against their plain float64 forms, within bounds derived from their
roundings (oracle/layer.py): widths around the kernels' chunks, lanes and groups, strides, types, values at the ends."""
import pytest
import torch

from monarch_muon_amd import rms_norm, rms_norm_fp8, rotary, rotary_table
from oracle import layer as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, F32 = torch.bfloat16, torch.float32


def within(got, ref, bound, what):
    got = got.detach().double()
    assert got.shape == ref.shape, what
    assert torch.equal(got.isnan(), ref.isnan()), what
    off = ((got - ref).abs() - bound)[~ref.isnan()]
    assert not off.numel() or float(off.max()) <= 0, (what, float(off.max()))


def randn(*shape, seed=0, dtype=BF, size=1.0):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(DEV).to(dtype)


# ----- norm ------------------------------------------------------------------------
def check_norm(x, w, r=None, eps=1e-6, grads=True):
    y, h, inv, tol = oracle.norm(x, w, r, eps)
    leaves = [t.detach().requires_grad_() for t in (x, w, *([] if r is None else [r]))]
    out = rms_norm(leaves[0], leaves[1], residual=None if r is None else leaves[2], eps=eps)
    if r is not None:
        out, hh = out
        assert torch.equal(hh.detach(), h)
    assert out.dtype == x.dtype
    within(out, y, tol, "y")
    if not grads:
        return
    dy = randn(*x.shape, seed=7, dtype=x.dtype)
    dh = None if r is None else randn(*x.shape, seed=8, dtype=x.dtype)
    dx, dw, (xt, wt) = oracle.norm_grad(h, w, dy, dh, eps)
    if r is None:
        gx, gw = torch.autograd.grad(out, leaves, dy)
    else:
        gx, gw, gr = torch.autograd.grad((out, hh), leaves, (dy, dh))
        assert torch.equal(gr, gx)
    assert gx.dtype == x.dtype and gw.dtype == w.dtype
    within(gx, dx, xt, "dx")
    within(gw, dw, wt, "dw")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows, width", [(1, 1), (1, 4096), (2, 7), (3, 8), (5, 9), (4, 127), (300, 128), (33, 129), (7, 255),
                                         (2, 513), (1000, 512), (19, 1000), (600, 1027), (257, 2736), (2100, 640),
                                         (9, 4095), (2500, 2048), (11, 8193), (3, 16384), (0, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, width, dtype, residual):
    x, w = randn(rows, width, dtype=dtype), 1 + randn(width, seed=1, dtype=dtype, size=0.3)
    check_norm(x, w, randn(rows, width, seed=2, dtype=dtype, size=3.0) if residual else None)


@pytest.mark.parametrize("width", [16385, 32767, 32768])
def test_norm_widest(width):
    check_norm(randn(5, width), randn(width, seed=1), randn(5, width, seed=2))


@pytest.mark.parametrize("rows", [1, 700, 40000])
def test_norm_float32_weight_of_bfloat16_rows(rows):
    check_norm(randn(rows, 264), randn(264, seed=1, dtype=F32), randn(rows, 264, seed=2))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_strides(dtype):
    """Rows of a wider tensor that begin at any element, a broadcast residual, gradients that are views."""
    wide = randn(40, 700, dtype=dtype)
    for first in (0, 1, 3, 8):
        check_norm(wide[:, first:first + 333], randn(333, seed=1, dtype=dtype), wide[:, 350:683])
        check_norm(wide[::3, first:first + 96], randn(96, seed=1, dtype=dtype), wide[:1, 5:101].expand(14, 96))
    check_norm(wide.t(), randn(40, seed=1, dtype=dtype))
    x, w = wide[:, :200].reshape(4, 10, 200).requires_grad_(), randn(400, seed=1, dtype=dtype)[::2].requires_grad_()
    y = rms_norm(x, w)
    assert y.shape == x.shape
    dy = randn(4, 10, 201, seed=3, dtype=dtype)[..., 1:]
    dx, dw, (xt, wt) = oracle.norm_grad(x.detach(), w.detach(), dy)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    within(gx, dx, xt, "dx")
    within(gw, dw, wt, "dw")


def test_norm_one_gradient_alone():
    """Only h is used, only y is, or only one input wants a gradient."""
    x, r, w = (t.requires_grad_() for t in (randn(30, 72), randn(30, 72, seed=1), randn(72, seed=2)))
    dy, dh = randn(30, 72, seed=3), randn(30, 72, seed=4)
    y, h = rms_norm(x, w, residual=r)
    gx, gw = torch.autograd.grad(h, (x, w), dh, retain_graph=True)
    assert torch.equal(gx, dh) and not gw.any()
    dx, dw, (xt, wt) = oracle.norm_grad(h.detach(), w.detach(), dy)
    for inputs, refs in (((x,), ((dx, xt),)), ((w,), ((dw, wt),)), ((r, w), ((dx, xt), (dw, wt)))):
        for got, (ref, tol) in zip(torch.autograd.grad(y, inputs, dy, retain_graph=True), refs):
            within(got, ref, tol, "one")


def test_norm_ends_of_the_numbers():
    """Zero rows, rows whose squares are below eps, rows with a NaN or an infinity beside others."""
    x = randn(6, 520, dtype=F32)
    x[1], x[2] = 0, x[2] * 1e-15
    x[3, 77], x[4, 5] = float("nan"), float("inf")
    w = randn(520, seed=1, dtype=F32)
    y = rms_norm(x, w)
    assert y[3].isnan().all() and y[4, 5].isnan() and not y[1].any()
    keep = [0, 1, 2, 5]
    ref, _, _, tol = oracle.norm(x[keep], w)
    within(y[keep], ref, tol, "rows beside")
    check_norm(x[keep], w, eps=0.1)


@pytest.mark.parametrize("rows, width", [(1, 1), (3, 130), (5, 64), (2, 1000), (400, 4096), (9000, 136), (7, 16384)])
def test_norm_gradients_against_differences(rows, width):
    """The directional derivative of a float32 loss, by differences of the float64 form."""
    x, w, dy = (randn(*s, seed=i, dtype=F32) for i, s in enumerate([(rows, width), (width,), (rows, width)]))
    leaves = x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(rms_norm(*leaves, eps=1e-3), leaves, dy)
    dx, dw = randn(rows, width, seed=5, dtype=F32), randn(width, seed=6, dtype=F32)
    def loss(t):
        y = oracle.norm(x.detach().double() + t * dx, w.detach().double() + t * dw, None, 1e-3)[0]
        return (y * dy).sum()
    e = 1e-5
    slope = float((loss(e) - loss(-e)) / (2 * e))
    got = float((gx.double() * dx).sum() + (gw.double() * dw).sum())
    size = float((gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum())
    assert abs(got - slope) <= 1e-5 * size + 1e-6


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("group", [128, None])
@pytest.mark.parametrize("rows, width", [(1, 4096), (1, 1), (3, 5), (4, 127), (5, 128), (70, 129), (33, 1001), (3000, 512),
                                         (600, 2736), (2, 16384), (0, 256)])
def test_norm_fp8(rows, width, group, fmt, dtype):
    x, w, r = randn(rows, width, dtype=dtype), randn(width, seed=1, dtype=dtype), randn(rows, width, seed=2, dtype=dtype)
    for res in (None, r):
        y, h, _, _ = oracle.norm(x, w, res)
        codes, scale, *hh = rms_norm_fp8(x, w, residual=res, dtype=fmt, group=group)
        assert codes.dtype == fmt and codes.shape == x.shape and scale.dtype == F32
        if res is not None:
            assert torch.equal(hh[0], h)
        ref = oracle.norm_scale(y, fmt, group)
        rel = (oracle._SUM / 2 + 8) * oracle.U32
        within(scale, ref, ref * rel, "scale")
        z = y / scale.double().repeat_interleave(group or width, -1)[:, :width]
        # half of a step, and what fp32 moves y by; the largest stands at the end of the codes
        within(codes.float(), z, oracle.code_step(z * (1 + 4 * rel), fmt) / 2 + z.abs() * 4 * rel, "codes")


def test_norm_fp8_ends_of_the_numbers():
    x = randn(5, 300, dtype=F32)
    x[1], x[2, :128] = 0, 0
    x[3, 4] = float("nan")
    codes, scale = rms_norm_fp8(x, torch.ones(300, device=DEV))
    assert not codes[1].float().any() and (scale[1] == 1).all() and scale[2, 0] == 1
    assert codes[3].float().isnan().all()
    ref = rms_norm(x, torch.ones(300, device=DEV))
    back = codes.float() * scale.repeat_interleave(128, 1)[:, :300]
    for row in (0, 2, 4):
        assert ((back[row] - ref[row]).abs() <= 2 ** -4 * ref[row].abs() + 2 ** -10 * scale[row].max()).all()


# ----- rotary ----------------------------------------------------------------------
def check_rotary(q, k, table, angles, positions=None, interleaved=False, size=1.0):
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    out = rotary(q, k, table, positions, interleaved=interleaved)
    grads = randn(*q.shape, seed=11, dtype=q.dtype), randn(*k.shape, seed=12, dtype=q.dtype)
    back = torch.autograd.grad(out, (q, k), grads)
    part = table.shape[1]
    for x, y, g, dx in zip((q, k), out, grads, back):
        assert y.dtype == x.dtype and y.is_contiguous()
        within(y, *oracle.rotary(x.detach(), angles, size, interleaved), "turned")
        within(dx, *oracle.rotary(g, angles, size, interleaved, back=True), "gradient")
        assert torch.equal(y[..., part:], x[..., part:]) and torch.equal(dx[..., part:], g[..., part:])


def angles_of(positions, part, base=10000.0):
    f = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / part)
    return positions.double().unsqueeze(-1) * f


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B, T, H, K, D, part", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 1, 128, 128), (1, 7, 3, 2, 64, 32), (3, 1, 32, 8, 128, 128), (1, 33, 5, 5, 80, 80),
    (2, 9, 2, 1, 96, 50), (1, 5, 1, 1, 37, 14), (1, 11, 6, 2, 256, 64), (2, 1000, 12, 12, 64, 64), (1, 300, 1, 3, 9, 6),
    (2, 2, 1, 1, 18, 18), (0, 4, 2, 2, 8, 8), (2, 0, 2, 2, 8, 8)])
def test_rotary(B, T, H, K, D, part, interleaved, dtype):
    table = rotary_table(part, 1024, device=DEV)
    q, k = randn(B, T, H, D, dtype=dtype), randn(B, T, K, D, seed=1, dtype=dtype)
    at = torch.arange(T, device=DEV).expand(B, T)
    check_rotary(q, k, table, angles_of(at, part), None, interleaved)
    at = torch.randint(0, 1024, (B, T), generator=torch.Generator().manual_seed(3)).to(DEV)
    check_rotary(q, k, table, angles_of(at, part), at.int(), interleaved)
    if B:
        check_rotary(q, k, table, angles_of(at[:1].expand(B, T), part), at[0], interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides(interleaved):
    """Heads of one fused projection, begun at odd elements, and heads before tokens."""
    B, T, H, K, D = 2, 50, 6, 2, 48
    fused = randn(B, T, 1 + (H + 2 * K) * D)
    q = fused[..., 1:1 + H * D].view(B, T, H, D)
    k = fused[..., 1 + H * D:1 + (H + K) * D].view(B, T, K, D)
    table, at = rotary_table(32, 64, device=DEV), torch.arange(T, device=DEV).expand(B, T)
    check_rotary(q, k, table, angles_of(at, 32), None, interleaved)
    check_rotary(randn(B, H, T, D).transpose(1, 2), randn(B, D, K, T, seed=4).permute(0, 3, 2, 1), table,
                 angles_of(at, 32), None, interleaved)
    check_rotary(randn(B, 1, H, D).expand(B, T, H, D), k, table, angles_of(at, 32), None, interleaved)


def test_rotary_far_positions():
    """A table of 2^20 positions: its angles, and those of its last ones, as 64 bits have them."""
    table = rotary_table(64, 1 << 20, base=500000.0, device=DEV)
    at = torch.tensor([[0, 1, (1 << 20) - 1, 777777]], device=DEV)
    check_rotary(randn(1, 4, 2, 64, dtype=F32), randn(1, 4, 1, 64, seed=1, dtype=F32), table, angles_of(at, 64, 500000.0), at)


def test_rotary_position_outside_the_table_is_nan():
    table = rotary_table(16, 10, device=DEV)
    q, k = randn(1, 4, 2, 24), randn(1, 4, 1, 24)
    out = rotary(q, k, table, torch.tensor([0, 10, -1, 9], device=DEV))
    for x, y in zip((q, k), out):
        assert y[0, 1:3, :, :16].isnan().all() and torch.equal(y[..., 16:], x[..., 16:])
        assert not y[0, ::3].isnan().any()
    assert rotary(randn(1, 12, 1, 16), randn(1, 12, 1, 16), table)[0][0, 10:].isnan().all()


def test_rotary_second_order():
    q, k = randn(1, 3, 2, 8, dtype=F32).requires_grad_(), randn(1, 3, 1, 8, dtype=F32).requires_grad_()
    table = rotary_table(8, 16, device=DEV)
    dout = randn(1, 3, 2, 8, seed=2, dtype=F32).requires_grad_()
    (dq,) = torch.autograd.grad(rotary(q, k, table)[0], q, dout, create_graph=True)
    up = randn(1, 3, 2, 8, seed=3, dtype=F32)
    (d,) = torch.autograd.grad(dq, dout, up)
    at = torch.arange(3, device=DEV)[None]
    within(d, *oracle.rotary(up, angles_of(at, 8)), "second")
