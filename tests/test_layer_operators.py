"""The operators between a layer's projections without a GPU: refusals, derivatives on meta tensors, tracing, the rotary
table's formulas, and the C entry points' checks."""
import ctypes as C
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

from monarch_muon_amd import _abi, differential_attention, rms_norm, rms_norm_fp8, rotary, rotary_table

HEADER = Path(__file__).resolve().parent.parent / "include" / "mmuon.h"


def meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="meta")


F32 = torch.float32


def heads(B=2, T=3, S=5, H=4, K=2, d=16):
    return meta(B, T, 2 * H, d), meta(B, S, 2 * K, d), meta(B, S, K, 2 * d), meta(H, dtype=F32)


# ----- refusals ----------------------------------------------------------------------
q, k, v, lam = heads()
CASES = {
    "x of another type": (lambda: rms_norm(meta(3, 8, dtype=torch.float16), meta(8)), TypeError, "bfloat16 or float32"),
    "weight narrower than x": (lambda: rms_norm(meta(3, 8, dtype=F32), meta(8)), TypeError, "weight must be"),
    "weight of another width": (lambda: rms_norm(meta(3, 8), meta(9)), ValueError, "expected x"),
    "x of no columns": (lambda: rms_norm(meta(3, 0), meta(0)), ValueError, "expected x"),
    "x of no dimension": (lambda: rms_norm(meta(), meta(1)), ValueError, "expected x"),
    "residual of another shape": (lambda: rms_norm(meta(3, 8), meta(8), residual=meta(8)), ValueError, "not of x's shape"),
    "residual of another type": (lambda: rms_norm(meta(3, 8), meta(8), residual=meta(3, 8, dtype=F32)), TypeError, "residual"),
    "negative eps": (lambda: rms_norm(meta(3, 8), meta(8), eps=-1e-6), ValueError, "eps"),
    "eps that is no number": (lambda: rms_norm(meta(3, 8), meta(8), eps=math.nan), ValueError, "eps"),
    "too wide": (lambda: rms_norm(meta(1, 32769), meta(32769)), ValueError, "beyond 32768"),
    "too wide in float32": (lambda: rms_norm(meta(1, 16385, dtype=F32), meta(16385, dtype=F32)), ValueError, "beyond 16384"),
    "codes of another type": (lambda: rms_norm_fp8(meta(3, 8), meta(8), dtype=torch.int8), TypeError, "float8"),
    "another group": (lambda: rms_norm_fp8(meta(3, 8), meta(8), group=64), ValueError, "group"),
    "codes with a gradient": (lambda: rms_norm_fp8(meta(3, 8).requires_grad_(), meta(8)), RuntimeError, "no gradient"),
    "q and k of two types": (lambda: rotary(q, k.float(), meta(9, 16, dtype=F32)), TypeError, "one type"),
    "q and k of two lengths": (lambda: rotary(q, k, meta(9, 16, dtype=F32)), ValueError, "expected q"),
    "a bfloat16 table": (lambda: rotary(q, q, meta(9, 16)), TypeError, "table must be float32"),
    "a table of an odd width": (lambda: rotary(q, q, meta(9, 15, dtype=F32)), ValueError, "even number"),
    "a table wider than heads": (lambda: rotary(q, q, meta(9, 18, dtype=F32)), ValueError, "even number"),
    "a table of no positions": (lambda: rotary(q, q, meta(0, 16, dtype=F32)), ValueError, "no positions"),
    "positions of another shape": (lambda: rotary(q, q, meta(9, 16, dtype=F32), meta(2, dtype=torch.long)), ValueError, "positions"),
    "positions of another type": (lambda: rotary(q, q, meta(9, 16, dtype=F32), meta(3, dtype=F32)), TypeError, "positions"),
    "a table with a gradient": (lambda: rotary(q, q, meta(9, 16, dtype=F32).requires_grad_()), RuntimeError, "no gradient"),
    "attention in float32": (lambda: differential_attention(q.float(), k, v, lam), TypeError, "computes in bfloat16; q"),
    "values in float32": (lambda: differential_attention(q, k, v.float(), lam), TypeError, "computes in bfloat16; v"),
    "heads of 12 columns": (lambda: differential_attention(*heads(d=12)), ValueError, "multiple of 8"),
    "heads of 136 columns": (lambda: differential_attention(*heads(d=136)), ValueError, "at most 128"),
    "heads that do not share evenly": (lambda: differential_attention(*heads(H=3, K=2)), ValueError, "multiple of K"),
    "values of half the width": (lambda: differential_attention(q, k, v[..., :16], lam), ValueError, "expected q"),
    "q of three dimensions": (lambda: differential_attention(q[0], k, v, lam), ValueError, "expected q"),
    "keys and values of two lengths": (lambda: differential_attention(q, k, v[:, :4], lam), ValueError, "expected q"),
    "lam of another number": (lambda: differential_attention(q, k, v, meta(3, dtype=F32)), ValueError, "lam"),
    "lengths of another number": (lambda: differential_attention(q, k, v, lam, lengths=meta(3, dtype=torch.long)), ValueError, "lengths"),
    "starts of another type": (lambda: differential_attention(q, k, v, lam, starts=meta(2, dtype=F32)), TypeError, "starts"),
    "scale of zero": (lambda: differential_attention(q, k, v, lam, scale=0.0), ValueError, "scale"),
    "scale that is no number": (lambda: differential_attention(q, k, v, lam, scale=math.nan), ValueError, "scale"),
}


@pytest.mark.parametrize("case", CASES)
def test_refused(case):
    """The operators' own checks, before any kernel: tensors on the CPU stand for those on a GPU."""
    call, error, match = CASES[case]
    with pytest.raises(error, match=match):
        on_cpu(call)


def on_cpu(call):
    """``call`` with its meta tensors made on the CPU (fakes take any shapes; the operators themselves do not)."""
    names = {n: globals()[n] for n in ("meta", "q", "k", "v", "lam")}
    globals()["meta"] = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype)
    globals().update(zip(("q", "k", "v", "lam"), heads()))
    try:
        return call()
    finally:
        globals().update(names)


def test_cpu_tensors_are_refused():
    for call in (lambda: rms_norm(meta(3, 8), meta(8)), lambda: rms_norm_fp8(meta(3, 8), meta(8)),
                 lambda: rotary(meta(1, 2, 2, 8), meta(1, 2, 2, 8), meta(9, 8, dtype=F32)),
                 lambda: differential_attention(q, k, v, lam)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            on_cpu(call)


# ----- derivatives -------------------------------------------------------------------
def test_shapes_and_types_of_gradients():
    x, r, w = meta(2, 6, 16).requires_grad_(), meta(2, 6, 16).requires_grad_(), meta(16, dtype=F32).requires_grad_()
    y, h = rms_norm(x, w, residual=r)
    for g, t in zip(torch.autograd.grad(y.float().sum() + h.float().sum(), (x, r, w)), (x, r, w)):
        assert g.shape == t.shape and g.dtype == t.dtype
    q, k, v, lam = (t.requires_grad_() for t in heads())
    o = differential_attention(q, k, v, lam)
    assert o.shape == (2, 3, 4, 32) and o.dtype == torch.bfloat16
    for g, t in zip(torch.autograd.grad(o.float().sum(), (q, k, v, lam)), (q, k, v, lam)):
        assert g.shape == t.shape and g.dtype == t.dtype
    one = meta(dtype=torch.bfloat16).requires_grad_()
    assert torch.autograd.grad(differential_attention(q, k, v, one).float().sum(), one)[0].shape == ()


@pytest.mark.parametrize("which", ["norm", "attention"])
def test_second_derivatives_are_refused(which):
    if which == "norm":
        x = meta(6, 16).requires_grad_()
        out = rms_norm(x, meta(16).requires_grad_())
    else:
        q, k, v, lam = heads()
        x = q.requires_grad_()
        out = differential_attention(q, k, v, lam)
    (g,) = torch.autograd.grad(out.float().sum(), x, create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula"):
        torch.autograd.grad(g.float().square().sum() + x.float().sum(), x)


def test_rotary_is_differentiable_to_any_order():
    q, k, table = meta(1, 3, 2, 8).requires_grad_(), meta(1, 3, 2, 8), meta(9, 8, dtype=F32)
    up = meta(1, 3, 2, 8).requires_grad_()
    (g,) = torch.autograd.grad(rotary(q, k, table)[0], q, up, create_graph=True)
    (d,) = torch.autograd.grad(g, up, meta(1, 3, 2, 8), create_graph=True)
    assert d.shape == up.shape


@pytest.mark.parametrize("call", [
    lambda t: rms_norm(t, meta(16)), lambda t: rms_norm(meta(5, 16), meta(16), residual=t),
    lambda t: rms_norm_fp8(t, meta(16))[1], lambda t: rotary(t.view(1, 5, 1, 16), meta(1, 5, 1, 16), meta(9, 8, dtype=F32))[0],
    lambda t: differential_attention(t.view(1, 5, 2, 8), meta(1, 5, 2, 8), meta(1, 5, 1, 16), meta(1, dtype=F32))])
def test_forward_mode_is_refused(call):
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (meta(5, 16),), (meta(5, 16),))


@pytest.mark.parametrize("dynamic", [False, True])
def test_traced(dynamic):
    """torch.compile's tracing of a layer's part, forward and backward, on meta tensors."""
    torch._dynamo.reset()

    def part(x, r, w, table, lam):
        y, h = rms_norm(x, w, residual=r)
        q, k = rotary(y.view(2, -1, 4, 16), y.view(2, -1, 4, 16), table)
        o = differential_attention(q, k, y.view(2, -1, 2, 32), lam)
        return (o.flatten(2) + h).float().square().sum()
    step = torch.compile(part, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T in (6, 7):
        x, r, w, lam = (t.requires_grad_() for t in (meta(2, T, 64), meta(2, T, 64), meta(64), meta(2, dtype=F32)))
        loss = step(x, r, w, meta(9, 16, dtype=F32), lam)
        for g, t in zip(torch.autograd.grad(loss, (x, r, w, lam)), (x, r, w, lam)):
            assert g.shape == t.shape
    torch._dynamo.reset()


# ----- the rotary table --------------------------------------------------------------
def by_hand(dim, p, base=10000.0, scaling=None, factor=1.0, trained=None):
    """The angles of position p, pair by pair."""
    out = []
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "ntk":
            f = (base * factor ** (dim / (dim - 2))) ** (-2 * i / dim)
        elif scaling == "yarn":
            lo, hi = (dim * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32, 1))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim - 1)
            ramp = min(max((i - lo) / (hi - lo), 0), 1)
            f = f * (1 - ramp) + f / factor * ramp
        elif scaling == "llama":
            turns = trained * f / (2 * math.pi)
            keep = min(max((turns - 1) / (4 - 1), 0), 1)
            f = f * keep + f / factor * (1 - keep)
        out.append(p * f)
    return out


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn", "llama"])
def test_rotary_table(scaling):
    dim, length, kw = 64, 4096, dict(scaling=scaling, factor=8.0, trained=512) if scaling else {}
    table = rotary_table(dim, length, **kw)
    assert table.shape == (length, dim) and table.dtype == F32
    size = 0.1 * math.log(8.0) + 1 if scaling == "yarn" else 1.0
    for p in (0, 1, 77, 4095):
        a = by_hand(dim, p, **kw)
        # cosines of angles up to 4095 in 64 bits, rounded once: half a step of float32, and 2^-52 of the angle
        ref = torch.tensor([size * math.cos(t) for t in a] + [size * math.sin(t) for t in a], dtype=torch.float64)
        assert float((table[p].double() - ref).abs().max()) <= 2 ** -24 * size + 4 * 4096 * 2 ** -52


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(length=-1), dict(scaling="other"), dict(factor=0.0),
                                dict(base=-1.0), dict(scaling="yarn", factor=2.0), dict(scaling="llama", factor=2.0)])
def test_rotary_table_refusals(kw):
    with pytest.raises(ValueError):
        rotary_table(**{"dim": 8, "length": 4, **kw})


# ----- C ABI -------------------------------------------------------------------------
def test_struct_layouts_match_the_header(tmp_path):
    structs = {"mmuon_norm_args": _abi.NormArgs, "mmuon_rotary_args": _abi.RotaryArgs, "mmuon_attention_args": _abi.AttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for name, py in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0].rstrip("_")}));' for f in py._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split("\n") if x)
    for name, py in structs.items():
        assert int(got[name]) == C.sizeof(py), name
        for f in py._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(py, f[0]).offset, f[0]
        body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name, HEADER.read_text(), re.S).group(1)
        assert len(re.findall(r";", re.sub(r"/\*.*?\*/", "", body, flags=re.S))) <= len(py._fields_)


def refusal(fn, args, *more):
    lib = _abi.lib()
    rc = getattr(lib, fn)(C.byref(args) if args is not None else None, *more, None)
    return rc, lib.mmuon_last_error().decode()


NORM = dict(rows=4, width=64, dtype=_abi.BF16, w_dtype=_abi.BF16, out_dtype=_abi.BF16, eps=1e-6, x_stride=64, dy_stride=64,
            x=4096, w=8192, y=12288, inv=16384, dy=20480, dx=24576, dw=28672, workspace=32768, workspace_bytes=1 << 40)
ROTARY = dict(batch=1, tokens=4, q_heads=2, k_heads=1, dim=64, part=64, dtype=_abi.BF16, table_rows=9, q=4096, k=8192,
              table=12288, q_out=16384, k_out=20480)
ATTENTION = dict(batch=1, queries=4, keys=4, heads=2, kv_heads=1, dim=64, dtype=_abi.BF16, scale=1.0, q=4096, k=8192, v=12288,
                 lam=16384, o=20480, o1=24576, o2=28672, lse=32768, dout=36864, dq=40960, dk=45056, dv=49152, dlam=53248,
                 workspace=65536, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change, code, match", [
    (dict(dtype=_abi.F8E4M3), -1, "dtype"), (dict(w_dtype=_abi.F8E4M3), -1, "w_dtype"), (dict(width=0), -3, "width"),
    (dict(width=32769), -3, "width"), (dict(rows=1 << 31), -3, "rows"), (dict(rows=-1), -3, "rows"), (dict(eps=-1.0), -1, "eps"),
    (dict(x=0), -1, "x"), (dict(x=4097), -1, "x"), (dict(w=0), -1, "w"), (dict(x_stride=-1), -1, "stride")])
def test_norm_entry_points_validate_before_launching(change, code, match):
    for fn in ("mmuon_norm_fwd", "mmuon_norm_bwd"):
        rc, why = refusal(fn, _abi.NormArgs(**{**NORM, **change}))
        assert rc == code and match in why
        assert refusal(fn, None)[0] == -1


@pytest.mark.parametrize("fn, change, match", [
    ("mmuon_norm_fwd", dict(y=0), "y"), ("mmuon_norm_fwd", dict(out_dtype=_abi.F32), "out_dtype"),
    ("mmuon_norm_fwd", dict(out_dtype=_abi.F8E4M3, group=64, scale=4096), "group"), ("mmuon_norm_fwd", dict(out_dtype=_abi.F8E5M2), "scale"),
    ("mmuon_norm_bwd", dict(inv=0), "inv"), ("mmuon_norm_bwd", dict(dy=0), "dy"), ("mmuon_norm_bwd", dict(workspace=32769), "workspace"),
    ("mmuon_norm_bwd", dict(workspace_bytes=8), "needed")])
def test_norm_directions_validate(fn, change, match):
    rc, why = refusal(fn, _abi.NormArgs(**{**NORM, **change}))
    assert rc == -1 and match in why


@pytest.mark.parametrize("change, code, match", [
    (dict(dtype=9), -1, "dtype"), (dict(part=63), -1, "part"), (dict(part=66), -1, "part"), (dict(dim=0), -1, "dim"),
    (dict(table_rows=0), -1, "table"), (dict(table=0), -1, "table"), (dict(q=0), -1, "queries"), (dict(k_out=0), -1, "keys"),
    (dict(tokens=1 << 40), -3, "too many"), (dict(batch=1 << 40), -3, "too many"), (dict(positions=12289), -1, "positions")])
def test_rotary_entry_point_validates(change, code, match):
    rc, why = refusal("mmuon_rotary", _abi.RotaryArgs(**{**ROTARY, **change}), 0)
    assert rc == code and match in why


@pytest.mark.parametrize("change, code, match", [
    (dict(dtype=_abi.F32), -1, "MMUON_BF16"), (dict(dim=12), -1, "dim"), (dict(dim=136), -1, "dim"), (dict(heads=3, kv_heads=2), -1, "heads"),
    (dict(kv_heads=0), -1, "heads"), (dict(batch=-1), -3, "negative"), (dict(batch=1 << 20, queries=1 << 20), -3, "too many"),
    (dict(scale=0.0), -1, "scale"), (dict(lam_stride=2), -1, "lam_stride"), (dict(q=4098), -1, "q, k or v"), (dict(lam=0), -1, "lam"),
    (dict(q_stride=(C.c_int64 * 3)(4, 0, 0)), -1, "strides"), (dict(k_stride=(C.c_int64 * 3)(0, 1 << 22, 0)), -3, "tile offsets"),
    (dict(lengths=4097), -1, "lengths"), (dict(o2=0), -1, "o1, o2"), (dict(workspace=1), 0, "")])
def test_attention_entry_points_validate(change, code, match):
    for fn in ("mmuon_attention_fwd", "mmuon_attention_bwd"):
        if code == 0:   # the forward of so few keys needs none
            if fn == "mmuon_attention_fwd":
                continue
            code, match = -1, "workspace"
        rc, why = refusal(fn, _abi.AttentionArgs(**{**ATTENTION, **change}))
        assert rc == code and match in why, why


@pytest.mark.parametrize("change, forward", [
    (dict(heads=1 << 22, kv_heads=1), True), (dict(batch=1 << 22), True), (dict(batch=1 << 18, queries=1 << 12), True),
    (dict(batch=1 << 16, queries=1 << 12), False), (dict(batch=1 << 16, keys=1 << 15), True), (dict(batch=1 << 16, keys=1 << 14), False),
    (dict(heads=1 << 14, kv_heads=1, dim=128, queries=2), False)])
def test_attention_entry_points_refuse_what_a_launch_cannot_hold(change, forward):
    sizes = {**ATTENTION, "heads": 1, "kv_heads": 1, "batch": 1, "queries": 1, "keys": 1, **change}
    for fn in ("mmuon_attention_fwd",) * forward + ("mmuon_attention_bwd",):
        rc, why = refusal(fn, _abi.AttentionArgs(**sizes))
        assert rc == -3 and ("too many" in why or "tile offsets" in why), why


def test_workspaces_of_sizes_at_the_ends():
    """No size makes the plans divide by zero, and none that is refused has a workspace."""
    lib = _abi.lib()
    for B in (0, 1, 3):
        for Tq in (0, 1, 1000):
            for Tk in (0, 1, 70000):
                for H, K in ((0, 1), (1, 1), (12, 3)):
                    for d in (8, 64, 128):
                        a = _abi.AttentionArgs(**{**ATTENTION, "batch": B, "queries": Tq, "keys": Tk, "heads": H, "kv_heads": K, "dim": d})
                        for bwd in (0, 1):
                            assert lib.mmuon_attention_workspace(C.byref(a), bwd) < 1 << 36
    assert lib.mmuon_attention_workspace(C.byref(_abi.AttentionArgs(**{**ATTENTION, "dim": 7})), 1) == 0
    assert lib.mmuon_norm_workspace(C.byref(_abi.NormArgs(**{**NORM, "rows": 0}))) == 0
    assert lib.mmuon_norm_workspace(None) == lib.mmuon_attention_workspace(None, 0) == 0
