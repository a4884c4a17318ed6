"""The plain forms of the language-model ends against torch's own ops, and what the operators refuse (no GPU)."""
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

from monarch_muon_amd import _abi, embedding, linear_cross_entropy
from oracle import lm as oracle


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_is_torchs(reduction):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(7, 16, generator=g).double().requires_grad_(), torch.randn(11, 16, generator=g).double().requires_grad_()
    y = torch.tensor([3, -100, 0, 10, 10, -100, 5])
    ref = F.cross_entropy(x @ w.T, y, reduction=reduction)
    up = torch.randn(7, generator=g).double()
    dx, dw = torch.autograd.grad(ref, (x, w), up if reduction == "none" else None)
    loss, ox, ow, tol = oracle.cross_entropy(x.detach(), w.detach(), y, reduction=reduction,
                                             grad=up if reduction == "none" else None)
    for a, b in ((loss, ref.detach()), (ox, dx), (ow, dw)):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-13)


def test_cross_entropy_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(3, 8, generator=g).double(), torch.randn(5, 8, generator=g).double()
    y = torch.tensor([4, 0, -100])
    _, dx, dw, _ = oracle.cross_entropy(x, w, y)
    h = 1e-6
    for t, d in ((x, dx), (w, dw)):
        for i in range(0, t.numel(), 7):
            lo, hi = t.clone(), t.clone()
            lo.view(-1)[i] -= h
            hi.view(-1)[i] += h
            args = [(lo, w), (hi, w)] if t is x else [(x, lo), (x, hi)]
            a, b = (oracle.cross_entropy(*p, y)[0] for p in args)
            assert abs((b - a) / (2 * h) - d.view(-1)[i]) < 1e-8


def test_embedding_gradient_is_torchs():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(9, 5, generator=g).double().requires_grad_()
    i = torch.tensor([[1, 1, 8], [0, 4, 1]])
    up = torch.randn(2, 3, 5, generator=g).double()
    ref, = torch.autograd.grad(F.embedding(i, w, padding_idx=4) * 3.0, w, up)
    torch.testing.assert_close(oracle.embedding_grad(up, i, 9, 3.0, 4)[0], ref, rtol=1e-13, atol=1e-13)


# ----- refusals ----------------------------------------------------------------
def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


IDS = torch.zeros(4, dtype=torch.long)


@pytest.mark.parametrize("x, w, y, kw, error, match", [
    (bf(4, 16), bf(5, 16), IDS, {}, RuntimeError, "ROCm GPU"),
    (bf(4, 16), bf(5, 24), IDS, {}, ValueError, "expected x"),
    (bf(4, 12), bf(5, 12), IDS, {}, ValueError, "multiple of"),
    (bf(4, 16), bf(0, 16), IDS, {}, ValueError, "at least one token"),
    (bf(3, 16), bf(5, 16), IDS, {}, ValueError, "do not match"),
    (bf(4, 16), bf(5, 16), IDS.float(), {}, TypeError, "int64 or int32"),
    (bf(4, 16).float(), bf(5, 16), IDS, {}, TypeError, "computes in bfloat16; x is torch.float32"),
    (bf(4, 16), bf(5, 16).half(), IDS, {}, TypeError, "weight is torch.float16"),
    (bf(4, 16), bf(5, 16), IDS, {"reduction": "batch"}, ValueError, "reduction"),
    (bf(4, 16), bf(5, 16), IDS, {"piece_tokens": 0}, ValueError, "piece_tokens"),
])
def test_cross_entropy_refuses(x, w, y, kw, error, match):
    for grad in (False, True):
        with pytest.raises(error, match=match):
            linear_cross_entropy(x.clone().requires_grad_(grad), w, y, **kw)


@pytest.mark.parametrize("i, w, kw, error, match", [
    (IDS, bf(5, 16), {}, RuntimeError, "ROCm GPU"),
    (IDS, bf(5), {}, ValueError, "expected weight"),
    (IDS, bf(5, 16).half(), {}, TypeError, "float32"),
    (IDS.float(), bf(5, 16), {}, TypeError, "int64 or int32"),
    (IDS, bf(5, 16), {"padding_idx": 5}, ValueError, "padding_idx"),
    (IDS, bf(5, 16), {"padding_idx": -6}, ValueError, "padding_idx"),
])
def test_embedding_refuses(i, w, kw, error, match):
    for grad in (False, True):
        with pytest.raises(error, match=match):
            embedding(i, w.clone().requires_grad_(grad), **kw)


def test_shapes_on_meta_tensors():
    x, w = bf(2, 3, 16).to("meta").requires_grad_(), bf(5, 16).to("meta").requires_grad_()
    y = torch.zeros(2, 3, dtype=torch.long, device="meta")
    for reduction, shape in (("mean", ()), ("sum", ()), ("none", (2, 3))):
        loss = linear_cross_entropy(x, w, y, reduction=reduction)
        assert loss.shape == shape and loss.dtype == torch.float32
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert dx.shape == x.shape and dw.shape == w.shape
    out = embedding(y, w, scale=2.0)
    assert out.shape == (2, 3, 16) and torch.autograd.grad(out.sum(), w)[0].shape == w.shape


def test_entry_points_validate_before_launching():
    """Every descriptor here is invalid, so no kernel is launched."""
    lib = _abi.lib()
    good = dict(tokens=4, vocab=100, width=64, dtype=_abi.BF16, reduction=_abi.CE_MEAN, x_stride=64, w_stride=64,
                piece_tokens=4, x=4096, w=8192, target=12288, loss=16384, dx=20480, dw=24576, workspace=32768,
                workspace_bytes=0)
    need = lib.mmuon_ce_workspace(C.byref(_abi.CeArgs(**good)), 1)
    assert need > lib.mmuon_ce_workspace(C.byref(_abi.CeArgs(**good)), 0) > 0
    good["workspace_bytes"] = need - 1
    assert lib.mmuon_ce_fwd(None, None) == lib.mmuon_ce_fwd_bwd(None, None) == -1
    for change, code, message in [({}, -1, b"workspace of"), ({"dtype": _abi.F32}, -1, b"MMUON_BF16"),
                                  ({"tokens": 1 << 24}, -3, b"2^24"), ({"vocab": 1 << 22}, -3, b"2^22"),
                                  ({"vocab": 0}, -3, b"vocab"), ({"width": 60}, -1, b"multiple of 8"),
                                  ({"x_stride": 60}, -1, b"strides"), ({"w_stride": 1 << 22}, -3, b"32-bit"),
                                  ({"x": 4104}, -1, b"unaligned"), ({"w": None}, -1, b"null"),
                                  ({"target": None}, -1, b"target"), ({"loss": None}, -1, b"nowhere"),
                                  ({"reduction": 3}, -1, b"reduction"), ({"piece_tokens": 0}, -1, b"piece_tokens"),
                                  ({"dw": 24584}, -1, b"unaligned dx or dw"), ({"workspace": 32770}, -1, b"256-B")]:
        assert lib.mmuon_ce_fwd_bwd(C.byref(_abi.CeArgs(**{**good, **change})), None) == code, change
        assert message in lib.mmuon_last_error(), (change, lib.mmuon_last_error())
    assert lib.mmuon_scale_bf16(4096, 12, None, 0, 8192, None) == lib.mmuon_scale_bf16(4100, 16, None, 0, 8192, None) == -1
    assert lib.mmuon_scale_bf16(4096, 16, None, 8, 8192, None) == -1
    emb = dict(tokens=4, vocab=100, width=7, dtype=_abi.F32, scale=1.0, padding_idx=-1, w_stride=7, dout_stride=7,
               index=4096, w=8192, out=12288, dout=16384, dw=20480, workspace=32768, workspace_bytes=0)
    for change, code, message in [({}, -1, b"workspace of"), ({"dtype": _abi.F8E4M3}, -1, b"dtype"),
                                  ({"tokens": 1 << 26}, -3, b"2^26"), ({"vocab": 0}, -3, b"vocab"),
                                  ({"width": 0}, -1, b"width"), ({"dout": 16386}, -1, b"unaligned"),
                                  ({"index": None}, -1, b"index"), ({"dout_stride": -7}, -1, b"stride")]:
        assert lib.mmuon_embedding_bwd(C.byref(_abi.EmbeddingArgs(**{**emb, **change})), None) == code, change
        assert message in lib.mmuon_last_error(), change
    assert lib.mmuon_embedding_fwd(C.byref(_abi.EmbeddingArgs(**{**emb, "out": None})), None) == -1
    assert lib.mmuon_embedding_fwd(None, None) == lib.mmuon_embedding_bwd(None, None) == -1


def test_struct_layouts_match_header(tmp_path):
    import subprocess
    from pathlib import Path
    header = Path(_abi.__file__).resolve().parent.parent / "include" / "mmuon.h"
    structs = {"mmuon_ce_args": _abi.CeArgs, "mmuon_embedding_args": _abi.EmbeddingArgs}
    body = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in p._fields_)
                   for c, p in structs.items())
    (tmp_path / "l.c").write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void){{{body}return 0;}}')
    subprocess.run(["gcc", "-std=c11", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [n for p in structs.values() for n in [C.sizeof(p)] + [getattr(p, f).offset for f, _ in p._fields_]]
