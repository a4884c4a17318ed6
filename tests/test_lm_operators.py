"""The language-model operators under torch's autograd, without a GPU: second derivatives on meta tensors."""
import warnings

import pytest
import torch

from monarch_muon_amd import butterfly_blk, embedding, linear_cross_entropy


def meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="meta")


def head(reduction):
    x, w = meta(6, 16).requires_grad_(), meta(5, 16).requires_grad_()
    return x, w, linear_cross_entropy(x, w, meta(6, dtype=torch.long), reduction=reduction)


# ----- second derivatives ----------------------------------------------------------
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("wrt", ["x", "w", "both", "factor"])
def test_second_derivative_of_the_loss_is_refused(reduction, wrt):
    """A gradient taken with create_graph knows that it depends on x, weight and the incoming gradient: a derivative of
    it raises, also where it is one term beside others that have a derivative of their own."""
    x, w, loss = head(reduction)
    factor = meta(dtype=torch.float32).requires_grad_()
    inputs = {"x": (x,), "w": (w,), "both": (x, w), "factor": (x,)}[wrt]
    grads = torch.autograd.grad((loss * factor if wrt == "factor" else loss).sum(), inputs, create_graph=True)
    assert all(g.requires_grad for g in grads)
    for g in grads:
        penalty = g.float().square().sum()
        for target in (x, w, *((factor,) if wrt == "factor" else ())):
            other = target.float().sum()
            with pytest.raises(RuntimeError, match="no autograd formula"):
                torch.autograd.grad(penalty + other, target, retain_graph=True, allow_unused=True)


def test_second_derivative_is_refused_by_backward():
    x, w, loss = head("mean")
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        (g.float().sum() + w.float().sum()).backward()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_first_derivatives_carry_no_graph(reduction):
    """Without create_graph the gradients are plain tensors, and nothing warns."""
    x, w, loss = head(reduction)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        grads = torch.autograd.grad(loss.sum(), (x, w))
    assert not any(g.requires_grad for g in grads)


def test_gradient_operator_has_no_derivative():
    """The gradient's own operator, called with tensors that require one."""
    x, w, _ = head("none")
    loss, dx, dw = torch.ops.mmuon.linear_cross_entropy_grad(x, w, meta(6, dtype=torch.long), None, -100, 1, 6, True, True)
    for out in (loss, dx, dw):
        with pytest.raises(RuntimeError, match="no autograd formula"):
            torch.autograd.grad(out.float().sum(), x, retain_graph=True)


@pytest.mark.parametrize("order", [2, 3])
def test_embedding_gradient_is_differentiable(order):
    """The table's gradient is linear in the gradient that arrives: its derivative by that is a lookup, and that of the
    lookup the table's gradient again."""
    w = meta(9, 16).requires_grad_()
    dout = meta(2, 3, 16).requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        out = embedding(meta(2, 3, dtype=torch.long), w, scale=3.0, padding_idx=4)
        (dw,) = torch.autograd.grad(out, w, dout, create_graph=True)
        assert dw.requires_grad
        up = meta(9, 16).requires_grad_()
        (d,) = torch.autograd.grad(dw, dout, up, create_graph=True)
        assert d.shape == dout.shape and d.dtype == dout.dtype
        if order == 3:
            (u,) = torch.autograd.grad(d, up, meta(2, 3, 16))
            assert u.shape == up.shape


# ----- first calls -------------------------------------------------------------------
def test_first_calls_of_many_threads():
    """A fresh process whose first calls come from many threads at once: each binds or finds the library bound."""
    import subprocess
    import sys
    from pathlib import Path
    program = """
import threading
from monarch_muon_amd import butterfly
start, results = threading.Barrier(16), []
def call():
    start.wait()
    results.append(butterfly._bind())
threads = [threading.Thread(target=call) for _ in range(16)]
for t in threads: t.start()
for t in threads: t.join()
assert results == [0] * 16, results
"""
    r = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


# ----- forward mode ------------------------------------------------------------------
@pytest.mark.parametrize("call", [
    lambda t: linear_cross_entropy(t, meta(5, 16), meta(5, dtype=torch.long)),
    lambda t: linear_cross_entropy(meta(5, 16), t, meta(5, dtype=torch.long), reduction="none"),
    lambda t: embedding(meta(5, dtype=torch.long), t),
    lambda t: torch.ops.mmuon.embedding_grad(t, meta(5, dtype=torch.long), 9, 1.0, -1),
    lambda t: torch.ops.mmuon.linear_cross_entropy_grad(t, meta(5, 16), meta(5, dtype=torch.long), None, -100, 1, 5,
                                                        True, True)[1],
    lambda t: butterfly_blk(t, meta(2, 8, 8), meta(2, 8, 8)),
], ids=["loss by x", "loss by weight", "embedding", "embedding_grad", "loss_grad", "layer"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(call, requires_grad):
    """A tangent that goes in raises; it is not dropped (torch.func.jvp would take that for zero)."""
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (meta(5, 16),), (meta(5, 16),))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(meta(5, 16).requires_grad_(requires_grad), meta(5, 16))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)


def test_transforms_are_refused():
    """torch.func's reverse mode raises; its vmap calls the operator once for each."""
    y = meta(6, dtype=torch.long)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: linear_cross_entropy(x, meta(5, 16), y))(meta(6, 16))
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda w: embedding(y, w).float().sum())(meta(5, 16))


# ----- tracing -----------------------------------------------------------------------
@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_traced_shapes(reduction, dynamic):
    """torch.compile's tracing of both operators, forward and backward, on meta tensors."""
    torch._dynamo.reset()
    step = torch.compile(lambda i, t, w, y: linear_cross_entropy(embedding(i, t, scale=2.0, padding_idx=1), w, y,
                                                                 reduction=reduction).sum() * 0.3,
                         backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T in (6, 7):
        t, w = meta(9, 16).requires_grad_(), meta(5, 16).requires_grad_()
        loss = step(meta(T, dtype=torch.long), t, w, meta(T, dtype=torch.long))
        assert loss.shape == () and loss.dtype == torch.float32
        dt, dw = torch.autograd.grad(loss, (t, w))
        assert dt.shape == t.shape and dw.shape == w.shape
    torch._dynamo.reset()


# ----- widths ------------------------------------------------------------------------
def test_widths_that_the_kernels_cannot_count_are_refused():
    """Columns count in 32 bits, with those of the chunk behind the last: refused before anything is launched."""
    import ctypes as C
    from monarch_muon_amd import _abi
    emb = dict(tokens=4, vocab=100, width=1 << 28, dtype=_abi.F32, scale=1.0, padding_idx=-1, w_stride=1 << 28,
               dout_stride=1 << 28, index=4096, w=8192, out=12288, dout=16384, dw=20480, workspace=32768,
               workspace_bytes=1 << 62)
    lib = _abi.lib()
    for width in (1 << 28, (1 << 31) - 1):
        args = C.byref(_abi.EmbeddingArgs(**{**emb, "width": width}))
        assert lib.mmuon_embedding_fwd(args, None) == lib.mmuon_embedding_bwd(args, None) == -3
        assert b"2^28" in lib.mmuon_last_error()


# ----- refusals ----------------------------------------------------------------------
@pytest.mark.parametrize("call, match", [
    (lambda: linear_cross_entropy(torch.zeros((), dtype=torch.bfloat16), torch.zeros(5, 16).bfloat16(), torch.tensor(0)),
     "do not match"),
    (lambda: linear_cross_entropy(torch.zeros(2, 2, 0).bfloat16(), torch.zeros(5, 0).bfloat16(),
                                  torch.zeros(2, 2, dtype=torch.long)), "multiple of 8"),
    (lambda: embedding(torch.zeros(4, dtype=torch.long), torch.zeros(()), padding_idx=0), "expected weight"),
], ids=["x of no dimension", "x of no columns", "weight of no dimension"])
def test_shapes_without_columns_are_refused_as_such(call, match):
    with pytest.raises(ValueError, match=match):
        call()
