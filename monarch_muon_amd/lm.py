"""The two ends of a language model on the MI355X kernels: the token embedding, and the head with its loss.

* ``embedding(index, weight)``: rows of a table, and the table's gradient.
* ``linear_cross_entropy(x, weight, target)``: softmax cross entropy of ``x @ weight.T``, and the gradients of ``x``
  and ``weight``, without the logits' matrix.

The reference computes both with torch's ops (``pretrain/src/models/llama.py``: ``wte``, ``lm_head`` and
``F.cross_entropy`` over the whole logits).  Both are native torch operators (``csrc/torch_lm.cpp``), registered with
fake implementations, on ``torch.cuda.current_stream()``; there is no fallback.
"""
from __future__ import annotations

import torch

from . import _abi, butterfly

__all__ = ["linear_cross_entropy", "embedding"]

_REDUCTIONS = {"none": _abi.CE_NONE, "mean": _abi.CE_MEAN, "sum": _abi.CE_SUM}
_loss_op = _embedding_op = None


def _load() -> None:
    """Register the operators' fakes; raises where the native library is not built."""
    global _loss_op, _embedding_op
    if butterfly._linear_op is None:
        butterfly._load_linear()

    @torch.library.register_fake("mmuon::linear_cross_entropy")
    def _(x, weight, target, ignore_index, reduction, piece_tokens):
        return x.new_empty(target.shape if reduction == _abi.CE_NONE else (), dtype=torch.float32)

    @torch.library.register_fake("mmuon::linear_cross_entropy_grad")
    def _(x, weight, target, grad, ignore_index, reduction, piece_tokens, need_dx, need_dw):
        return (x.new_empty(target.shape if reduction == _abi.CE_NONE else (), dtype=torch.float32),
                x.new_empty(x.shape if need_dx else (0,)), weight.new_empty(weight.shape if need_dw else (0,)))

    @torch.library.register_fake("mmuon::scale_")
    def _(x, y, factor):
        return None

    @torch.library.register_fake("mmuon::embedding")
    def _(index, weight, scale, padding_idx):
        return weight.new_empty(*index.shape, weight.shape[1])

    @torch.library.register_fake("mmuon::embedding_grad")
    def _(dout, index, vocab, scale, padding_idx):
        return dout.new_empty(vocab, dout.shape[-1])

    _loss_op = torch.ops.mmuon.linear_cross_entropy.default
    _embedding_op = torch.ops.mmuon.embedding.default


try:
    _load()
except (RuntimeError, OSError):   # not built yet: the calls try again and raise
    pass


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", piece_tokens: int | None = None) -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T`` (float32 result), as
    ``F.cross_entropy(F.linear(x, weight).float(), target)`` with a loss of float32 logits, which are not kept: the
    gradients are of probabilities off by 3.4e-4 of themselves at most, rounded to bfloat16 before the products.

    ``x`` (..., D) and ``weight`` (V, D) bfloat16 (cast under bf16 autocast), D a multiple of 8, V any; ``target``
    (...) int64 or int32.  Tokens whose target is ``ignore_index`` count for nothing; a target that is neither that
    nor a token gives NaN.  ``reduction``: "mean" over the tokens that count (NaN if none does), "sum", or "none" (the
    shape of ``target``).

    Differentiable in ``x`` and ``weight``.  With "mean" and "sum" the forward makes the gradients, so one backward
    can be taken of it, and a factor that arrives then (``loss / 3``) is multiplied into their bfloat16 values: a second
    rounding, none for a power of two, and a pass over both where it is not 1.  With "none" the backward makes the
    logits again.  There is no second derivative: one of gradients taken with ``create_graph`` raises.

    A token with a logit of +inf or NaN, or with none above -inf, has NaN for its loss and gradients; so has one with
    a logit beyond 2.3e38, which float32 does not hold in base 2.

    ``piece_tokens``: tokens whose logits are held at a time, 16 bits each; by default as many as fit 1 GiB.  Several
    pieces also hold float32 sums of ``weight``'s gradient, where it is wanted, so a smaller piece can take more memory
    than one of all tokens (which the default then is).
    """
    if _loss_op is None:
        _load()
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    if piece_tokens is not None and piece_tokens < 1:
        raise ValueError(f"piece_tokens must be positive, not {piece_tokens}")
    if torch.is_autocast_enabled():
        dt = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dt), weight.to(dt)
    shape = target.shape
    if x.dim() == 0 or x.shape[:-1] != shape:
        raise ValueError(f"x {tuple(x.shape)} and target {tuple(shape)} do not match")
    if x.dim() != 2:
        x, target = x.reshape(target.numel(), x.shape[-1]), target.reshape(-1)
    out = _loss_op(x, weight, target, ignore_index, _REDUCTIONS[reduction], piece_tokens or 0)
    return out.view(shape) if out.dim() else out


def embedding(index: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[index]`` (..., D) in ``weight``'s type (bfloat16 or float32; one rounding).

    ``index`` int64 or int32, ``weight`` (V, D).  An id outside [0, V) gives a row of NaN.  Differentiable in
    ``weight``: the gradient is dense, the same whatever the timing, each row the float32 sum over its tokens in a
    fixed order; ids outside [0, V) and ``padding_idx`` (counted from the end where negative) take none.  The
    gradient is differentiable in the one that arrives.
    """
    if _embedding_op is None:
        _load()
    pad = -1
    if padding_idx is not None and weight.dim() == 2:   # (the operator refuses others)
        rows = weight.shape[0]
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx {padding_idx} is not one of {rows} rows")
        pad = padding_idx % rows
    return _embedding_op(index, weight, float(scale), pad)
