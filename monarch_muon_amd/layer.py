"""What stands between a decoder layer's Monarch projections, on the MI355X kernels.

* ``rms_norm(x, weight, residual=r)``: the norm with the residual's addition; ``rms_norm_fp8`` with an output in 8 bits.
* ``rotary(q, k, table)``: rotary positions of queries and keys, by a table that ``rotary_table`` makes.
* ``differential_attention(q, k, v, lam)``: the difference of two softmax maps over shared values; for training, for
  prompts, and for new tokens of a cache.

The reference computes with torch's ops what it has of these (``pretrain/src/models/llama.py``: ``RMSNorm``,
``apply_rotary_emb``, ``F.scaled_dot_product_attention``).  All
are native torch operators (``csrc/torch_layer.cpp``), registered with fake implementations, on
``torch.cuda.current_stream()``; there is no fallback.
"""
from __future__ import annotations

import math

import torch

from . import butterfly

__all__ = ["rms_norm", "rms_norm_fp8", "rotary", "rotary_table", "differential_attention"]

_norm_op = _norm_fp8_op = _rotary_op = _attention_op = None


def _load() -> None:
    """Register the operators' fakes; raises where the native library is not built."""
    global _norm_op, _norm_fp8_op, _rotary_op, _attention_op
    if butterfly._linear_op is None:
        butterfly._load_linear()

    @torch.library.register_fake("mmuon::rms_norm")
    def _(x, residual, weight, eps):
        return (x.new_empty(x.shape), x.new_empty((0,) if residual is None else x.shape),
                x.new_empty((math.prod(x.shape[:-1]),), dtype=torch.float32))

    @torch.library.register_fake("mmuon::rms_norm_grad")
    def _(h, inv, weight, dy, dh, need_dw):
        return h.new_empty(h.shape), weight.new_empty(weight.shape if need_dw else (0,))

    @torch.library.register_fake("mmuon::rms_norm_fp8")
    def _(x, residual, weight, eps, dtype, group):
        groups = (x.shape[-1] + 127) // 128 if group else 1
        return (x.new_empty(x.shape, dtype=dtype), x.new_empty((*x.shape[:-1], groups), dtype=torch.float32),
                x.new_empty((0,) if residual is None else x.shape))

    @torch.library.register_fake("mmuon::rotary")
    def _(q, k, table, positions, interleaved, back):
        return q.new_empty(q.shape), k.new_empty(k.shape)

    @torch.library.register_fake("mmuon::differential_attention")
    def _(q, k, v, lam, lengths, starts, causal, scale, save):
        B, T, heads = q.shape[:3]
        o = q.new_empty(B, T, heads // 2, v.shape[3])
        if not save:
            return o, q.new_empty(0), q.new_empty(0), q.new_empty(0, dtype=torch.float32)
        f32 = dict(dtype=torch.float32)
        return o, torch.empty_like(o, **f32), torch.empty_like(o, **f32), q.new_empty(B, heads // 2, T, 4, dtype=torch.float32)

    @torch.library.register_fake("mmuon::differential_attention_grad")
    def _(q, k, v, lam, lengths, starts, o1, o2, lse, dout, causal, scale, need_q, need_kv):
        return (q.new_empty(q.shape if need_q else (0,)), k.new_empty(k.shape if need_kv else (0,)),
                v.new_empty(v.shape if need_kv else (0,)), lam.new_empty(lam.shape if need_q else (0,)))

    _norm_op = torch.ops.mmuon.rms_norm.default
    _norm_fp8_op = torch.ops.mmuon.rms_norm_fp8.default
    _rotary_op = torch.ops.mmuon.rotary.default
    _attention_op = torch.ops.mmuon.differential_attention.default


try:
    _load()
except (RuntimeError, OSError):   # not built yet: the calls try again and raise
    pass


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``y = h * weight / sqrt(mean(h ** 2) + eps)`` over the last dimension, in fp32 with one rounding.

    Without ``residual``, ``h`` is ``x`` and the result ``y``.  With it, ``h = x + residual`` rounded to their type, which
    is what the residual stream keeps, and the result is ``(y, h)``.  ``x`` (..., D) bfloat16 or float32 at any row
    stride, D at most 32768 (bfloat16) or 16384, fewer than 2 ** 31 rows; ``residual`` of its shape and type; ``weight`` (D) of its
    type or float32.

    Differentiable in all three; ``weight``'s gradient is the fp32 sum over the rows in an order that depends on the
    sizes alone.  There is no second derivative.  A row with a NaN or an infinity has NaN in ``y``; one whose squares' sum
    is beyond float32 (magnitudes around 1e19) has zeros.
    """
    if _norm_op is None:
        _load()
    y, h, _ = _norm_op(x, residual, weight, float(eps))
    return y if residual is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6,
                 dtype: torch.dtype = torch.float8_e4m3fn, group: int | None = 128):
    """``rms_norm`` with ``y`` in 8 bits: ``(codes, scale)``, or ``(codes, scale, h)`` with ``residual``.

    ``y ~ codes.float() * scale``, a float32 scale for each 128 columns, (..., ceil(D / 128)), or with ``group=None`` for the
    row, (..., 1): the largest magnitude over 448 (``float8_e4m3fn``) or 57344 (``float8_e5m2``), 1 where that is zero or
    below float32's normal numbers (the codes are then zeros).
    A code is ``y / scale`` rounded once, from fp32, to the nearest even.  It has no gradient: inputs that require one
    raise.
    """
    if _norm_fp8_op is None:
        _load()
    if group not in (128, None):
        raise ValueError(f"group must be 128 columns or None, not {group}")
    codes, scale, h = _norm_fp8_op(x, residual, weight, float(eps), dtype, group or 0)
    return (codes, scale) if residual is None else (codes, scale, h)


def rotary_table(dim: int, length: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                 trained: int | None = None, fast: float | None = None, slow: float = 1.0,
                 attention_factor: float | None = None, device=None) -> torch.Tensor:
    """The float32 table (``length``, ``dim``) that ``rotary`` reads: for each position the cosines and then the sines of
    ``dim / 2`` angles ``position * base ** (-2 i / dim)``, computed in 64 bits.

    ``scaling`` for contexts ``factor`` times as long as the ``trained`` length:

    * "linear": all angles over ``factor``;
    * "ntk": ``base`` times ``factor ** (dim / (dim - 2))``;
    * "yarn": angles of over ``fast`` (32) turns within ``trained`` as they are, of under ``slow`` (1) over ``factor``, a
      ramp over the pairs between; cosines and sines times ``attention_factor`` (``0.1 ln(factor) + 1``);
    * "llama": as they are over ``fast`` (4) turns, over ``factor`` under ``slow`` (1), a ramp over the turns between.
    """
    if dim < 2 or dim % 2 or length < 0:
        raise ValueError(f"a table needs an even number of columns and a length, not {dim} and {length}")
    if scaling not in (None, "linear", "ntk", "yarn", "llama"):
        raise ValueError(f"scaling must be 'linear', 'ntk', 'yarn', 'llama' or None, not {scaling!r}")
    if not factor > 0 or not base > 0:
        raise ValueError(f"base and factor must be positive, not {base} and {factor}")
    if scaling in ("yarn", "llama") and (trained is None or trained < 1):
        raise ValueError(f"scaling {scaling!r} needs the trained length")
    if scaling in ("yarn", "llama"):
        fast = {"yarn": 32.0, "llama": 4.0}[scaling] if fast is None else fast
        if not (slow < fast if scaling == "llama" else 0 < slow <= fast):
            raise ValueError(f"scaling {scaling!r} needs {'slow < fast' if scaling == 'llama' else '0 < slow <= fast'}, not {slow} and {fast}")
    if scaling == "yarn" and not base > 1:
        raise ValueError(f"scaling 'yarn' needs a base above 1, not {base}")
    i = torch.arange(0, dim, 2, dtype=torch.float64, device=device)
    if scaling == "ntk":
        base = base * factor ** (dim / max(dim - 2, 1))
    f = base ** (-i / dim)
    size = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):   # that takes so many turns within the trained length
            return dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        size = (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0) if attention_factor is None else attention_factor
    elif scaling == "llama":
        keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    a = torch.arange(length, dtype=torch.float64, device=device).unsqueeze(1) * f
    return (torch.cat([a.cos(), a.sin()], 1) * size).float()


def rotary(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor | None = None, *,
           interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``q`` (B, T, H, D) and ``k`` (B, T, K, D) with their first ``table.shape[1]`` columns rotated by position, in fp32
    with one rounding; the columns behind are copied.

    Pairs are columns ``i`` and ``i + part / 2``, or with ``interleaved`` ``2 i`` and ``2 i + 1``.  ``positions`` (T) or
    (B, T), int64 or int32, by default 0 .. T - 1; one outside the table gives NaN.  bfloat16 or float32 at any strides;
    the results are contiguous.  Differentiable in ``q`` and ``k``, to any order.
    """
    if _rotary_op is None:
        _load()
    return _rotary_op(q, k, table, positions, bool(interleaved), False)


def differential_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, *, causal: bool = True,
                           scale: float | None = None, lengths: torch.Tensor | None = None,
                           starts: torch.Tensor | None = None) -> torch.Tensor:
    """``(softmax(q1 k1^T scale) - lam softmax(q2 k2^T scale)) v`` for each head, (B, T, H, 2 D) bfloat16.

    ``q`` (B, T, 2 H, D), ``k`` (B, S, 2 K, D) and ``v`` (B, S, K, 2 D) bfloat16 (cast under bf16 autocast) at any strides (copied
    where rows of a head are no whole 16-byte chunks or tokens stand 2 ** 22 elements apart), D a multiple of 8 up to 128: query
    heads ``2 h`` and ``2 h + 1`` are head ``h``'s two maps, key heads ``2 g`` and ``2 g + 1`` with value head ``g`` are shared by
    H / K heads.  ``lam``: one value or one for each head (taken as float32).  ``scale`` is ``D ** -0.5`` by default.

    ``lengths`` (B): the keys of each sequence that count; those behind are not read (a cache).  ``causal``: query ``t`` of
    sequence ``b`` sees keys up to ``starts[b] + t``, by default ``lengths[b] - T + t``: the queries are the last ones of their
    sequence.  A query that sees no key has zeros and reaches nothing, whatever it holds; a key that no query sees has zeros
    for gradients.  Between a query and a later key that ``causal`` alone hides an infinity or a NaN may show as NaN: of the key
    or its value in the query's output and gradient, of the query or its output's gradient in the key's and the value's.

    B H T is below 2 ** 29 and B K S below 2 ** 31 - 1024; with gradients B H T is at most 2 ** 28 - 16, B K S below 2 ** 30 and, for
    T > 1, H D below 2 ** 21.

    Differentiable in ``q``, ``k``, ``v`` and ``lam``; every sum has an order that depends on the sizes alone, so gradients are
    the same bits every time.  Probabilities are rounded to bfloat16 before their products with the values, as are the
    scores' gradients before theirs.  There is no second derivative.
    """
    if _attention_op is None:
        _load()
    if torch.is_autocast_enabled():
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if q.dim() != 4:
        raise ValueError(f"expected q (B, T, 2 H, D), got {tuple(q.shape)}")
    heads = q.shape[2] // 2
    lam = lam.float()
    if lam.numel() == 1 and lam.dim() <= 1:
        lam = lam.reshape(1).expand(heads)
    return _attention_op(q, k, v, lam, lengths, starts, bool(causal), float(q.shape[3] ** -0.5 if scale is None else scale),
                         False)[0]
