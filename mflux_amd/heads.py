"""What an attention block does to its heads between the stacked q/k/v product
and the output projection: ``rotary_tables``, ``rotary`` (RMS norm of the heads
and rotary positions) and ``attention``.

In the reference: AttentionUtils.process_qkv, apply_rope and compute_attention
(src/mflux/models/flux/model/flux_transformer/common/attention_utils.py:21-49,
76-80), there with ``[B, H, S, D]`` arrays.  Here heads stay where the linear
layers leave them, ``[B, S, H, D]`` (or packed ``[T, H, D]``), and are read through
their strides: a slice of a stacked product needs no copy.

The calls run on the current stream of their tensors' device and launch nothing
anywhere else; sums are made in a fixed order, so the same inputs give the same
bits.  All three can be captured into a graph.  Gradients are first derivatives in
reverse mode: a second derivative and forward mode are refused.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .core import _DTYPE_CODE, _require_hip


def _integers(fn: str, name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"[{fn}] {name} must be int32 or int64, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"[{fn}] {name} lives on {t.device}, expected {device}")
    return t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _is_integer(value) -> bool:
    return isinstance(value, int) and not isinstance(value, bool)


# ---- tables -----------------------------------------------------------------

_SCALINGS = {"linear": (1, {"type", "factor"}), "ntk": (2, {"type", "factor"}),
             "yarn": (3, {"type", "factor", "original_length", "beta_fast", "beta_slow", "attention_factor"})}


_FLOAT32_MAX = torch.finfo(torch.float32).max


def _number(value) -> bool:
    return isinstance(value, (int, float)) and not isinstance(value, bool) and math.isfinite(value)


def _scaling(scaling: dict | None, base: float, dims: tuple[int, ...]) -> tuple:
    """``(kind, factor, original length, beta_fast, beta_slow, factor of the tables)`` as the op takes them."""
    if scaling is None:
        return 0, 1.0, 1.0, 32.0, 1.0, 1.0
    kind = scaling.get("type")
    if kind not in _SCALINGS:
        raise ValueError(f"[rotary_tables] scaling type must be 'linear', 'ntk' or 'yarn', got {kind!r}")
    code, known = _SCALINGS[kind]
    if set(scaling) - known:
        raise ValueError(f"[rotary_tables] unknown scaling entries for '{kind}': {sorted(map(str, set(scaling) - known))}")
    factor = scaling.get("factor")
    if not _number(factor) or factor < 1:
        raise ValueError(f"[rotary_tables] scaling factor must be at least 1, got {factor!r}")
    if kind == "ntk" and 2 in dims:
        raise ValueError("[rotary_tables] 'ntk' needs dimensions above 2")
    if kind != "yarn":
        return code, factor, 1.0, 32.0, 1.0, 1.0
    length, fast, slow = scaling.get("original_length"), scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)
    if not _number(length) or length <= 0:
        raise ValueError(f"[rotary_tables] 'yarn' needs a positive original_length, got {length!r}")
    if not (_number(fast) and _number(slow) and fast >= slow > 0) or base <= 1:
        raise ValueError("[rotary_tables] 'yarn' needs beta_fast >= beta_slow > 0 and a base above 1")
    tables = scaling.get("attention_factor")
    if tables is None:
        tables = 0.1 * math.log(factor) + 1.0
    elif not _number(tables) or abs(tables) > _FLOAT32_MAX:
        raise ValueError(f"[rotary_tables] attention_factor must be a number that float32 holds, got {tables!r}")
    return code, factor, length, fast, slow, tables


def _fastest(d: int, base: float, kind: int, factor: float) -> float:
    """The logarithm of the angle that a position adds to the last of ``d / 2`` pairs, the fastest where ``base`` is below 1;
    'linear' and 'ntk' both divide it."""
    return -(1 - 2 / d) * math.log(base) - (math.log(factor) if kind in (1, 2) else 0.0)


def rotary_tables(positions: torch.Tensor, dims: int | tuple[int, ...], base: float = 10000.0,
                  scaling: dict | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)`` of the rotary angles of ``positions``, float32 ``[S, R / 2]``.

    ``positions``: integers ``[S]`` with ``dims`` the number of channels that turn, or
    ``[S, A]`` with one such number for each of ``A`` axes, whose pairs lie side by
    side (an image token's id, row and column in the DiT blocks: ``(16, 56, 56)``).
    Negative positions are fine; int64 ones count as the nearest that int32 holds (the
    device is not waited for to look at them).  At most 512 channels in all.

    ``scaling`` stretches the angles for contexts longer than a model was trained
    on: ``{"type": "linear", "factor": f}`` divides positions, ``"ntk"`` raises the base so
    that the slowest pair is divided by ``f`` and the fastest by nothing, and ``"yarn"``
    (``original_length``, ``beta_fast``, ``beta_slow``, ``attention_factor``) divides the pairs
    that turn less than ``beta_slow`` times over the original length, leaves those that turn more
    than ``beta_fast`` times, and multiplies the tables by ``0.1 ln f + 1``.

    Angles are taken in float64: a float32 product is off by thousandths at far
    positions.  ``base`` is such that a position adds at most 4 to an angle (any from 0.25 on)."""
    fn = "rotary_tables"
    if not isinstance(positions, torch.Tensor) or positions.ndim not in (1, 2):
        raise ValueError(f"[{fn}] positions must be a tensor [S] or [S, A]")
    if positions.ndim == 1:
        axes = (dims,)
    else:
        axes = tuple(dims) if isinstance(dims, (tuple, list)) else (dims,)
        if len(axes) != positions.shape[1]:
            raise ValueError(f"[{fn}] positions have {positions.shape[1]} axes, dims {len(axes)}")
    if not axes or not all(_is_integer(d) and d > 0 and d % 2 == 0 for d in axes):
        raise ValueError(f"[{fn}] dims must be a positive even number, or one for each axis, got {dims!r}")
    if sum(axes) > 512:
        raise ValueError(f"[{fn}] at most 512 channels turn, got {sum(axes)}")
    if not _number(base) or base <= 0:
        raise ValueError(f"[{fn}] base must be positive, got {base!r}")
    arguments = _scaling(scaling, base, axes)
    if base < 0.25 and any(_fastest(d, base, *arguments[:2]) > math.log(4) for d in axes):
        raise ValueError(f"[{fn}] base is too small: a position may add at most 4 to an angle, got {base!r}")
    positions = _integers(fn, "positions", positions, positions.device)
    _require_hip(fn, positions, "positions")
    return _lib.ops().rotary_tables(positions.reshape(positions.shape[0], len(axes)), axes, base, *arguments)


# ---- RMS norm of the heads and rotary positions -------------------------------------

def rotary(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, *, layout: str = "interleaved",
           positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
           eps: float = 1e-6):
    """Rotary positions of ``q`` and ``k`` in one pass, with the RMS norm of their heads in
    front where a weight is given.  Returns ``(q', k')``, or ``q'`` for ``k=None``.

    ``q``: ``[B, S, H, D]`` or packed ``[T, H, D]``, ``k`` the same with its own number of
    heads; float32, float16 or bfloat16, ``D`` even and up to 512; any strides (a last
    axis that is not dense is copied), results densely packed.
    ``cos``, ``sin``: float32 ``[P, R / 2]`` of ``rotary_tables``; the first ``R`` channels turn and the
    others pass.  ``layout``: ``"interleaved"`` turns channels ``(2i, 2i + 1)``, ``"half"``
    ``(i, i + R / 2)``.
    ``positions``: the tables' row of every token, int32 or int64 ``[S]`` or ``[B, S]`` (packed: ``[T]``),
    clamped to the tables; without them a token's row is its place in its sequence axis.
    ``q_weight``, ``k_weight``: ``[D]`` of the tensors' type: ``x / sqrt(mean(x^2) + eps) * weight``
    before the turn.

    Everything in between is float32 and rounded once.  Gradients for ``q``, ``k`` and the
    weights; none for the tables."""
    fn = "rotary"
    if layout not in _lib.ROTARY_LAYOUTS:
        raise ValueError(f"[{fn}] layout must be 'interleaved' or 'half', got {layout!r}")
    if q.ndim not in (3, 4):
        raise ValueError(f"[{fn}] q must be [B, S, H, D] or packed [T, H, D], got {tuple(q.shape)}")
    if q.dtype not in _DTYPE_CODE:
        raise ValueError(f"[{fn}] q must be float32, float16 or bfloat16, got {q.dtype}")
    D = q.shape[-1]
    if D % 2 or not 0 < D <= 512:
        raise ValueError(f"[{fn}] heads must have an even size up to 512, got {D}")
    if k is not None and (k.ndim != q.ndim or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != D or k.dtype != q.dtype):
        raise ValueError(f"[{fn}] q and k must agree in type and in all axes but the heads, got {tuple(q.shape)} {q.dtype} and "
                         f"{tuple(k.shape)} {k.dtype}")
    if not 0 < q.shape[-2] <= 65536 or (k is not None and not 0 < k.shape[-2] <= 65536):
        raise ValueError(f"[{fn}] q and k need between 1 and 65536 heads")
    if any(t is not None and t.numel() // D >= 2 ** 31 - 1 for t in (q, k)):
        raise ValueError(f"[{fn}] fewer than 2^31 rows (token, head) fit a call")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"[{fn}] cos and sin must be float32 [P, R / 2] of one shape, got {tuple(cos.shape)} {cos.dtype} and "
                         f"{tuple(sin.shape)} {sin.dtype}")
    if 2 * cos.shape[1] > D:
        raise ValueError(f"[{fn}] the tables turn {2 * cos.shape[1]} channels, heads have {D}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"[{fn}] the tables have no gradient here: detach them")
    tokens = q.shape[-3]
    if cos.shape[0] == 0 and q.numel():
        raise ValueError(f"[{fn}] the tables are empty")
    if positions is None:
        if cos.shape[0] < tokens:
            raise ValueError(f"[{fn}] the tables have {cos.shape[0]} rows for {tokens} tokens")
    else:
        shapes = ((tokens,),) if q.ndim == 3 else ((tokens,), (1, tokens), (q.shape[0], tokens))
        if tuple(positions.shape) not in shapes:
            raise ValueError(f"[{fn}] positions must have the shape {shapes[-1]}, got {tuple(positions.shape)}")
    for name, w, t in (("q_weight", q_weight, q), ("k_weight", k_weight, k)):
        if w is not None and (t is None or tuple(w.shape) != (D,) or w.dtype != q.dtype):
            raise ValueError(f"[{fn}] {name} must be a [{D}] vector of {q.dtype}" + (" and needs its tensor" if t is None else ""))
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"[{fn}] eps must not be negative, got {eps!r}")
    for name, t in (("k", k), ("cos", cos), ("sin", sin), ("positions", positions), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and t.device != q.device:
            raise ValueError(f"[{fn}] `{name}` lives on {t.device}, q on {q.device}")
    if positions is not None:
        positions = _integers(fn, "positions", positions, q.device)
        positions = positions[None] if positions.ndim == 1 else positions
    _require_hip(fn, q, "q")
    packed = q.ndim == 3
    if packed:
        q, k = q[None], None if k is None else k[None]
    yq, yk = _lib.ops().rotary_call(q, k, cos, sin, positions, q_weight, k_weight, _lib.ROTARY_LAYOUTS[layout], eps)
    if packed:
        yq, yk = yq[0], None if k is None else yk[0]
    return yq if k is None else (yq, yk)


# ---- attention ------------------------------------------------------------------------

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: float | None = None,
              q_lengths: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None,
              q_offsets: torch.Tensor | None = None, k_offsets: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T + mask) v`` with grouped heads, for batched or packed sequences
    (``mx.fast.scaled_dot_product_attention`` in the reference).

    Batched: ``q [B, Sq, H, D]``, ``k`` and ``v [B, Sk, Hkv, D]``; ``q_lengths`` and ``k_lengths`` (``[B]``
    integers on the device, each optional) say how many queries and keys of an entry there are.
    Packed: ``q [Tq, H, D]``, ``k`` and ``v [Tk, Hkv, D]``, sequence ``s`` having the rows ``q_offsets[s]`` to
    ``q_offsets[s + 1]`` of ``q`` and the same of ``k_offsets`` (default: ``q_offsets``) of ``k`` and ``v``; offsets
    must not decrease.  Lengths and offsets are read by the kernels alone, clamped to the
    tensors: a call never waits for the device, and wrong ones never reach outside them.

    float16 or bfloat16, ``D`` a multiple of 8 up to 256, ``H`` a multiple of ``Hkv`` (head ``h`` reads
    key head ``h // (H // Hkv)``).  Any strides of rows of whole 16 bytes; others are copied first.
    ``scale``: ``1 / sqrt(D)`` unless given; positive.
    ``causal``: aligned to the last token, query ``i`` of ``n`` sees the first ``i + 1 + m - n`` of ``m`` keys, so one
    query behind a cache sees all of it.  A query that sees no key gets zeros, and so does every
    row that belongs to no sequence (padding; rows behind the last offset), in the result and
    in the gradients.  What a query does not see never reaches it, infinities and NaN included; one whose
    visible scores are all ``-inf`` has no softmax and gets NaN.

    Statistics and sums are float32; the probabilities (and in the backward pass the
    scores' gradients) are rounded to the tensors' type for the second product.  The backward
    pass makes the scores again from one saved float32 per row and head, and takes ``sum(dy y)``
    from ``y`` and what its rounding left, which the forward pass keeps when a gradient is wanted."""
    fn = "attention"
    packed = q_offsets is not None
    if k_offsets is not None and not packed:
        raise ValueError(f"[{fn}] k_offsets need q_offsets")
    if packed and (q_lengths is not None or k_lengths is not None):
        raise ValueError(f"[{fn}] packed sequences have offsets, batched ones lengths, not both")
    n = 3 if packed else 4
    if q.ndim != n or k.ndim != n or v.ndim != n:
        raise ValueError(f"[{fn}] q, k and v must be " + ("packed [T, H, D] with offsets" if packed else "[B, S, H, D] without offsets") +
                         f", got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape != v.shape or q.shape[-1] != k.shape[-1] or (not packed and q.shape[0] != k.shape[0]):
        raise ValueError(f"[{fn}] k and v must have one shape and q's batch and head size, got {tuple(q.shape)}, {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"[{fn}] q, k and v must all be float16 or all bfloat16, got {q.dtype}, {k.dtype} and {v.dtype}")
    H, D = q.shape[-2:]
    if D % 8 or not 0 < D <= 256:
        raise ValueError(f"[{fn}] the head size must be a multiple of 8 up to 256, got {D}")
    if not 0 < k.shape[-2] <= H or H % k.shape[-2] or H > 65536:
        raise ValueError(f"[{fn}] {H} query heads do not share {k.shape[-2]} key heads evenly")
    if q.shape[-3] * H > 2 ** 30 or k.shape[-3] > 2 ** 30:
        raise ValueError(f"[{fn}] at most 2^30 queries times heads, and keys, in an entry")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not 0 < scale <= 1e30:
        raise ValueError(f"[{fn}] scale must be positive and finite, got {scale!r}")
    for name, t in (("k", k), ("v", v), ("q_offsets", q_offsets), ("k_offsets", k_offsets), ("q_lengths", q_lengths), ("k_lengths", k_lengths)):
        if t is not None and t.device != q.device:
            raise ValueError(f"[{fn}] `{name}` lives on {t.device}, q on {q.device}")

    def counts(name, t, length):
        if t is None:
            return None
        if t.ndim != 1 or (length is not None and t.shape[0] != length):
            raise ValueError(f"[{fn}] {name} must be a vector" + ("" if length is None else f" of {length} values") + f", got {tuple(t.shape)}")
        return _integers(fn, name, t, q.device)

    if packed:
        q_offsets = counts("q_offsets", q_offsets, None)
        if q_offsets.shape[0] < 2:
            raise ValueError(f"[{fn}] offsets are one more than the sequences, of which there is at least one")
        k_offsets = q_offsets if k_offsets is None else counts("k_offsets", k_offsets, q_offsets.shape[0])
    else:
        q_lengths, k_lengths = counts("q_lengths", q_lengths, q.shape[0]), counts("k_lengths", k_lengths, q.shape[0])
    _require_hip(fn, q, "q")
    return _lib.ops().attention_call(q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale)
