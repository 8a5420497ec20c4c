"""Rotary positions of query and key heads, with the optional store to the paged cache.

``rotary_embed`` rotates queries and keys, in place or to other buffers;
``rotary_store`` rotates the queries and writes the rotated keys and the values to the
paged main cache in the same launch, for layers whose cache is not written by
``qsa_prepare``.  ``rotary_frequencies`` builds the per-pair angles both take.

For pair ``i`` of a token at position ``p``, with ``a = p * frequencies[i]``::

    y1 = factor * (x1 * cos(a) - x2 * sin(a))
    y2 = factor * (x2 * cos(a) + x1 * sin(a))

``(x1, x2)`` are ``x[i], x[i + rotary_dim / 2]``, or ``x[2i], x[2i + 1]`` when
``interleaved``; dims from ``rotary_dim`` on pass through.  Angles are formed and reduced
in 64 bits, to within 2^-24 of a turn up to position 2^30 (and with 2^-54 of the position
beyond); no table is kept.
``inverse=True`` turns back, and with the same ``factor`` is the operator's gradient:
``dx = rotary_embed(dy, ..., inverse=True)``.
"""

from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none",
                       scaling_factor: float = 1.0, original_length: int | None = None,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """``(frequencies, factor)``: float64 ``[rotary_dim / 2]`` radians per position, and the
    factor on the rotated values.

    ``scaling``: "none"; "linear" (positions divided by ``scaling_factor``); "ntk" (the base
    grown so that the slowest pair is divided by it and the fastest unchanged); "yarn" (pairs
    that turn more than ``beta_fast`` times over ``original_length`` positions unchanged, those
    that turn fewer than ``beta_slow`` times divided, and a factor of ``0.1 ln(scaling_factor) +
    1``).  Between them yarn's share of the division grows linearly with the pair's index, from
    the last whole index at ``beta_fast`` turns to the first at ``beta_slow``, as in the code
    that checkpoints are trained and served with (the paper's ramp is linear in the turns)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (base > 0 and scaling_factor >= 1):
        raise ValueError("base must be positive and scaling_factor at least 1")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    factor = 1.0
    if scaling == "ntk":
        base = base * scaling_factor ** (rotary_dim / max(rotary_dim - 2, 1))
    f = float(base) ** (-i / half)
    if scaling == "linear":
        f = f / scaling_factor
    elif scaling == "yarn":
        if original_length is None or original_length <= 0:
            raise ValueError("yarn scaling needs original_length")
        if not beta_fast > beta_slow:
            raise ValueError("yarn scaling needs beta_fast > beta_slow")
        if not base > 1 or not beta_slow > 0:
            raise ValueError("yarn scaling needs a base above 1 and a positive beta_slow")

        def index(turns):  # of the pair that turns so often, as a real number
            return half * math.log(original_length / (2 * math.pi * turns)) / math.log(base)
        last = min(math.ceil(index(beta_slow)), rotary_dim - 1)
        first = min(max(math.floor(index(beta_fast)), 0), last)
        # a ramp of no length is a step behind `first`
        divided = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        f = f / scaling_factor * divided + f * (1 - divided)
        factor = 0.1 * math.log(scaling_factor) + 1
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return (f if device is None else f.to(device)), factor


def _heads(name: str, t: torch.Tensor, like: tuple, heads: int = 0) -> tuple:
    """(pointer, row stride, head stride) of a tensor [tokens, heads, dim] that fits ``like``
    (tokens, dim, dtype, device index)."""
    shape, (row, head, unit) = t.shape, t.stride() if t.dim() == 3 else (0, 0, 0)
    if len(shape) != 3 or shape[0] != like[0] or shape[2] != like[1] \
            or (heads and shape[1] != heads):
        raise ValueError(f"rotary: {name} must be [tokens, heads, dim] matching the others, "
                         f"got {tuple(shape)}")
    if t.dtype != like[2] or t.get_device() != like[3]:
        raise TypeError(f"rotary: {name} must be {like[2]} on the others' device, got {t.dtype} "
                        f"on {t.device}")
    if unit != 1 and like[1] > 1:
        raise ValueError(f"rotary: {name} needs a unit head-dim stride")
    return t.data_ptr(), row, head


def _like(t: torch.Tensor) -> tuple:
    if t.dim() != 3:
        raise ValueError("rotary: queries and keys must be [tokens, heads, dim]")
    shape = t.shape
    return shape[0], shape[2], t.dtype, t.get_device()


def _scalars(like: tuple, positions: torch.Tensor, frequencies: torch.Tensor) -> tuple:
    """Pointers, stride and rotary dim of positions and frequencies that fit ``like``, and the
    code of its dtype."""
    kind = _DTYPES.get(like[2])
    if kind is None:
        raise TypeError(f"rotary: bfloat16, float16 or float32 expected, got {like[2]}")
    if positions.dim() != 1 or positions.shape[0] != like[0] or positions.dtype != torch.int64:
        raise ValueError("rotary: positions must be int64 [tokens]")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 \
            or not frequencies.is_contiguous():
        raise TypeError("rotary: frequencies must be a contiguous float64 vector")
    rotary_dim = 2 * frequencies.shape[0]
    if not 2 <= rotary_dim <= like[1]:
        raise ValueError(f"rotary: {rotary_dim // 2} frequencies for a head of {like[1]}")
    if positions.get_device() != like[3] or frequencies.get_device() != like[3]:
        raise TypeError("rotary: positions and frequencies must be on the others' device")
    return positions.data_ptr(), positions.stride(0), frequencies.data_ptr(), rotary_dim, kind


_NO_SIDE = (None, 0, 0)
_NO_CACHE = (None, 0, 0, None, 0, 0, 0, None, 0, 0, 0, 0, 0, None, 0)


def rotary_embed(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor,
                 frequencies: torch.Tensor, *, interleaved: bool = False, inverse: bool = False,
                 factor: float = 1.0, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
    """Rotates queries and keys; returns ``(q_out, k_out)``.

    q ``[tokens, H_q, d]``, k ``[tokens, H_kv, d]`` (either may be None): bf16, fp16 or fp32,
    unit head-dim stride, other strides free (views of one projection).  positions: int64
    ``[tokens]``; frequencies: float64 ``[rotary_dim / 2]``.  ``q_out`` / ``k_out`` may be the
    inputs themselves (in place); other overlaps are not allowed.  New contiguous tensors are
    returned where they are None."""
    first = q if q is not None else k
    if first is None:
        raise ValueError("rotary: q or k expected")
    like = _like(first)
    tokens, dim, kind, index = like
    q_side = q_to = k_side = k_to = _NO_SIDE
    q_heads = k_heads = 0
    if q is not None:
        q_side = _heads("q", q, like)
        q_heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=kind, device=q.device)
        q_to = q_side if q_out is q else _heads("q_out", q_out, like, q_heads)
    else:
        q_out = None
    if k is not None:
        k_side = _heads("k", k, like)
        k_heads = k.shape[1]
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=kind, device=k.device)
        k_to = k_side if k_out is k else _heads("k_out", k_out, like, k_heads)
    else:
        k_out = None
    pos, pos_step, freq, rotary_dim, code = _scalars(like, positions, frequencies)
    _lib.ready(first)
    if tokens:
        with _lib.on_device(index):
            status = _lib.load_library().qsa_rotary(
                *q_side, q_heads, *q_to, *k_side, k_heads, *k_to, *_NO_CACHE, tokens, dim, pos,
                pos_step, freq, rotary_dim, factor, interleaved, inverse, code,
                _lib.raw_stream(index))
        if status:
            _lib.check(status, "rotary")
    return q_out, k_out


def rotary_store(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                 positions: torch.Tensor, frequencies: torch.Tensor, key_cache: torch.Tensor,
                 value_cache: torch.Tensor, slots: torch.Tensor, *, interleaved: bool = False,
                 factor: float = 1.0, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotates queries and keys and writes keys and values to the paged cache; returns the
    rotated queries (None without queries).

    As :func:`rotary_embed`, and: v ``[tokens, H_kv, d]``; key_cache / value_cache
    ``[blocks, page, H_kv, d]`` (the two halves of one ``[.., 2 d]`` buffer, or apart); slots:
    int64 ``[tokens]``, page * page_size + offset.  Tokens with a slot below 0 are not stored;
    one past the cache is not stored either and sets the device error word.  No two tokens may
    share a slot."""
    like = _like(k)
    tokens, dim, kind, index = like
    k_side = _heads("k", k, like)
    kv_heads = k.shape[1]
    v_side = _heads("v", v, like, kv_heads)
    cache = key_cache.shape
    if len(cache) != 4 or cache[2] != kv_heads or cache[3] != dim:
        raise ValueError(f"rotary: key_cache must be [blocks, page, {kv_heads}, {dim}]")
    if value_cache.shape != cache:
        raise ValueError("rotary: value_cache must be like key_cache")
    kc, vc = key_cache.stride(), value_cache.stride()
    if (kc[3] != 1 or vc[3] != 1) and dim > 1:
        raise ValueError("rotary: the caches need a unit head-dim stride")
    if key_cache.dtype != kind or value_cache.dtype != kind \
            or key_cache.get_device() != index or value_cache.get_device() != index:
        raise TypeError(f"rotary: the caches must be {kind} on {k.device}")
    if slots.dim() != 1 or slots.shape[0] != tokens or slots.dtype != torch.int64 \
            or slots.get_device() != index:
        raise ValueError(f"rotary: slots must be int64 [tokens] on {k.device}")
    q_side = q_to = _NO_SIDE
    heads = 0
    if q is not None:
        q_side = _heads("q", q, like)
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=kind, device=q.device)
        q_to = q_side if q_out is q else _heads("q_out", q_out, like, heads)
    else:
        q_out = None
    pos, pos_step, freq, rotary_dim, code = _scalars(like, positions, frequencies)
    _lib.ready(k)
    if tokens:
        with _lib.on_device(index):
            status = _lib.load_library().qsa_rotary(
                *q_side, heads, *q_to, *k_side, kv_heads, None, 0, 0, *v_side,
                key_cache.data_ptr(), kc[0], kc[1], kc[2],
                value_cache.data_ptr(), vc[0], vc[1], vc[2], cache[0], cache[1],
                slots.data_ptr(), slots.stride(0), tokens, dim, pos, pos_step, freq, rotary_dim,
                factor, interleaved, False, code, _lib.raw_stream(index))
        if status:
            _lib.check(status, "rotary")
    return q_out


__all__ = ["rotary_frequencies", "rotary_embed", "rotary_store"]
