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
in 64 bits, so positions of any size keep their precision; no table is kept.
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
    that turn fewer than ``beta_slow`` times divided, a linear ramp over the number of turns
    between them, and a factor of ``0.1 ln(scaling_factor) + 1``)."""
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
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        f = f / scaling_factor * (1 - keep) + f * keep
        factor = 0.1 * math.log(scaling_factor) + 1
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return (f if device is None else f.to(device)), factor


def _heads(name: str, t: torch.Tensor, like: torch.Tensor, heads: int | None = None) -> None:
    if t.dim() != 3 or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2] \
            or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"rotary: {name} must be [tokens, heads, dim] matching the others, "
                         f"got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"rotary: {name} must be {like.dtype} on {like.device}, "
                        f"got {t.dtype} on {t.device}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"rotary: {name} needs a unit head-dim stride")


def _call(q, q_out, k, k_out, v, k_cache, v_cache, slots, positions, frequencies, interleaved,
          inverse, factor) -> None:
    like = q if q is not None else k
    if like.dtype not in _DTYPES:
        raise TypeError(f"rotary: bfloat16, float16 or float32 expected, got {like.dtype}")
    tokens, _, dim = like.shape
    dev = like.device
    if positions.dim() != 1 or positions.shape[0] != tokens or positions.dtype != torch.int64:
        raise ValueError("rotary: positions must be int64 [tokens]")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64:
        raise TypeError("rotary: frequencies must be a float64 vector")
    rotary_dim = 2 * frequencies.shape[0]
    if not 2 <= rotary_dim <= dim:
        raise ValueError(f"rotary: {frequencies.shape[0]} frequencies for a head of {dim}")
    if positions.device != dev or frequencies.device != dev:
        raise TypeError(f"rotary: positions and frequencies must be on {dev}")
    _lib.ensure_device(dev)
    if tokens == 0:
        return
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    none = (None, 0, 0)

    def rows(t):
        return none if t is None else (t.data_ptr(), t.stride(0), t.stride(1))

    if k_cache is None:
        caches = (None, 0, 0, 0, None, 0, 0, 0, 0, 0, None, 0)
    else:
        caches = (k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
                  v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
                  k_cache.shape[0], k_cache.shape[1], slots.data_ptr(), slots.stride(0))
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().qsa_rotary(
            *rows(q), 0 if q is None else q.shape[1], *rows(q_out),
            *rows(k), 0 if k is None else k.shape[1], *rows(k_out), *rows(v), *caches,
            tokens, dim, positions.data_ptr(), positions.stride(0), frequencies.data_ptr(),
            rotary_dim, factor, 1 if interleaved else 0, 1 if inverse else 0,
            _DTYPES[like.dtype], _lib.stream_ptr(dev)), "rotary")


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
    if q is None and k is None:
        raise ValueError("rotary: q or k expected")
    like = q if q is not None else k
    outs = []
    for name, x, out in (("q", q, q_out), ("k", k, k_out)):
        if x is None:
            outs.append(None)
            continue
        _heads(name, x, like)
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _heads(name + "_out", out, x, x.shape[1])
        outs.append(out)
    _call(q, outs[0], k, outs[1], None, None, None, None, positions, frequencies, interleaved,
          inverse, float(factor))
    return outs[0], outs[1]


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
    like = k
    _heads("k", k, like)
    _heads("v", v, like, k.shape[1])
    for name, c in (("key_cache", key_cache), ("value_cache", value_cache)):
        if c.dim() != 4 or c.shape[2:] != k.shape[1:] or c.shape != key_cache.shape:
            raise ValueError(f"rotary: {name} must be [blocks, page, {k.shape[1]}, {k.shape[2]}]")
        if c.dtype != k.dtype or c.device != k.device:
            raise TypeError(f"rotary: {name} must be {k.dtype} on {k.device}")
        if c.stride(3) != 1 and c.shape[3] > 1:
            raise ValueError(f"rotary: {name} needs a unit head-dim stride")
    if slots.dim() != 1 or slots.shape[0] != k.shape[0] or slots.dtype != torch.int64 \
            or slots.device != k.device:
        raise ValueError(f"rotary: slots must be int64 [tokens] on {k.device}")
    if q is not None:
        _heads("q", q, like)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _heads("q_out", q_out, q, q.shape[1])
    else:
        q_out = None
    _call(q, q_out, k, None, v, key_cache, value_cache, slots, positions, frequencies,
          interleaved, False, float(factor))
    return q_out


__all__ = ["rotary_frequencies", "rotary_embed", "rotary_store"]
