"""Keeping a paged cache small: the attention weight each cached token has received, the
eviction that goes by it, and the compaction of cached tokens.

* ``accumulate_attention_weights`` adds up, per KV head and cached token, the probabilities
  that chosen rows gave it, from the log-sum-exp that ``tree_paged_attention`` left;
* ``cache_evict`` keeps, per request and KV head, the first ``sinks`` tokens, the last
  ``recent`` ones and the heaviest of the rest, ``budget`` in all, and moves them to the front
  of the request's pages (or to other pages) in their order;
* ``cache_compact`` moves listed tokens to consecutive places: the commit of an accepted path
  of drafted tokens, or a context without a passage.

Attention does not depend on the order or the numbering of cached tokens: keys keep the rotary
positions they were stored with.  After an eviction the tokens' numbers are new ones, so the
caller goes on counting positions for itself, frees the pages behind the new lengths, and
appends at the new length.
"""

from __future__ import annotations

import torch

from . import _lib
from .qsa import aligned_head_rows
from .tree_attention import check_tree_arguments, mask_arguments

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _caches(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.shape != k_cache.shape:
            raise ValueError(f"{what}: {name} must be [blocks, page, kv_heads, dim], both alike")
        if c.dtype not in _DTYPES or c.dtype != k_cache.dtype:
            raise TypeError(f"{what}: {name} must be bfloat16, float16 or float32, both alike")
        if c.device != k_cache.device:
            raise TypeError(f"{what}: {name} must be on {k_cache.device}")
        if c.stride(3) != 1 and c.shape[3] > 1:
            raise ValueError(f"{what}: {name} needs a unit head-dim stride")


def _int32(what: str, name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> None:
    """int32 of this shape (None: any size), with unit stride over its last dim."""
    if t.dtype != torch.int32 or t.device != device:
        raise TypeError(f"{what}: {name} must be int32 on {device}, got {t.dtype} on {t.device}")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        want = tuple("any" if n is None else n for n in shape)
        raise ValueError(f"{what}: {name} must be {want}, got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: {name} needs a unit stride over its last dim")


def _cache_args(k_cache, v_cache, block_table, out_table) -> tuple:
    out = (None, 0, 0) if out_table is None else (out_table.data_ptr(), out_table.stride(0),
                                                  out_table.shape[1])
    return (k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            k_cache.shape[0], k_cache.shape[1], k_cache.shape[2], k_cache.shape[3],
            _DTYPES[k_cache.dtype], block_table.data_ptr(), block_table.stride(0),
            block_table.shape[1], *out)


def accumulate_attention_weights(
        q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor,
        seq_lens: torch.Tensor, query_start_loc: torch.Tensor, lse: torch.Tensor,
        weights: torch.Tensor, out: torch.Tensor | None = None, *, max_query_len: int,
        tree_mask: torch.Tensor | None = None, row_factors: torch.Tensor | None = None,
        scale: float | None = None) -> torch.Tensor:
    """``out[b, h, t] = weights[b, h, t] + sum_i row_factors[i] sum_g exp(scale q_ig.k_t -
    lse_ig)`` over request b's rows i that see token t and the query heads g of KV head h.

    Arguments as in ``tree_paged_attention``, whose ``lse`` this takes.  row_factors: fp32
    ``[rows]``, 1 where None; 0 leaves a row out (a rejected draft).  weights, out: fp32 ``[B,
    H_kv, capacity]``; out is weights itself (in place) where None.  Tokens from
    ``min(seq_lens[b], capacity)`` on are not written."""
    what = "accumulate_attention_weights"
    max_query_len = int(max_query_len)
    check_tree_arguments(what, q, (("k_cache", k_cache),), block_table, seq_lens,
                         query_start_loc, tree_mask, max_query_len)
    dev = q.device
    rows, hq, d = q.shape
    requests, hkv = block_table.shape[0], k_cache.shape[2]
    if out is None:
        out = weights
    for name, w in (("weights", weights), ("out", out)):
        if w.dtype != torch.float32 or w.device != dev:
            raise TypeError(f"{what}: {name} must be float32 on {dev}")
        if w.dim() != 3 or w.shape[:2] != (requests, hkv) or w.shape != weights.shape \
                or (w.shape[2] > 1 and w.stride(2) != 1):
            raise ValueError(f"{what}: {name} must be [{requests}, {hkv}, capacity] with a unit "
                             "token stride")
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] or lse.device != dev \
            or (lse.stride(1) != 1 and hq > 1):
        raise ValueError(f"{what}: lse must be float32 [rows, heads] with a unit head stride")
    if row_factors is not None and (row_factors.dtype != torch.float32
                                    or row_factors.shape != q.shape[:1]
                                    or row_factors.device != dev):
        raise ValueError(f"{what}: row_factors must be float32 [rows]")
    _lib.ensure_device(dev)
    if rows:
        q = aligned_head_rows(q)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().qsa_attention_weights(
            q.data_ptr(), q.stride(0), q.stride(1), rows, hq, d, _DTYPES[q.dtype],
            k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            k_cache.shape[0], k_cache.shape[1], hkv,
            block_table.data_ptr(), block_table.stride(0), block_table.shape[1], requests,
            seq_lens.data_ptr(), query_start_loc.data_ptr(),
            *mask_arguments(tree_mask, seq_lens), max_query_len,
            d ** -0.5 if scale is None else float(scale), lse.data_ptr(), lse.stride(0),
            None if row_factors is None else row_factors.data_ptr(),
            0 if row_factors is None else row_factors.stride(0),
            weights.data_ptr(), weights.stride(0), weights.stride(1),
            out.data_ptr(), out.stride(0), out.stride(1), weights.shape[2],
            _lib.stream_ptr(dev)), what)
    return out


def cache_compact(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  indices: torch.Tensor, starts: torch.Tensor | None = None, *,
                  out_table: torch.Tensor | None = None) -> None:
    """Moves the K/V rows of cached token ``indices[b, (h,) j]`` to token ``starts[b] + j``.

    k_cache / v_cache: ``[blocks, page, H_kv, d]``; block_table, out_table: int32 ``[B, width]``;
    indices: int32 ``[B, n]`` or ``[B, H_kv, n]``, negative entries move nothing; starts: int32
    ``[B]`` (0 where None).  Without ``out_table`` the move is in place: lists ascend, and no
    token moves to a higher number.  With it, destinations are pages that the call does not
    read.  Entries outside the tables or on unmapped pages are skipped and set the device error
    word."""
    what = "cache_compact"
    _caches(what, k_cache, v_cache)
    dev = k_cache.device
    requests = block_table.shape[0]
    _int32(what, "block_table", block_table, (None, None), dev)
    if indices.dim() == 3:
        _int32(what, "indices", indices, (requests, k_cache.shape[2], None), dev)
        head_stride = indices.stride(1)
    else:
        _int32(what, "indices", indices, (requests, None), dev)
        head_stride = 0
    if starts is not None:
        _int32(what, "starts", starts, (requests,), dev)
    if out_table is not None:
        _int32(what, "out_table", out_table, (requests, None), dev)
    _lib.ensure_device(dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().qsa_cache_compact(
            *_cache_args(k_cache, v_cache, block_table, out_table), requests,
            indices.data_ptr(), indices.stride(0), head_stride, indices.shape[-1],
            None if starts is None else starts.data_ptr(), _lib.stream_ptr(dev)), what)


def cache_evict_workspace_bytes(requests: int, list_heads: int, budget: int, sinks: int,
                                recent: int) -> int:
    return int(_lib.load_library().qsa_cache_evict_workspace_bytes(requests, list_heads, budget,
                                                                   sinks, recent))


def cache_evict(weights: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, budget: int, *, sinks: int = 0,
                recent: int = 0, out_table: torch.Tensor | None = None,
                weights_out: torch.Tensor | None = None, kept: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keeps ``budget`` tokens of each request that has more; returns ``(kept, lengths)``.

    weights: fp32 ``[B, H_kv, capacity]`` (or ``[B, 1, capacity]``: one choice for all heads),
    0 or above, as ``accumulate_attention_weights`` leaves them; seq_lens: int32 ``[B]`` cached
    tokens (at most ``capacity`` count), not written.  Kept are the first ``sinks`` tokens, the
    last ``recent`` and the heaviest of the others, ties to the lowest token.  Their K/V rows
    move to tokens ``0 .. budget - 1`` in place, or to the pages of ``out_table``; their weights
    to the front of ``weights_out`` (``weights`` itself where None), with zeros up to the old
    length.  kept: int32 ``[B, heads of weights, budget]``, the old token numbers, -1 behind the
    last; lengths: int32 ``[B]``."""
    what = "cache_evict"
    _caches(what, k_cache, v_cache)
    dev = k_cache.device
    requests, heads = block_table.shape[0], k_cache.shape[2]
    _int32(what, "block_table", block_table, (None, None), dev)
    _int32(what, "seq_lens", seq_lens, (requests,), dev)
    if out_table is not None:
        _int32(what, "out_table", out_table, (requests, None), dev)
    if weights_out is None:
        weights_out = weights
    for name, w in (("weights", weights), ("weights_out", weights_out)):
        if w.dtype != torch.float32 or w.device != dev:
            raise TypeError(f"{what}: {name} must be float32 on {dev}")
        if w.dim() != 3 or w.shape[0] != requests or w.shape[1] not in (1, heads) \
                or w.shape != weights.shape:
            raise ValueError(f"{what}: {name} must be [{requests}, {heads} or 1, capacity]")
        if w.shape[2] > 1 and w.stride(2) != 1:
            raise ValueError(f"{what}: {name} needs a unit token stride")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if sinks < 0 or recent < 0 or budget < sinks + recent:
        raise ValueError(f"{what}: sinks {sinks} + recent {recent} must fit the budget {budget}")
    if kept is None:
        kept = torch.empty(requests, weights.shape[1], budget, dtype=torch.int32, device=dev)
    else:
        _int32(what, "kept", kept, (requests, weights.shape[1], budget), dev)
        if not kept.is_contiguous():
            raise ValueError(f"{what}: kept must be contiguous")
    lengths = torch.empty(requests, dtype=torch.int32, device=dev)
    _lib.ensure_device(dev)
    if not requests:
        return kept, lengths
    need = cache_evict_workspace_bytes(requests, weights.shape[1], budget, sinks, recent)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().qsa_cache_evict(
            weights.data_ptr(), weights.stride(0), weights.stride(1), weights.shape[1],
            weights.shape[2], seq_lens.data_ptr(), requests, budget, sinks, recent,
            *_cache_args(k_cache, v_cache, block_table, out_table), weights_out.data_ptr(),
            weights_out.stride(0), weights_out.stride(1), kept.data_ptr(), lengths.data_ptr(),
            workspace.data_ptr(), need, _lib.stream_ptr(dev)), what)
    return kept, lengths


__all__ = ["accumulate_attention_weights", "cache_compact", "cache_evict", "cache_evict_workspace_bytes"]
