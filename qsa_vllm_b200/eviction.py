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

These are operators for layers with dense attention.  The cache of a QSA layer must not be passed:
only its keys and values would move, while its compressed index keys and its ring of raw ones,
which ``qsa_prepare`` wrote, would go on describing the tokens that were there before.  Its sparse
attention leaves no log-sum-exp over all tokens either.
"""

from __future__ import annotations

import torch

from . import _lib
from .qsa import aligned_head_rows
from .tree_attention import check_lse, check_tree_arguments

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NO_COLUMNS = 16


def _caches(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple:
    """The arguments that describe two caches, once they are found in order."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{what}: the caches must be [blocks, page, kv_heads, dim], both alike")
    kind = _DTYPES.get(k_cache.dtype)
    if kind is None or v_cache.dtype != k_cache.dtype:
        raise TypeError(f"{what}: the caches must be bfloat16, float16 or float32, both alike")
    if v_cache.get_device() != k_cache.get_device():
        raise TypeError(f"{what}: v_cache must be on {k_cache.device}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and shape[3] > 1:
        raise ValueError(f"{what}: the caches need a unit head-dim stride")
    return (k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
            shape[0], shape[1], shape[2], shape[3], kind)


def _int32(what: str, name: str, t: torch.Tensor, dev: int, *shape) -> None:
    """int32 of this shape (None: any size), with unit stride over its last dim."""
    if t.dtype != torch.int32 or t.get_device() != dev:
        raise TypeError(f"{what}: {name} must be int32 on the caches' device, got {t.dtype} on "
                        f"{t.device}")
    got = t.shape
    if len(got) != len(shape) or any([n is not None and n != m for n, m in zip(shape, got)]):
        want = tuple("any" if n is None else n for n in shape)
        raise ValueError(f"{what}: {name} must be {want}, got {tuple(got)}")
    if got[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: {name} needs a unit stride over its last dim")


def _tables(what: str, dev: int, block_table: torch.Tensor, out_table) -> tuple:
    _int32(what, "block_table", block_table, dev, None, None)
    requests, width = block_table.shape
    if out_table is None:
        return block_table.data_ptr(), block_table.stride(0), width, None, 0, 0
    _int32(what, "out_table", out_table, dev, requests, None)
    # A table without columns has no storage, but it is not the in-place move that a null pointer
    # means: any other pointer does, as none of it is read.
    return (block_table.data_ptr(), block_table.stride(0), width,
            out_table.data_ptr() or _NO_COLUMNS, out_table.stride(0), out_table.shape[1])


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
    ``min(seq_lens[b], capacity, width * page)`` on (past the lengths, the capacity or the block
    table) are not written; tokens on unmapped pages keep their weight."""
    what = "accumulate_attention_weights"
    keys, _, tables = check_tree_arguments(what, q, k_cache, None, block_table, seq_lens,
                                           query_start_loc, tree_mask, max_query_len)
    rows, hq, d = q.shape
    hkv, requests = tables[2], tables[6]
    dev = q.get_device()
    if out is None:
        out = weights
    shape = weights.shape
    if len(shape) != 3 or shape[0] != requests or shape[1] != hkv or out.shape != shape:
        raise ValueError(f"{what}: weights and out must be [{requests}, {hkv}, capacity]")
    ws, os = weights.stride(), out.stride()
    if weights.dtype != torch.float32 or out.dtype != torch.float32 \
            or weights.get_device() != dev or out.get_device() != dev:
        raise TypeError(f"{what}: weights and out must be float32 on {q.device}")
    if (ws[2] != 1 or os[2] != 1) and shape[2] > 1:
        raise ValueError(f"{what}: weights and out need a unit token stride")
    check_lse(what, lse, q)
    if row_factors is not None and (row_factors.dtype != torch.float32 or row_factors.dim() != 1
                                    or row_factors.shape[0] != rows
                                    or row_factors.get_device() != dev):
        raise ValueError(f"{what}: row_factors must be float32 [rows]")
    _lib.ready(q)
    if rows:
        q = aligned_head_rows(q)
    qs = q.stride()
    with _lib.on_device(dev):
        status = _lib.load_library().qsa_attention_weights(
            q.data_ptr(), qs[0], qs[1], rows, hq, d, _DTYPES[q.dtype], *keys, *tables,
            d ** -0.5 if scale is None else scale, lse.data_ptr(), lse.stride(0),
            None if row_factors is None else row_factors.data_ptr(),
            0 if row_factors is None else row_factors.stride(0),
            weights.data_ptr(), ws[0], ws[1], out.data_ptr(), os[0], os[1], shape[2],
            _lib.raw_stream(dev))
    if status:
        _lib.check(status, what)
    return out


def cache_compact(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  indices: torch.Tensor, starts: torch.Tensor | None = None, *,
                  out_table: torch.Tensor | None = None) -> None:
    """Moves the K/V rows of cached token ``indices[b, (h,) j]`` to token ``starts[b] + j``.

    k_cache / v_cache: ``[blocks, page, H_kv, d]``; block_table, out_table: int32 ``[B, width]``;
    indices: int32 ``[B, n]`` or ``[B, H_kv, n]``, negative entries move nothing; starts: int32
    ``[B]`` (0 where None).  Without ``out_table`` the move is in place: lists ascend, no token
    moves to a higher number, and no two requests share a page.  With it, destinations are pages
    that the call does not read.  Entries outside the tables or on unmapped pages are skipped and
    set the device error word."""
    what = "cache_compact"
    caches = _caches(what, k_cache, v_cache)
    dev = k_cache.get_device()
    tables = _tables(what, dev, block_table, out_table)
    requests = block_table.shape[0]
    if indices.dim() == 3:
        _int32(what, "indices", indices, dev, requests, caches[10], None)
        head_stride = indices.stride(1)
    else:
        _int32(what, "indices", indices, dev, requests, None)
        head_stride = 0
    if starts is not None:
        _int32(what, "starts", starts, dev, requests)
    _lib.ready(k_cache)
    with _lib.on_device(dev):
        status = _lib.load_library().qsa_cache_compact(
            *caches, *tables, requests, indices.data_ptr(), indices.stride(0), head_stride,
            indices.shape[-1], None if starts is None else starts.data_ptr(),
            _lib.raw_stream(dev))
    if status:
        _lib.check(status, what)


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
    move to tokens ``0 .. budget - 1`` in place (no two requests may share a page then), or to
    the pages of ``out_table``, which the call does not read; their weights
    to the front of ``weights_out`` (``weights`` itself where None), with zeros up to the old
    length.  kept: int32 ``[B, heads of weights, budget]``, the old token numbers, -1 behind the
    last; lengths: int32 ``[B]``.

    Refused with :class:`QSAError`: weights whose (request, head) rows are not evenly spaced (a
    slice of the heads of more), and more than 524288 tokens to choose from (``capacity - sinks
    - recent``, where the budget is below the capacity).  Kept tokens outside a table or on
    unmapped pages are not moved and set the device error word."""
    what = "cache_evict"
    caches = _caches(what, k_cache, v_cache)
    dev = k_cache.get_device()
    tables = _tables(what, dev, block_table, out_table)
    requests, heads = block_table.shape[0], caches[10]
    _int32(what, "seq_lens", seq_lens, dev, requests)
    if weights_out is None:
        weights_out = weights
    shape = weights.shape
    if len(shape) != 3 or shape[0] != requests or shape[1] not in (1, heads) \
            or weights_out.shape != shape:
        raise ValueError(f"{what}: weights and weights_out must be [{requests}, {heads} or 1, "
                         "capacity]")
    if weights.dtype != torch.float32 or weights_out.dtype != torch.float32 \
            or weights.get_device() != dev or weights_out.get_device() != dev:
        raise TypeError(f"{what}: weights and weights_out must be float32 on {k_cache.device}")
    ws, os = weights.stride(), weights_out.stride()
    if (ws[2] != 1 or os[2] != 1) and shape[2] > 1:
        raise ValueError(f"{what}: weights and weights_out need a unit token stride")
    if sinks < 0 or recent < 0 or budget < sinks + recent:
        raise ValueError(f"{what}: sinks {sinks} + recent {recent} must fit the budget {budget}")
    if kept is None:
        kept = torch.empty(requests, shape[1], budget, dtype=torch.int32, device=k_cache.device)
    else:
        _int32(what, "kept", kept, dev, requests, shape[1], budget)
        if not kept.is_contiguous():
            raise ValueError(f"{what}: kept must be contiguous")
    lengths = torch.empty(requests, dtype=torch.int32, device=k_cache.device)
    _lib.ready(k_cache)
    if not requests:
        return kept, lengths
    lib = _lib.load_library()
    need = lib.qsa_cache_evict_workspace_bytes(requests, shape[1], budget, sinks, recent)
    workspace = _lib.workspace_of(what, workspace, need, k_cache)
    with _lib.on_device(dev):
        status = lib.qsa_cache_evict(
            weights.data_ptr(), ws[0], ws[1], shape[1], shape[2], seq_lens.data_ptr(), requests,
            budget, sinks, recent, *caches, *tables, weights_out.data_ptr(), os[0], os[1],
            kept.data_ptr(), lengths.data_ptr(), workspace.data_ptr(), need,
            _lib.raw_stream(dev))
    if status:
        _lib.check(status, what)
    return kept, lengths


__all__ = ["accumulate_attention_weights", "cache_compact", "cache_evict", "cache_evict_workspace_bytes"]
