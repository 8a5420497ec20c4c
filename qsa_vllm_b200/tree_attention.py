"""Attention of a tree of drafted tokens over the paged cache.

``tree_paged_attention`` verifies speculative drafts: each request brings a few rows whose keys
and values are already in its pages (``rotary_store`` or ``qsa_prepare`` wrote them), every row
attends the request's whole context, and among the drafted tokens a mask says who sees whom.
Without a mask the rows are a chain, which makes it a dense decode step (one row) or a causal
prompt chunk.  The log-sum-exp it can leave is what ``accumulate_attention_weights`` reads.
"""

from __future__ import annotations

import torch

from . import _lib
from .qsa import aligned_head_rows

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def tree_attention_workspace_bytes(rows: int, num_requests: int, num_q_heads: int,
                                   num_kv_heads: int, head_dim: int, max_query_len: int) -> int:
    return int(_lib.load_library().qsa_tree_attention_workspace_bytes(
        rows, num_requests, num_q_heads, num_kv_heads, head_dim, max_query_len))


def check_tree_arguments(what: str, q, k_cache, v_cache, block_table, seq_lens, query_start_loc,
                         tree_mask, max_query_len) -> tuple:
    """Types, shapes, strides and devices of what the tree operators share (v_cache may be
    None).  Returns the C arguments of the keys' cache and of the tables, the value cache's, and
    the mask's."""
    kind, dev, shape = q.dtype, q.get_device(), q.shape
    if kind not in _DTYPES:
        raise TypeError(f"{what}: q must be bfloat16 or float16, got {kind}")
    if len(shape) != 3 or (q.stride(2) != 1 and shape[2] > 1):
        raise ValueError(f"{what}: q must be [rows, heads, dim] with a unit dim stride")
    cache, ks = k_cache.shape, k_cache.stride()
    if k_cache.dtype != kind or k_cache.get_device() != dev:
        raise TypeError(f"{what}: k_cache must be {kind} on {q.device}")
    if len(cache) != 4 or cache[3] != shape[2] or (ks[3] != 1 and shape[2] > 1):
        raise ValueError(f"{what}: k_cache must be [blocks, page, kv_heads, {shape[2]}] with a "
                         "unit head-dim stride")
    values = ()
    if v_cache is not None:
        vs = v_cache.stride()
        if v_cache.dtype != kind or v_cache.get_device() != dev:
            raise TypeError(f"{what}: v_cache must be {kind} on {q.device}")
        if v_cache.shape != cache or (vs[3] != 1 and shape[2] > 1):
            raise ValueError(f"{what}: v_cache must be like k_cache, with a unit head-dim stride")
        values = (v_cache.data_ptr(), vs[0], vs[1], vs[2])
    table, lens, start = block_table.shape, seq_lens.shape, query_start_loc.shape
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens),
                    ("query_start_loc", query_start_loc)):
        if t.dtype != torch.int32 or t.get_device() != dev:
            raise TypeError(f"{what}: {name} must be int32 on {q.device}")
    if len(table) != 2 or len(lens) != 1 or lens[0] != table[0] or len(start) != 1 \
            or start[0] != table[0] + 1:
        raise ValueError(f"{what}: block_table [B, width], seq_lens [B] and query_start_loc "
                         "[B + 1] expected")
    row, unit = block_table.stride()
    if (unit != 1 and table[1] > 1) or (seq_lens.stride(0) != 1 and lens[0] > 1) \
            or query_start_loc.stride(0) != 1:
        raise ValueError(f"{what}: block_table, seq_lens and query_start_loc need a unit stride "
                         "over their last dim")
    mask = (None, 0, 0)
    if tree_mask is not None:
        if tree_mask.dtype not in (torch.bool, torch.uint8) or tree_mask.get_device() != dev:
            raise TypeError(f"{what}: tree_mask must be bool or uint8 on {q.device}")
        size, steps = tree_mask.shape, tree_mask.stride()
        if len(size) != 2 or size[0] != shape[0] or (steps[1] != 1 and size[1] > 1):
            raise ValueError(f"{what}: tree_mask must be [rows, drafted tokens] with a unit "
                             "stride over the tokens")
        # A mask without columns has no storage, but it is not the chain that a null pointer
        # means: any pointer does, as none of it is read.
        mask = (tree_mask.data_ptr() or seq_lens.data_ptr(), steps[0], size[1])
    if max_query_len < 1:
        raise ValueError(f"{what}: max_query_len must be positive")
    return ((k_cache.data_ptr(), ks[0], ks[1], ks[2]), values,
            (cache[0], cache[1], cache[2], block_table.data_ptr(), row, table[1], table[0],
             seq_lens.data_ptr(), query_start_loc.data_ptr(), *mask, max_query_len))


def check_lse(what: str, lse, q) -> None:
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] \
            or lse.get_device() != q.get_device() or (lse.stride(1) != 1 and lse.shape[1] > 1):
        raise ValueError(f"{what}: lse must be float32 [rows, heads] with a unit head stride")


def tree_paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         block_table: torch.Tensor, seq_lens: torch.Tensor,
                         query_start_loc: torch.Tensor, out: torch.Tensor | None = None, *,
                         max_query_len: int, tree_mask: torch.Tensor | None = None,
                         scale: float | None = None, lse: torch.Tensor | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q.K^T + mask).V over every cached token of each row's request.

    q: bf16 or fp16 ``[rows, H_q, d]``, the rows of request ``b`` being ``query_start_loc[b] ..
    query_start_loc[b+1] - 1`` (int32 ``[B + 1]``); k_cache / v_cache: ``[blocks, page, H_kv,
    d]`` of the same type; block_table: int32 ``[B, width]``; seq_lens: int32 ``[B]`` cached
    tokens, the request's rows' own tokens the last of them.  tree_mask: bool or uint8 ``[rows,
    tokens]``, nonzero where the row sees its request's drafted token (itself too); None for a
    chain.  scale: ``d ** -0.5`` where None.  lse: fp32 ``[rows, H_q]``, receives the natural
    log-sum-exp.  max_query_len: the longest request's rows (a host number that sizes the work
    split, and through it the order of 32-bit sums); 1 in a batch of single rows beside a few
    prompt chunks, which would all be split as the chunks are (63 rows and a chunk of 512 over
    8192 tokens: 259 us with 1, 1026 with 512).  Rows that see nothing give 0 and -inf; rows of no request are left
    as they are.
    workspace: uint8, at least ``tree_attention_workspace_bytes(...)``; allocated where None."""
    what = "tree_paged_attention"
    keys, values, tables = check_tree_arguments(what, q, k_cache, v_cache, block_table, seq_lens,
                                                query_start_loc, tree_mask, max_query_len)
    rows, hq, d = shape = q.shape
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    elif out.shape != shape or out.dtype != q.dtype or out.get_device() != q.get_device() \
            or (out.stride(2) != 1 and d > 1):
        raise ValueError(f"{what}: out must be like q, with a unit dim stride")
    if lse is not None:
        check_lse(what, lse, q)
    index = _lib.ready(q)
    if not rows:
        return out
    q = aligned_head_rows(q)
    qs, os = q.stride(), out.stride()
    lib = _lib.load_library()
    with _lib.on_device(index):
        need = lib.qsa_tree_attention_workspace_bytes(rows, tables[6], hq, tables[2], d,
                                                      max_query_len)
        workspace = _lib.workspace_of(what, workspace, need, q)
        status = lib.qsa_tree_attention(
            q.data_ptr(), qs[0], qs[1], rows, hq, d, _DTYPES[q.dtype], *keys, *values, *tables,
            d ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1],
            None if lse is None else lse.data_ptr(), 0 if lse is None else lse.stride(0),
            workspace.data_ptr() if need else None, need, _lib.raw_stream(index))
    if status:
        _lib.check(status, what)
    return out


__all__ = ["tree_paged_attention", "tree_attention_workspace_bytes"]
