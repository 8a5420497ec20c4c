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


def check_tree_arguments(what: str, q, caches, block_table, seq_lens, query_start_loc,
                         tree_mask, max_query_len) -> None:
    """Types, shapes, strides and devices of what the tree operators share."""
    dev = q.device
    if q.dtype not in _DTYPES:
        raise TypeError(f"{what}: q must be bfloat16 or float16, got {q.dtype}")
    if q.dim() != 3 or (q.stride(2) != 1 and q.shape[2] > 1):
        raise ValueError(f"{what}: q must be [rows, heads, dim] with a unit dim stride")
    for name, c in caches:
        if c.dtype != q.dtype or c.device != dev:
            raise TypeError(f"{what}: {name} must be {q.dtype} on {dev}")
        if c.dim() != 4 or c.shape != caches[0][1].shape or c.shape[3] != q.shape[2]:
            raise ValueError(f"{what}: {name} must be [blocks, page, kv_heads, {q.shape[2]}]")
        if c.stride(3) != 1 and c.shape[3] > 1:
            raise ValueError(f"{what}: {name} needs a unit head-dim stride")
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens),
                    ("query_start_loc", query_start_loc)):
        if t.dtype != torch.int32 or t.device != dev:
            raise TypeError(f"{what}: {name} must be int32 on {dev}")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{what}: {name} needs a unit stride over its last dim")
    if block_table.dim() != 2 or seq_lens.shape != block_table.shape[:1] \
            or query_start_loc.dim() != 1 \
            or query_start_loc.shape[0] != block_table.shape[0] + 1:
        raise ValueError(f"{what}: block_table [B, width], seq_lens [B] and query_start_loc "
                         "[B + 1] expected")
    if tree_mask is not None:
        if tree_mask.dtype not in (torch.bool, torch.uint8) or tree_mask.device != dev:
            raise TypeError(f"{what}: tree_mask must be bool or uint8 on {dev}")
        if tree_mask.dim() != 2 or tree_mask.shape[0] != q.shape[0] \
                or (tree_mask.stride(1) != 1 and tree_mask.shape[1] > 1):
            raise ValueError(f"{what}: tree_mask must be [rows, drafted tokens] with a unit "
                             "stride over the tokens")
    if max_query_len < 1:
        raise ValueError(f"{what}: max_query_len must be positive")


def mask_arguments(tree_mask: torch.Tensor | None, any_tensor: torch.Tensor) -> tuple:
    """Pointer, row stride and width.  A mask without columns has no storage, but it is not
    the chain that a null pointer means: any pointer does, as none of it is read."""
    if tree_mask is None:
        return None, 0, 0
    return (tree_mask.data_ptr() or any_tensor.data_ptr(), tree_mask.stride(0),
            tree_mask.shape[1])


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
    split).  Rows that see nothing give 0 and -inf; rows of no request are left as they are.
    workspace: uint8, at least ``tree_attention_workspace_bytes(...)``; allocated where None."""
    what = "tree_paged_attention"
    max_query_len = int(max_query_len)
    check_tree_arguments(what, q, (("k_cache", k_cache), ("v_cache", v_cache)), block_table,
                         seq_lens, query_start_loc, tree_mask, max_query_len)
    dev = q.device
    rows, hq, d = q.shape
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev \
            or (out.stride(2) != 1 and d > 1):
        raise ValueError(f"{what}: out must be like q, with a unit dim stride")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2]
                            or lse.device != dev or (lse.stride(1) != 1 and hq > 1)):
        raise ValueError(f"{what}: lse must be float32 [rows, heads] with a unit head stride")
    _lib.ensure_device(dev)
    if not rows:
        return out
    q = aligned_head_rows(q)
    requests, hkv = block_table.shape[0], k_cache.shape[2]
    need = tree_attention_workspace_bytes(rows, requests, hq, hkv, d, max_query_len)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().qsa_tree_attention(
            q.data_ptr(), q.stride(0), q.stride(1), rows, hq, d, _DTYPES[q.dtype],
            k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            k_cache.shape[0], k_cache.shape[1], hkv,
            block_table.data_ptr(), block_table.stride(0), block_table.shape[1], requests,
            seq_lens.data_ptr(), query_start_loc.data_ptr(),
            *mask_arguments(tree_mask, seq_lens), max_query_len,
            d ** -0.5 if scale is None else float(scale),
            out.data_ptr(), out.stride(0), out.stride(1),
            None if lse is None else lse.data_ptr(), 0 if lse is None else lse.stride(0),
            workspace.data_ptr() if need else None, need, _lib.stream_ptr(dev)), what)
    return out


__all__ = ["tree_paged_attention", "tree_attention_workspace_bytes"]
