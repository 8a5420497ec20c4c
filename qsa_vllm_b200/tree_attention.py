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
    kind, dev = q.dtype, q.get_device()
    if kind not in _DTYPES:
        raise TypeError(f"{what}: q must be bfloat16 or float16, got {kind}")
    shape = q.shape
    if len(shape) != 3 or (q.stride(2) != 1 and shape[2] > 1):
        raise ValueError(f"{what}: q must be [rows, heads, dim] with a unit dim stride")
    first = caches[0][1].shape
    for name, c in caches:
        if c.dtype != kind or c.get_device() != dev:
            raise TypeError(f"{what}: {name} must be {kind} on {q.device}")
        if len(first) != 4 or c.shape != first or first[3] != shape[2]:
            raise ValueError(f"{what}: {name} must be [blocks, page, kv_heads, {shape[2]}]")
        if c.stride(3) != 1 and first[3] > 1:
            raise ValueError(f"{what}: {name} needs a unit head-dim stride")
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens),
                    ("query_start_loc", query_start_loc)):
        if t.dtype != torch.int32 or t.get_device() != dev:
            raise TypeError(f"{what}: {name} must be int32 on {q.device}")
        if t.dim() == 0 or (t.stride(-1) != 1 and t.shape[-1] > 1):
            raise ValueError(f"{what}: {name} needs a unit stride over its last dim")
    table, lens, start = block_table.shape, seq_lens.shape, query_start_loc.shape
    if len(table) != 2 or len(lens) != 1 or lens[0] != table[0] or len(start) != 1 \
            or start[0] != table[0] + 1:
        raise ValueError(f"{what}: block_table [B, width], seq_lens [B] and query_start_loc "
                         "[B + 1] expected")
    if tree_mask is not None:
        if tree_mask.dtype not in (torch.bool, torch.uint8) or tree_mask.get_device() != dev:
            raise TypeError(f"{what}: tree_mask must be bool or uint8 on {q.device}")
        mask = tree_mask.shape
        if len(mask) != 2 or mask[0] != shape[0] or (tree_mask.stride(1) != 1 and mask[1] > 1):
            raise ValueError(f"{what}: tree_mask must be [rows, drafted tokens] with a unit "
                             "stride over the tokens")
    if max_query_len < 1:
        raise ValueError(f"{what}: max_query_len must be positive")


def check_lse(what: str, lse, q) -> None:
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] \
            or lse.get_device() != q.get_device() or (lse.stride(1) != 1 and lse.shape[1] > 1):
        raise ValueError(f"{what}: lse must be float32 [rows, heads] with a unit head stride")


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
    requests, width = block_table.shape
    blocks, page, hkv, _ = k_cache.shape
    qs, ks, vs, os = q.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    lib = _lib.load_library()
    with _lib.on_device(index):
        need = lib.qsa_tree_attention_workspace_bytes(rows, requests, hq, hkv, d, max_query_len)
        if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        status = lib.qsa_tree_attention(
            q.data_ptr(), qs[0], qs[1], rows, hq, d, _DTYPES[q.dtype],
            k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
            blocks, page, hkv, block_table.data_ptr(), block_table.stride(0), width, requests,
            seq_lens.data_ptr(), query_start_loc.data_ptr(),
            *mask_arguments(tree_mask, seq_lens), max_query_len,
            d ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1],
            None if lse is None else lse.data_ptr(), 0 if lse is None else lse.stride(0),
            workspace.data_ptr() if need else None, need, _lib.raw_stream(index))
    if status:
        _lib.check(status, what)
    return out


__all__ = ["tree_paged_attention", "tree_attention_workspace_bytes"]
