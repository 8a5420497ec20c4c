"""What the rotary, tree attention and eviction entry points refuse, and host-side helpers
(no GPU: every refusal comes before a device is touched)."""

import math

import pytest
import torch

BF16 = torch.bfloat16


def test_rotary_frequencies():
    from qsa_vllm_b200.rotary import rotary_frequencies
    f, factor = rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and factor == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    g, _ = rotary_frequencies(8, 10000.0, scaling="linear", scaling_factor=4.0)
    assert torch.equal(g, f / 4)
    n, _ = rotary_frequencies(8, 10000.0, scaling="ntk", scaling_factor=4.0)
    assert n[0] == 1.0 and math.isclose(n[-1], f[-1] / 4, rel_tol=1e-12)
    y, factor = rotary_frequencies(64, 10000.0, scaling="yarn", scaling_factor=4.0,
                                   original_length=4096)
    f, _ = rotary_frequencies(64, 10000.0)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32])
    assert torch.equal(y[turns <= 1], f[turns <= 1] / 4)
    assert ((y >= f / 4) & (y <= f)).all() and math.isclose(factor, 0.1 * math.log(4) + 1)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=8, scaling_factor=0.5),
                dict(rotary_dim=8, base=0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_rotary_refusals():
    from qsa_vllm_b200 import QSAError
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies, rotary_store
    f, _ = rotary_frequencies(64)
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    pos = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError):
        rotary_embed(None, None, pos, f)
    with pytest.raises(ValueError, match="positions"):
        rotary_embed(q, k, pos[:2], f)
    with pytest.raises(ValueError, match="positions"):
        rotary_embed(q, k, pos.to(torch.int32), f)
    with pytest.raises(TypeError, match="frequencies"):
        rotary_embed(q, k, pos, f.float())
    with pytest.raises(ValueError, match="frequencies"):
        rotary_embed(q[..., :32], None, pos, f)
    with pytest.raises(TypeError):
        rotary_embed(q, k.float(), pos, f)
    with pytest.raises(TypeError):
        rotary_embed(q.double(), None, pos, f)
    with pytest.raises(ValueError):
        rotary_embed(q, k[:2], pos, f)
    with pytest.raises(ValueError, match="stride"):
        rotary_embed(q.transpose(1, 2).contiguous().transpose(1, 2), None, pos, f)
    with pytest.raises(ValueError):
        rotary_embed(q, k, pos, f, q_out=k)
    cache = torch.zeros(2, 16, 2, 64, dtype=BF16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="slots"):
        rotary_store(q, k, k, pos, f, cache, cache, slots[:2])
    with pytest.raises(ValueError, match="value_cache"):
        rotary_store(q, k, k, pos, f, cache, cache[:1], slots)
    with pytest.raises(TypeError):
        rotary_store(q, k, k, pos, f, cache.half(), cache.half(), slots)
    # a CPU tensor that passes every check is refused by device
    with pytest.raises(QSAError):
        rotary_embed(q, k, pos, f)


def test_rotary_c_abi_refusals():
    from qsa_vllm_b200 import _lib
    lib = _lib.load_library()

    def call(tokens=1, q=4096, hq=1, hkv=0, dim=64, rot=64, dtype=0, page=16, slots=None, pos=4096):
        return lib.qsa_rotary(q, 64, 64, hq, q, 64, 64, None, 0, 0, hkv, None, 0, 0, None, 0, 0,
                              None, 0, 0, 0, None, 0, 0, 0, 1, page, slots, 1, tokens, dim, pos, 1,
                              4096, rot, 1.0, 0, 0, dtype, None)
    assert call(tokens=0) == 0 and call(hq=0) == 0
    for bad, status, word in (
            (dict(tokens=-1), 1, b"negative"), (dict(dtype=3), 1, b"dtype"),
            (dict(dim=0, rot=0), 2, b"head_dim"), (dict(dim=1026), 2, b"head_dim"),
            (dict(rot=3), 1, b"rotary"), (dict(rot=66), 1, b"rotary"), (dict(q=None), 1, b"null"),
            (dict(pos=None), 1, b"null"), (dict(hkv=1), 1, b"null"), (dict(q=4097), 1, b"aligned"),
            (dict(hq=70000), 2, b"heads")):
        assert call(**bad) == status and word in lib.qsa_last_error(), bad


def _cache(requests=2, page=16, hkv=2, d=64, dtype=BF16):
    kv = torch.zeros(8, page, hkv, 2 * d, dtype=dtype)
    return kv[..., :d], kv[..., d:], torch.zeros(requests, 4, dtype=torch.int32)


def test_compact_refusals():
    from qsa_vllm_b200 import QSAError
    from qsa_vllm_b200.eviction import cache_compact
    k, v, table = _cache()
    idx = torch.zeros(2, 3, dtype=torch.int32)
    for args, err in (((k[0], v[0], table, idx), ValueError), ((k, v.float(), table, idx), TypeError),
                      ((k, v, table.long(), idx), TypeError), ((k, v, table, idx.long()), TypeError),
                      ((k, v, table, idx[:1]), ValueError),
                      ((k, v, table, idx[:, None].expand(2, 3, 3)), ValueError),
                      ((k, v, table, idx.t().contiguous().t()), ValueError),
                      ((k, v, table, idx, idx[:, 0].long()), TypeError),
                      ((k, v, table, idx, torch.zeros(3, dtype=torch.int32)), ValueError),
                      ((k.double(), v.double(), table, idx), TypeError)):
        with pytest.raises(err):
            cache_compact(*args)
    with pytest.raises(ValueError, match="out_table"):
        cache_compact(k, v, table, idx, out_table=table[:1])
    with pytest.raises(QSAError):
        cache_compact(k, v, table, idx)


def test_evict_refusals():
    from qsa_vllm_b200 import QSAError
    from qsa_vllm_b200.eviction import cache_evict, cache_evict_workspace_bytes
    k, v, table = _cache()
    w, seq = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)

    def call(err, w=w, seq=seq, budget=16, match=None, **more):
        with pytest.raises(err, match=match):
            cache_evict(w, seq, table, k, v, budget, **more)
    call(TypeError, w=w.double())
    call(ValueError, w=w[0])
    call(ValueError, w=torch.zeros(2, 3, 64))
    call(ValueError, w=w.transpose(1, 2).contiguous().transpose(1, 2))
    call(ValueError, weights_out=torch.zeros(2, 2, 63))
    call(TypeError, seq=seq.long())
    call(ValueError, seq=seq[:1])
    call(ValueError, sinks=10, recent=7)
    call(ValueError, sinks=-1)
    call(ValueError, kept=torch.zeros(2, 2, 15, dtype=torch.int32))
    call(QSAError)
    assert cache_evict_workspace_bytes(0, 2, 16, 0, 0) == 0
    assert cache_evict_workspace_bytes(2, 2, 16, 10, 7) == 0
    assert cache_evict_workspace_bytes(2, 2, 16, 2, 4) == 256 + 2 * 2 * 10 * 4


def test_cache_move_c_abi_refusals():
    from qsa_vllm_b200 import _lib
    lib = _lib.load_library()

    def compact(k=4096, page=16, heads=2, dim=64, dtype=0, requests=2, idx=4096, n=3, table=4096):
        return lib.qsa_cache_compact(k, 1, 1, 64, 4096, 64, 64, 64, 8, page, heads, dim, dtype,
                                     table, 4, 4, None, 0, 0, requests, idx, 3, 0, n, None, None)
    assert compact(requests=0) == 0 and compact(n=0) == 0
    for bad, status, word in (
            (dict(k=None), 1, b"null"), (dict(idx=None), 1, b"null"), (dict(table=None), 1, b"null"),
            (dict(page=0), 1, b"sizes"), (dict(heads=0), 1, b"sizes"), (dict(dim=-1), 1, b"sizes"),
            (dict(dtype=7), 1, b"dtype"), (dict(n=-1), 1, b"count"), (dict(k=4097), 1, b"aligned"),
            (dict(requests=65536), 2, b"65535"), (dict(dim=4096), 2, b"units")):
        assert compact(**bad) == status and word in lib.qsa_last_error(), bad

    def evict(w=4096, heads=2, cap=64, budget=16, sinks=2, recent=4, stride=128, ws=4096, n=1 << 20):
        return lib.qsa_cache_evict(w, stride, 64, heads, cap, 4096, 2, budget, sinks, recent, 4096,
                                   64, 64, 64, 4096, 64, 64, 64, 8, 16, 2, 64, 0, 4096, 4, 4, None,
                                   0, 0, 4096, 128, 64, 4096, 4096, ws, n, None)
    for bad, status, word in (
            (dict(w=None), 1, b"null"), (dict(heads=3), 1, b"heads"), (dict(budget=5), 1, b"budget"),
            (dict(budget=-1), 1, b"budget"), (dict(stride=100), 1, b"evenly"),
            (dict(cap=1 << 20, heads=1, stride=1 << 20), 2, b"choose"),
            (dict(ws=None), 3, b"workspace"), (dict(n=100), 3, b"workspace"),
            (dict(ws=4100), 1, b"aligned"), (dict(cap=65, heads=1, stride=64), 1, b"stride")):
        assert evict(**bad) == status and word in lib.qsa_last_error(), bad


def _tree(rows=5, hq=4, hkv=2, d=64, dtype=BF16):
    k, v, table = _cache(hkv=hkv, d=d, dtype=dtype)
    return dict(q=torch.zeros(rows, hq, d, dtype=dtype), k_cache=k, v_cache=v, block_table=table,
                seq_lens=torch.zeros(2, dtype=torch.int32),
                query_start_loc=torch.tensor([0, 2, 5], dtype=torch.int32), max_query_len=3)


@pytest.mark.parametrize("error,change", [
    (TypeError, dict(q=torch.zeros(5, 4, 64))),
    (TypeError, dict(q=torch.zeros(5, 4, 64, dtype=torch.float16))),
    (ValueError, dict(q=torch.zeros(5, 4, 32, dtype=BF16))),
    (ValueError, dict(q=torch.zeros(5, 64, 4, dtype=BF16).transpose(1, 2))),
    (ValueError, dict(q=torch.zeros(5, 64, dtype=BF16))),
    (TypeError, dict(block_table=torch.zeros(2, 4, dtype=torch.int64))),
    (ValueError, dict(block_table=torch.zeros(3, 4, dtype=torch.int32))),
    (ValueError, dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t())),
    (TypeError, dict(seq_lens=torch.zeros(2))),
    (ValueError, dict(seq_lens=torch.zeros((), dtype=torch.int32))),
    (ValueError, dict(query_start_loc=torch.zeros(2, dtype=torch.int32))),
    (TypeError, dict(tree_mask=torch.zeros(5, 3))),
    (ValueError, dict(tree_mask=torch.zeros(4, 3, dtype=torch.bool))),
    (ValueError, dict(tree_mask=torch.zeros(3, 5, dtype=torch.bool).t())),
    (ValueError, dict(max_query_len=0)),
    (ValueError, dict(out=torch.zeros(5, 4, 64))),
    (ValueError, dict(lse=torch.zeros(5, 3))),
    (ValueError, dict(lse=torch.zeros(5, 4, dtype=torch.float64))),
    (ValueError, dict(v_cache=torch.zeros(7, 16, 2, 64, dtype=BF16))),
])
def test_tree_attention_refusals(error, change):
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    with pytest.raises(error):
        tree_paged_attention(**{**_tree(), **change})


def test_tree_attention_needs_the_device():
    from qsa_vllm_b200 import QSAError
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    with pytest.raises(QSAError):
        tree_paged_attention(**_tree(), tree_mask=torch.zeros(5, 3, dtype=torch.bool),
                             lse=torch.zeros(5, 4))


@pytest.mark.parametrize("error,change", [
    (TypeError, dict(weights=torch.zeros(2, 2, 64, dtype=torch.float64))),
    (ValueError, dict(weights=torch.zeros(2, 1, 64))),
    (ValueError, dict(weights=torch.zeros(2, 64, 2).transpose(1, 2))),
    (ValueError, dict(out=torch.zeros(2, 2, 63))),
    (ValueError, dict(lse=torch.zeros(4, 4))),
    (ValueError, dict(row_factors=torch.zeros(4))),
    (ValueError, dict(row_factors=torch.zeros(5, dtype=torch.float64))),
    (ValueError, dict(max_query_len=-1)),
])
def test_attention_weights_refusals(error, change):
    from qsa_vllm_b200 import QSAError
    from qsa_vllm_b200.eviction import accumulate_attention_weights
    args = _tree()
    del args["v_cache"]
    args.update(lse=torch.zeros(5, 4), weights=torch.zeros(2, 2, 64))
    with pytest.raises(QSAError):
        accumulate_attention_weights(**args)
    with pytest.raises(error):
        accumulate_attention_weights(**{**args, **change})


def test_tree_c_abi_refusals():
    from qsa_vllm_b200 import _lib
    lib = _lib.load_library()

    def tree(rows=4, hq=8, d=128, dtype=0, k=4096, blocks=8, page=16, hkv=2, table=4096, width=4,
             requests=2, mask=None, mask_width=0, most=2, scale=0.1, out=4096, v=4096, q=4096,
             ws=None, n=0):
        return lib.qsa_tree_attention(
            q, hq * d, d, rows, hq, d, dtype, k, 64, 64, 64, v, 64, 64, 64, blocks, page, hkv, table,
            4, width, requests, 4096, 4096, mask, 0, mask_width, most, scale, out, 8, 8, None, 0,
            ws, n, None)
    assert tree(rows=0) == 0 and tree(requests=0) == 0
    for bad, status, word in (
            (dict(rows=-1), 1, b"negative"), (dict(dtype=2), 2, b"dtype"), (dict(d=260), 2, b"head_dim"),
            (dict(d=12), 2, b"head_dim"), (dict(d=0), 2, b"head_dim"), (dict(hq=7), 1, b"multiple"),
            (dict(hkv=0), 1, b"multiple"), (dict(requests=40000), 2, b"65535"),
            (dict(page=0), 1, b"page"), (dict(width=1 << 27), 2, b"2^30"),
            (dict(scale=0.0), 1, b"scale"), (dict(scale=-1.0), 1, b"scale"),
            (dict(scale=float("nan")), 1, b"scale"), (dict(scale=float("inf")), 1, b"scale"),
            (dict(most=0), 1, b"max_query_len"), (dict(q=None), 1, b"null"),
            (dict(table=None), 1, b"null"), (dict(out=None), 1, b"null"), (dict(v=None), 1, b"null"),
            (dict(k=4104), 1, b"aligned"), (dict(q=4098), 1, b"aligned"), (dict(v=4104), 1, b"aligned"),
            (dict(out=4097), 1, b"aligned"), (dict(), 3, b"workspace"),
            (dict(ws=4096, n=100), 3, b"workspace")):
        assert tree(**bad) == status and word in lib.qsa_last_error(), bad
    assert lib.qsa_tree_attention_workspace_bytes(4, 2, 8, 2, 128, 2) > 0
    # neither the longest request nor the batch makes it grow past two tiles of rows per block
    most = lib.qsa_tree_attention_workspace_bytes(1 << 20, 2, 8, 2, 128, 1 << 30)
    assert most <= 2 * 160 * 256 * 129 * 4 + 160 * 64
    for bad in ((0, 2, 8, 2, 128, 2), (4, 0, 8, 2, 128, 2), (4, 2, 7, 2, 128, 2), (4, 2, 8, 2, 128, 0),
                (4, 2, 8, 2, 72, 2)):
        assert lib.qsa_tree_attention_workspace_bytes(*bad) == 0


def test_evict_takes_any_budget():
    """Budgets past what the selection's own entry points take are not refused (a missing
    workspace is, behind every check of sizes)."""
    from qsa_vllm_b200 import _lib
    lib = _lib.load_library()
    for cap, budget in (65536, 60000), (524288, 524287), (1 << 20, 1 << 20):
        assert lib.qsa_cache_evict(4096, cap, cap, 1, cap, 4096, 1, budget, 0, 0, 4096, 64, 64, 64,
                                   4096, 64, 64, 64, 8, 16, 1, 64, 0, 4096, 4, 4, None, 0, 0, 4096,
                                   cap, cap, 4096, 4096, None, 0, None) == 3, (cap, budget)


def test_a_table_without_columns_is_not_in_place():
    from qsa_vllm_b200.eviction import _tables
    table = torch.zeros(2, 4, dtype=torch.int32)
    for empty in table[:, :0], torch.zeros(2, 0, dtype=torch.int32):
        got = _tables("cache_compact", -1, table, empty)
        assert got[3] and got[3] != got[0] and got[5] == 0
    assert _tables("cache_compact", -1, table, None)[3] is None


@pytest.mark.parametrize("dim,base,length,factor,first,last", [
    # indexes of the pairs that turn 32 times and once: 20.94 and 45.03; 38.99 and 63.07 of 64;
    # 10.47 and 22.51 of 32; 11.97 and 68.67 of 64, whose ramp does not end within the head
    (128, 10000.0, 4096, 4.0, 20, 46),
    (128, 10000.0, 55000, 16.0, 38, 64),
    (64, 10000.0, 4096, 4.0, 10, 23),
    (128, 50.0, 418, 2.0, 11, 69),
    (128, 10000.0, 6, 2.0, 0, 0),      # hardly a turn at all: only the first pair is kept
    (128, 10000.0, 3, 2.0, -6, -5),    # not even that
])
def test_yarn_ramps_over_the_pairs(dim, base, length, factor, first, last):
    """Between whole indexes of pairs the division sets in linearly with the index."""
    from qsa_vllm_b200.rotary import rotary_frequencies
    got, scale = rotary_frequencies(dim, base, scaling="yarn", scaling_factor=factor,
                                    original_length=length)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        share = float(i > first) if first == last else min(max((i - first) / (last - first), 0), 1)
        want = plain * (1 - share + share / factor)
        assert math.isclose(float(got[i]), want, rel_tol=1e-12), (i, share)
    assert math.isclose(scale, 0.1 * math.log(factor) + 1)


def test_yarn_refusals():
    from qsa_vllm_b200.rotary import rotary_frequencies
    for bad in (dict(base=1.0), dict(beta_slow=0.0), dict(beta_slow=33.0), dict(original_length=0)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, **{**dict(scaling="yarn", scaling_factor=2.0,
                                             original_length=4096), **bad})


def test_workspaces_are_checked():
    from qsa_vllm_b200._lib import workspace_of
    like, ws = torch.zeros(1), torch.zeros(100, dtype=torch.uint8)
    assert workspace_of("op", ws, 100, like) is ws
    assert workspace_of("op", ws.view(torch.float32), 100, like).numel() == 25
    assert workspace_of("op", ws, 101, like).numel() == 101   # too small: a fresh one
    assert workspace_of("op", None, 7, like).numel() == 7
    assert workspace_of("op", None, 0, like) is None and workspace_of("op", ws, 0, like) is None
    for need in 100, 0:
        with pytest.raises(TypeError, match="workspace"):
            workspace_of("op", ws.to("meta"), need, like)
        with pytest.raises(ValueError, match="workspace"):
            workspace_of("op", ws[:1].expand(100), need, like)
        with pytest.raises(ValueError, match="workspace"):
            workspace_of("op", torch.zeros(200, dtype=torch.uint8)[::2], need, like)


def test_weights_without_rows_take_any_strides_of_q():
    """A slice without rows of an unaligned projection has nothing to align (a capacity of 0:
    behind the checks nothing is launched)."""
    from qsa_vllm_b200 import _lib
    lib = _lib.load_library()

    def weights(rows, q, head):
        return lib.qsa_attention_weights(
            q, 4 * head, head, rows, 4, 64, 0, 4096, 64, 64, 64, 8, 16, 2, 4096, 4, 4, 2, 4096,
            4096, None, 0, 0, 1, 0.125, 4096, 4, None, 0, 4096, 0, 0, 4096, 0, 0, 0, None)
    assert weights(0, None, 67) == 0 and weights(0, 4098, 67) == 0 and weights(3, 4096, 64) == 0
    for bad in (3, 4098, 64), (3, 4096, 67), (3, None, 64):
        assert weights(*bad) == 1, bad
