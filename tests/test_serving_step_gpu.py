"""A speculative serving step from end to end, as a dense layer beside the sparse ones would run
it: rotate and store the drafts, verify the tree, commit the accepted path, add up the weights of
the accepted rows, evict, and go on decoding; against the same step in 64 bits on the host."""

import math

import pytest
import torch

import tree_cases as tc

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def gather(kv, table, b, n, page):
    t = torch.arange(n)
    return kv[table[b][t // page].long(), t % page].double()


@pytest.mark.parametrize("hq,hkv,d,page,steps", [(8, 2, 128, 16, 4), (4, 4, 64, 64, 3)])
@pytest.mark.parametrize("captured", [False, True])
def test_speculative_steps(dev, hq, hkv, d, page, steps, captured):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import accumulate_attention_weights, cache_compact, cache_evict
    from qsa_vllm_b200.rotary import rotary_frequencies, rotary_store
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    g = torch.Generator().manual_seed(d + steps)
    batch, nodes, budget, sinks, recent, cap = 3, 6, 150, 4, 32, 320
    width = cap // page
    kv = torch.randn(batch * width, page, hkv, 2 * d, generator=g).to(BF16).to(dev)
    table = torch.randperm(batch * width, generator=g).view(batch, width).to(torch.int32).to(dev)
    k_cache, v_cache = kv[..., :d], kv[..., d:]
    freq, factor = rotary_frequencies(d // 2, scaling="linear", scaling_factor=2.0, device=dev)
    # parents of the tree's nodes, and the path that is accepted: nodes 0, 2, 5
    parents, path = [-1, 0, 0, 1, 2, 2], [0, 2, 5]
    mask = torch.zeros(nodes, nodes, dtype=torch.bool)
    depth = []
    for i, p in enumerate(parents):
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
        depth.append(0 if p < 0 else depth[p] + 1)
    depth = torch.tensor(depth)
    rows = batch * nodes
    start = torch.arange(0, rows + 1, nodes, dtype=torch.int32, device=dev)
    lens = torch.tensor([100, 147, 160], dtype=torch.int32, device=dev)   # cached tokens
    where = torch.tensor([1000, 5, 70000], device=dev)                     # positions go on
    weights = torch.rand(batch, hkv, cap, generator=g).to(dev)
    weights *= torch.arange(cap, device=dev) < lens[:, None, None]
    factors = torch.tensor([1.0 if i in path else 0.0 for i in range(nodes)] * batch, device=dev)
    tree_mask = mask.repeat(batch, 1).to(dev)
    qkv = torch.empty(rows, (hq + 2 * hkv) * d, dtype=BF16, device=dev)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    out = torch.empty(rows, hq, d, dtype=BF16, device=dev)
    lse = torch.empty(rows, hq, device=dev)
    q_rot = torch.empty(rows, hq, d, dtype=BF16, device=dev)
    node = torch.arange(nodes, device=dev)
    depth_d, path_d = depth.to(dev), torch.tensor(path, device=dev)

    def step():
        pos = (where[:, None] + depth_d).flatten()
        at = lens[:, None] + node
        slots = (table.gather(1, (at // page).long()).long() * page + at % page).flatten()
        rotary_store(q, k, v, pos, freq, k_cache, v_cache, slots, factor=factor, q_out=q_rot)
        seq = lens + nodes
        tree_paged_attention(q_rot, k_cache, v_cache, table, seq, start, out, lse=lse,
                             max_query_len=nodes, tree_mask=tree_mask)
        accumulate_attention_weights(q_rot, k_cache, table, seq, start, lse, weights,
                                     max_query_len=nodes, tree_mask=tree_mask,
                                     row_factors=factors)
        accepted = lens[:, None] + path_d
        cache_compact(k_cache, v_cache, table, accepted.to(torch.int32), lens)
        # the accepted tokens' weights go with them; rejected ones received none
        kept_w = weights.gather(2, accepted[:, None].expand(-1, hkv, -1).long())
        weights.scatter_(2, at[:, None].expand(-1, hkv, -1).long(), 0.0)
        weights.scatter_(2, at[:, None, :3].expand(-1, hkv, -1).long(), kept_w)
        lens.add_(3)
        _, now = cache_evict(weights, lens, table, k_cache, v_cache, budget, sinks=sinks,
                             recent=recent)
        lens.copy_(now)
        where.add_(3)

    graph = None
    if captured:
        saved = [t.clone() for t in (kv, weights, lens, where)]
        qkv.normal_()
        step()
        for t, s in zip((kv, weights, lens, where), saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for t, s in zip((kv, weights, lens, where), saved):
            t.copy_(s)
    for _ in range(steps):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        before = dict(kv=kv.cpu(), w=weights.cpu().double(), lens=lens.tolist(),
                      pos=where.tolist())
        if graph is not None:
            graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        host_table = table.cpu()
        turned_q, turned_k = q_rot.cpu(), None
        # rotation of the queries, by the formula
        pos = torch.tensor([p + int(x) for p in before["pos"] for x in depth]).double()
        a = pos[:, None, None] * freq.cpu()
        half = d // 4
        x = q.double().cpu()
        y = x.clone()
        y[..., :half] = x[..., :half] * a.cos() - x[..., half:2 * half] * a.sin()
        y[..., half:2 * half] = x[..., half:2 * half] * a.cos() + x[..., :half] * a.sin()
        assert (turned_q.double() - y).abs().max() <= 2.0 ** -8 * 8
        x = k.double().cpu()
        y = x.clone()
        y[..., :half] = x[..., :half] * a.cos() - x[..., half:2 * half] * a.sin()
        y[..., half:2 * half] = x[..., half:2 * half] * a.cos() + x[..., :half] * a.sin()
        turned_k = y.to(BF16)
        for b in range(batch):
            n = before["lens"][b]
            # the cache with the drafts, as the attention saw it
            cached = gather(before["kv"], host_table, b, n, page)
            drafts = torch.cat([turned_k[b * nodes:(b + 1) * nodes],
                                v.cpu()[b * nodes:(b + 1) * nodes]], -1).double()
            full = torch.cat([cached, drafts])
            see = torch.cat([torch.ones(nodes, n, dtype=torch.bool), mask], 1)
            got_w = before["w"][b].clone()
            for h in range(hkv):
                qs = turned_q[b * nodes:(b + 1) * nodes, h * (hq // hkv):(h + 1) * (hq // hkv)]
                s = torch.einsum("igd,td->igt", qs.double(), full[:, h, :d]) / math.sqrt(d)
                s = s.masked_fill(~see[:, None], -math.inf)
                p = s.softmax(-1)
                o = torch.einsum("igt,td->igd", p, full[:, h, d:])
                got = out[b * nodes:(b + 1) * nodes, h * (hq // hkv):(h + 1) * (hq // hkv)]
                # p and the output rounded (2^-9 of weights that add up to 1, values within 5),
                # keys rounded once more at a border of bf16 move a score by a little
                assert (got.double().cpu() - o).abs().max() <= 2.0 ** -8 * 5 + 0.02
                got_w[h, :n + nodes] += p[path].sum((0, 1))
            # commit, then eviction
            order = list(range(n)) + [n + i for i in path]
            total = n + 3
            committed = full[order]
            w_new = got_w[:, order]
            now = int(lens[b])
            assert now == min(total, budget)
            final = gather(kv.cpu(), host_table, b, now, page)
            w_final = weights[b].cpu().double()
            for h in range(hkv):
                if total <= budget:
                    keep = list(range(total))
                else:
                    # the device's own weights decide; they are near the host's
                    mid = total - sinks - recent
                    cut = w_new[h, sinks:total - recent].sort(descending=True).values
                    limit = cut[budget - sinks - recent - 1]
                    free = {i for i in range(sinks, total - recent)
                            if abs(w_new[h, i] - limit) < 1e-3 * (1 + limit)}
                    sure = [i for i in range(total) if i < sinks or i >= total - recent
                            or (i not in free and w_new[h, i] > limit)]
                    assert mid > 0
                    keep, rest = sure, budget - len(sure)
                    held = [i for i in sorted(free)
                            if (final[:, h] == committed[i, h]).all(-1).any()]
                    assert len(held) == rest
                    keep = sorted(sure + held)
                assert (final[:, h, d:] == committed[keep, h, d:]).all()
                assert (final[:, h, :d] - committed[keep, h, :d]).abs().max() <= 2.0 ** -7 * 8
                assert (w_final[h, :now] - w_new[h, keep]).abs().max() < 1e-3 * (
                    1 + w_new[h].max())
                assert (w_final[h, now:total] == 0).all()
    assert _lib.device_error_poll() == 0


def test_workspaces_of_another_device_are_refused(dev):
    """A host address, or one byte for all, does not go to a kernel."""
    from qsa_vllm_b200.eviction import cache_evict
    from qsa_vllm_b200.qsa import qsa_sparse_paged_attention
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    kv = torch.zeros(4, 16, 2, 256, dtype=torch.bfloat16, device=dev)
    k, v = kv[..., :128], kv[..., 128:]
    table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    lens = torch.full((1,), 60, dtype=torch.int32, device=dev)
    start = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=dev)
    idx = torch.arange(32, dtype=torch.int32, device=dev).view(1, 32)
    w = torch.zeros(1, 2, 64, device=dev)
    host = torch.empty(1 << 25, dtype=torch.uint8)
    one = torch.empty(1, dtype=torch.uint8, device=dev).expand(1 << 25)
    for ws, err in (host, TypeError), (one, ValueError):
        with pytest.raises(err, match="workspace"):
            tree_paged_attention(q, k, v, table, lens, start, max_query_len=1, workspace=ws)
        with pytest.raises(err, match="workspace"):
            cache_evict(w, lens, table, k, v, 40, workspace=ws)
        with pytest.raises(err, match="workspace"):
            qsa_sparse_paged_attention(q, k, v, idx, table, start[:1], workspace=ws)
