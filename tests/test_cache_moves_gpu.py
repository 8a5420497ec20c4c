"""Compaction and eviction of cached tokens: exact, against a plain restatement on the host."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def pool(g, dev, requests, ctx, page, hkv, d, dtype, more=0, fused=True, shift=0):
    width = -(-ctx // page) if ctx else 1
    blocks = requests * (width + more) + 2
    if fused:
        buf = torch.randn(blocks, page, hkv, 2 * d + shift, generator=g).to(dtype).to(dev)
        k, v = buf[..., shift:d + shift], buf[..., d + shift:]
    else:
        buf = torch.randn(2, blocks, hkv, page, d, generator=g).to(dtype).to(dev)
        k, v = buf[0].transpose(1, 2), buf[1].transpose(1, 2)
    pages = torch.randperm(blocks, generator=g)[: requests * (width + more)].to(torch.int32)
    return (k, v, pages[: requests * width].view(requests, width).to(dev),
            pages[requests * width:].view(requests, more).to(dev))


def moved(k, v, table, out_table, lists, starts):
    """The caches after the moves; lists[b][h]: the sources."""
    k0, v0, page = k.cpu(), v.cpu(), k.shape[1]
    k1, v1 = k0.clone(), v0.clone()
    table, out_table = table.cpu().long(), out_table.cpu().long()
    for b, heads in enumerate(lists):
        for h, sources in enumerate(heads):
            for j, s in enumerate(sources):
                if s < 0:
                    continue
                t = starts[b] + j
                a, at = table[b, s // page], s % page
                o, ot = out_table[b, t // page], t % page
                k1[o, ot, h], v1[o, ot, h] = k0[a, at, h], v0[a, at, h]
    return k1, v1


CASES = [  # requests, ctx, page, heads, d, dtype, count, start, per head, fused, shift
    (1, 1, 16, 1, 64, BF16, 1, 0, False, True, 0),
    (3, 200, 16, 2, 128, BF16, 37, 11, True, True, 0),
    (5, 333, 1, 4, 64, F16, 300, 0, False, False, 0),
    (2, 2500, 64, 8, 128, BF16, 1900, 100, True, True, 0),
    (1, 9000, 48, 1, 128, F32, 8000, 5, True, True, 0),
    (2, 700, 20, 3, 40, BF16, 600, 50, False, True, 4),   # rows at odd offsets: 8-byte aligned
    (2, 300, 16, 2, 31, F16, 250, 7, True, True, 1),       # rows of an odd length: 2-byte copies
    (40, 257, 32, 8, 256, BF16, 100, 1, True, True, 0),
    (2, 600, 16, 1, 2048, BF16, 100, 3, False, True, 0),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("requests,ctx,page,hkv,d,dtype,count,start,per_head,fused,shift", CASES)
def test_compact(dev, in_place, requests, ctx, page, hkv, d, dtype, count, start, per_head, fused,
                 shift):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_compact
    g = torch.Generator().manual_seed(ctx + count)
    k, v, table, other = pool(g, dev, requests, ctx, page, hkv, d, dtype,
                              0 if in_place else -(-ctx // page), fused, shift)
    heads = hkv if per_head else 1
    idx = torch.rand(requests, heads, ctx - start, generator=g).argsort(-1)[..., :count]
    idx = (idx.sort(-1).values + start).to(torch.int32)
    idx[torch.rand(idx.shape, generator=g) < 0.1] = -1
    starts = torch.full((requests,), start, dtype=torch.int32)
    lists = idx.expand(-1, hkv, -1).tolist()
    want = moved(k, v, table, table if in_place else other, lists, starts.tolist())
    arg = idx.to(dev) if per_head else idx[:, 0].contiguous().to(dev)
    cache_compact(k, v, table, arg, starts.to(dev), out_table=None if in_place else other)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    assert _lib.device_error_poll() == 0


def test_compact_in_place_many_times_over_itself(dev):
    """Dense lists of long contexts: each destination is another row's source, several groups
    and several clusters' rounds apart."""
    from qsa_vllm_b200.eviction import cache_compact
    g = torch.Generator().manual_seed(1)
    k, v, table, _ = pool(g, dev, 2, 20000, 16, 2, 64, BF16)
    for drop in (1, 2, 700):
        idx = torch.stack([torch.cat([torch.arange(3), torch.arange(3 + drop + b, 19000 + b)])[:18000]
                           for b in range(2)]).to(torch.int32)
        want = moved(k, v, table, table, [[r] * 2 for r in idx.tolist()], [0, 0])
        cache_compact(k, v, table, idx.to(dev))
        assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_compact_skips_and_reports_what_it_cannot_move(dev):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_compact
    g = torch.Generator().manual_seed(2)
    k, v, table, _ = pool(g, dev, 1, 64, 16, 1, 64, BF16)
    table[0, 2] = -1
    for idx, start in ([40], 0), ([64], 0), ([2**31 - 1], 0), ([3], 5), ([5], 40), ([5], -1):
        k0, v0 = k.clone(), v.clone()
        cache_compact(k, v, table, torch.tensor([idx], dtype=torch.int32, device=dev),
                      torch.tensor([start], dtype=torch.int32, device=dev))
        assert _lib.device_error_poll() == 2, (idx, start)
        assert torch.equal(k, k0) and torch.equal(v, v0)
    cache_compact(k, v, table, torch.empty(1, 0, dtype=torch.int32, device=dev))
    cache_compact(k, v, table[:0], torch.empty(0, 4, dtype=torch.int32, device=dev))
    assert torch.equal(k, k0) and _lib.device_error_poll() == 0


def chosen(w, n, budget, sinks, recent):
    if n <= budget:
        return list(range(n))
    middle = w[sinks:n - recent].double()
    best = (-middle).sort(stable=True).indices[: budget - sinks - recent].sort().values + sinks
    return list(range(sinks)) + best.tolist() + list(range(n - recent, n))


EVICT = [  # lengths, capacity, budget, sinks, recent, page, heads, d, dtype, shared
    ([0, 1, 5, 9, 17], 17, 9, 2, 3, 16, 2, 64, BF16, False),
    ([100, 257, 64, 65], 257, 64, 4, 16, 16, 4, 128, BF16, False),
    ([300] * 3, 300, 299, 0, 0, 32, 1, 64, F16, False),
    ([777, 2], 1000, 100, 100, 0, 8, 2, 128, BF16, False),   # nothing left to choose
    ([777, 500], 800, 100, 0, 100, 8, 2, 128, BF16, True),
    ([5000, 3000, 5001], 5003, 1201, 4, 128, 64, 2, 128, BF16, True),
    ([40000], 40000, 5000, 16, 1024, 64, 1, 64, F32, False),
    ([2112, 2049, 2048], 2112, 2048, 4, 512, 16, 8, 128, BF16, False),
    ([50, 60], 60, 0, 0, 0, 16, 2, 64, BF16, False),          # a budget of nothing
    ([70, 300], 64, 32, 1, 1, 16, 2, 64, BF16, False),        # lengths past the capacity
    ([70, 300], 0, 8, 1, 1, 16, 2, 64, BF16, False),          # a capacity of nothing
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths,capacity,budget,sinks,recent,page,hkv,d,dtype,shared", EVICT)
def test_evict(dev, in_place, lengths, capacity, budget, sinks, recent, page, hkv, d, dtype,
               shared):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_evict
    g = torch.Generator().manual_seed(capacity + budget)
    requests, heads = len(lengths), 1 if shared else hkv
    k, v, table, other = pool(g, dev, requests, max(capacity, *lengths), page, hkv, d, dtype,
                              0 if in_place else -(-max(budget, capacity) // page))
    # weights with many ties, at zero and elsewhere
    w = torch.randint(0, 40, (requests, heads, capacity + 3), generator=g).float()
    w = torch.where(torch.rand(w.shape, generator=g) < 0.3, w * torch.rand(w.shape, generator=g), w)
    w = w.to(dev)[..., :capacity]
    counted = [min(n, capacity) for n in lengths]
    keep = [[chosen(w[b, h].cpu(), n, budget, sinks, recent) for h in range(heads)]
            for b, n in enumerate(counted)]
    lists = [r * hkv if shared else r for r in keep]
    want = moved(k, v, table, table if in_place else other, lists, [0] * requests)
    w_out = None if in_place else torch.full((requests, heads, capacity), -5.0, device=dev)
    w_want = (w.clone() if in_place else w_out.clone()).cpu()
    for b, n in enumerate(counted):
        for h in range(heads):
            at = keep[b][h]
            w_want[b, h, :len(at)] = w[b, h].cpu()[at]
            w_want[b, h, len(at):n] = 0
    seq = torch.tensor(lengths, dtype=torch.int32, device=dev)
    kept, count = cache_evict(w, seq, table, k, v, budget, sinks=sinks, recent=recent,
                              out_table=None if in_place else other, weights_out=w_out)
    assert count.tolist() == [min(n, budget) for n in counted]
    assert seq.tolist() == lengths
    for b in range(requests):
        for h in range(heads):
            n = len(keep[b][h])
            assert kept[b, h, :n].tolist() == keep[b][h] and (kept[b, h, n:] == -1).all()
    assert torch.equal((w if in_place else w_out).cpu(), w_want)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    assert _lib.device_error_poll() == 0


@pytest.mark.parametrize("cache_in_place", [True, False])
def test_evict_with_one_of_cache_and_weights_in_place(dev, cache_in_place):
    from qsa_vllm_b200.eviction import cache_evict
    g = torch.Generator().manual_seed(5)
    k, v, table, other = pool(g, dev, 3, 900, 16, 2, 128, BF16, 57)
    w = torch.rand(3, 2, 900, generator=g).to(dev)
    lengths, budget = [900, 640, 500], 600
    keep = [[chosen(w[b, h].cpu(), n, budget, 4, 64) for h in range(2)]
            for b, n in enumerate(lengths)]
    want = moved(k, v, table, table if cache_in_place else other, keep, [0] * 3)
    w_out = torch.zeros_like(w) if cache_in_place else w
    w_want = torch.zeros(3, 2, 900) if cache_in_place else w.cpu().clone()
    for b, n in enumerate(lengths):
        for h in range(2):
            w_want[b, h, :len(keep[b][h])] = w[b, h].cpu()[keep[b][h]]
            w_want[b, h, len(keep[b][h]):n] = 0
    seq = torch.tensor(lengths, dtype=torch.int32, device=dev)
    cache_evict(w, seq, table, k, v, budget, sinks=4, recent=64,
                out_table=None if cache_in_place else other, weights_out=w_out)
    assert torch.equal(w_out.cpu(), w_want)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_evict_captured_again_and_again(dev):
    """A captured step that grows and evicts: the lengths are the device's, not the capture's."""
    from qsa_vllm_b200.eviction import cache_evict
    g = torch.Generator().manual_seed(8)
    k, v, table, _ = pool(g, dev, 2, 128, 16, 2, 64, BF16)
    w = torch.rand(2, 2, 128, generator=g).to(dev)
    seq = torch.tensor([100, 90], dtype=torch.int32, device=dev)
    start = [t.clone() for t in (k, v, w, seq)]

    def step():
        _, count = cache_evict(w, seq, table, k, v, 64, sinks=2, recent=8)
        seq.copy_(count + 30)

    for _ in range(3):
        step()
    want = [t.clone() for t in (k, v, w, seq)]
    for t, s in zip((k, v, w, seq), start):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for t, s in zip((k, v, w, seq), want):
        assert torch.equal(t, s)


@pytest.mark.parametrize("requests,hkv,ctx,budget", [
    (300, 2, 96, 40),       # 600 lists: the lengths come from several blocks of several warps
    (61, 8, 2300, 700),     # 488 lists, a wider form of the selection
    (1000, 4, 2000, 64),    # a warp for each list
    (40, 1, 9000, 1000),    # a cluster for each list
])
def test_evict_many_lists_of_different_lengths(dev, requests, hkv, ctx, budget):
    """Each list is chosen from its own request's length, call after call in one workspace: the
    lengths of a call must be neither the one's before nor what the workspace held."""
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_evict, cache_evict_workspace_bytes
    g = torch.Generator().manual_seed(requests + ctx)
    kv = torch.randn(32, 16, hkv, 16, generator=g).to(BF16).to(dev)
    k, v = kv[..., :8], kv[..., 8:]
    table = torch.randint(0, 32, (requests, -(-ctx // 16)), generator=g).to(torch.int32).to(dev)
    other = torch.full((requests, 1), -1, dtype=torch.int32, device=dev)
    need = cache_evict_workspace_bytes(requests, hkv, budget, 3, 5)
    workspace = torch.full((need,), 0x7f, dtype=torch.uint8, device=dev)
    calls = []
    for n in range(3):  # queued one behind another, read afterwards
        seq = torch.randint(0, ctx + 1, (requests,), generator=g).to(torch.int32)
        w = torch.rand(requests, hkv, ctx, generator=g)
        kept = torch.empty(requests, hkv, budget, dtype=torch.int32, device=dev)
        lens, weights, out = seq.to(dev), w.to(dev), torch.zeros_like(w, device=dev)
        calls.append((seq, w, kept, lens, weights, out))
    torch.cuda.synchronize()
    keep_k = k.clone()
    for seq, w, kept, lens, weights, out in calls:
        # destinations without pages: no row finds a place, which is reported
        cache_evict(weights, lens, table, k, v, budget, sinks=3, recent=5, out_table=other,
                    weights_out=out, kept=kept, workspace=workspace)
    torch.cuda.synchronize()
    assert torch.equal(k, keep_k) and _lib.device_error_poll() == 2
    for seq, w, kept, lens, weights, out in calls:
        t = torch.arange(ctx)
        n = seq.long()[:, None, None]
        rank = torch.where((t < 3) | (t >= n - 5), 2.0, w)
        rank = torch.where(t < n, rank, -1.0)
        order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
        here = torch.arange(budget) < n.clamp(max=budget)
        want = torch.where(here, order, ctx).sort(-1).values
        want = torch.where(here, want, -1)
        assert torch.equal(kept.cpu().long(), want)
        w_want = torch.where(here, w.gather(2, want.clamp(min=0)), 0.0)
        assert torch.equal(out.cpu()[..., :budget], w_want) and not out[..., budget:].any()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths,budget,sinks,recent", [
    ([70000, 55001, 64], 55000, 0, 0),
    ([65536], 65535, 0, 0),                    # one token goes
    ([300000, 299000], 200000, 16, 1024),
    ([524288 + 9, 524288], 500000, 4, 5),      # the most there is to choose from
])
def test_evict_large_budgets(dev, in_place, lengths, budget, sinks, recent):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_evict
    g = torch.Generator().manual_seed(budget)
    requests, capacity = len(lengths), max(lengths)
    k, v, table, other = pool(g, dev, requests, capacity, 64, 1, 8, BF16,
                              0 if in_place else -(-budget // 64))
    w = torch.randint(0, 1 << 16, (requests, 1, capacity), generator=g).float()
    w[torch.rand(w.shape, generator=g) < 0.2] = 0
    keep = [torch.tensor(chosen(w[b, 0], n, budget, sinks, recent)) for b, n in enumerate(lengths)]
    k0, v0, table0 = k.cpu(), v.cpu(), table.cpu().long()
    to = table0 if in_place else other.cpu().long()
    k1, v1 = k0.clone(), v0.clone()
    for b, at in enumerate(keep):
        t = torch.arange(at.numel())
        k1[to[b][t // 64], t % 64], v1[to[b][t // 64], t % 64] = \
            k0[table0[b][at // 64], at % 64], v0[table0[b][at // 64], at % 64]
    weights = w.to(dev)
    out = None if in_place else torch.zeros_like(weights)
    kept, count = cache_evict(weights, torch.tensor(lengths, dtype=torch.int32, device=dev), table,
                              k, v, budget, sinks=sinks, recent=recent,
                              out_table=None if in_place else other, weights_out=out)
    got = (weights if in_place else out).cpu()
    for b, at in enumerate(keep):
        n = at.numel()
        assert torch.equal(kept[b, 0, :n].cpu().long(), at) and (kept[b, 0, n:] == -1).all()
        assert count[b] == n and torch.equal(got[b, 0, :n], w[b, 0, at])
        assert not got[b, 0, n:lengths[b]].any()
    assert torch.equal(k.cpu(), k1) and torch.equal(v.cpu(), v1)
    assert _lib.device_error_poll() == 0


def test_compact_to_a_table_without_columns_moves_nothing(dev):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.eviction import cache_compact
    g = torch.Generator().manual_seed(4)
    k, v, table, _ = pool(g, dev, 2, 64, 16, 2, 64, BF16)
    k0, v0 = k.clone(), v.clone()
    idx = torch.tensor([[5, 9], [-1, 7]], dtype=torch.int32, device=dev)
    cache_compact(k, v, table, idx, out_table=table[:, :0])
    assert _lib.device_error_poll() == 2
    assert torch.equal(k, k0) and torch.equal(v, v0)
