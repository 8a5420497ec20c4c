"""Attention of drafted-token trees, and the weights of cached tokens, against 64 bits."""

import pytest
import torch

import tree_cases as tc
from tree_cases import BF16, F16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def call(c, lse=True, out=None, **more):
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    if lse is True:
        lse = torch.full(c["q"].shape[:2], -77.0, device=c["q"].device)
    if out is None:
        out = torch.full_like(c["q"], 55.0, memory_format=torch.contiguous_format)
    more.setdefault("max_query_len", c["most"])
    got = tree_paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["start"], out,
                               tree_mask=c["mask"], lse=lse, **more)
    assert got is out
    return out, lse


def check(c, scale=None, **more):
    from qsa_vllm_b200 import _lib
    out, lse = call(c, scale=scale, **more)
    want, tol, z, ztol = tc.attention(c, scale)
    n = c["rows"]
    first = int(c["start"][0])
    tc.compare(out[first:n], want[first:n], tol[first:n], "out")
    tc.compare(lse[first:n], z[first:n], ztol[first:n], "lse")
    # rows of no request are left as they were
    assert (out[n:] == 55).all() and (lse[n:] == -77).all()
    assert (out[:first] == 55).all()
    assert _lib.device_error_poll() == 0
    return out, lse


# lens, counts, hq, hkv, d, page, dtype, mask
CASES = [
    ([1], [1], 1, 1, 64, 16, BF16, "tree"),
    ([5], [1], 2, 1, 128, 16, F16, "chain"),
    ([8], [8], 8, 1, 128, 16, BF16, "tree"),              # drafts only, no context
    ([130, 128, 127, 129], [3, 0, 1, 2], 16, 2, 128, 16, BF16, "tree"),
    ([300, 1000, 17], [16, 16, 16], 32, 4, 128, 64, BF16, "tree"),
    ([300, 77, 513], [13, 16, 9], 8, 8, 64, 32, F16, "random"),
    ([1500], [64], 8, 1, 128, 128, BF16, "tree"),
    ([700, 900], [64, 33], 32, 4, 64, 64, BF16, "random"),
    ([515], [130], 3, 1, 128, 48, BF16, "random"),         # three heads a group, odd pages
    ([600, 100], [40, 7], 14, 2, 64, 16, F16, "tree"),     # seven heads a group
    ([400], [33], 32, 1, 128, 8, BF16, "none"),
    ([2000, 333], [1, 1], 64, 1, 128, 64, BF16, "chain"),  # one KV head
    ([260], [200], 4, 1, 128, 24, BF16, "chain"),          # a prompt chunk
    ([900, 650], [513, 300], 4, 2, 64, 64, F16, "chain"),
    ([200], [9], 130, 1, 64, 16, BF16, "tree"),            # more heads than a tile's rows
    ([4000], [5], 8, 8, 128, 16, BF16, "tree"),
    # layouts of the general form
    ([70, 33], [5, 6], 4, 2, 64, 1, BF16, "tree"),
    ([70, 33], [5, 6], 4, 2, 128, 5, F16, "random"),
    ([300], [4], 6, 3, 72, 16, BF16, "tree"),
    ([300, 2], [4, 2], 9, 1, 256, 16, F16, "chain"),
    ([150], [20], 2, 2, 8, 32, BF16, "random"),
]


@pytest.mark.parametrize("lens,counts,hq,hkv,d,page,dtype,mask", CASES)
def test_matches_definition(dev, lens, counts, hq, hkv, d, page, dtype, mask):
    check(tc.make(sum(lens) + d, lens, counts, hq, hkv, d, page, dtype, mask, dev, spread=1.5,
                  pad=3))


@pytest.mark.parametrize("d,page", [(128, 16), (64, 64), (128, 5)])
@pytest.mark.parametrize("spread", [0.0, 0.05, 8.0])
def test_flat_and_peaked_scores(dev, d, page, spread):
    """Equal scores, nearly equal ones, and ones so far apart that single tokens take all."""
    check(tc.make(3, [1000, 257], [8, 3], 8, 2, d, page, BF16, "tree", dev, spread=spread))


@pytest.mark.parametrize("d", [64, 128])
def test_rising_scores(dev, d):
    """Each tile's scores are far above the last one's, so that the running maximum moves with
    every tile."""
    c = tc.make(4, [1300, 900], [6, 2], 4, 1, d, 16, BF16, "tree", "cpu")
    q = torch.ones_like(c["q"])
    c["q"] = q
    for b, n in enumerate(c["lens"].tolist()):
        t = torch.arange(n)
        level = (t // 100).double() * (0.5 if b else 3.0) * d ** -0.5
        c["kv"][c["table"][b][t // 16].long(), t % 16, :, :d] = \
            level[:, None, None].to(BF16).expand(-1, 1, d)
    check(tc.to(c, dev))


@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_scale(dev, scale):
    check(tc.make(5, [300, 40], [7, 4], 8, 2, 128, 16, BF16, "tree", dev), scale=scale)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (128, 5)])
@pytest.mark.parametrize("mask", ["tree", "random", "none"])
def test_infinities_and_nans_in_unseen_places(dev, d, page, mask):
    """Drafted tokens with infinite or NaN keys and values reach the rows that see them, and no
    other; so do infinite values of single channels."""
    c = tc.make(6, [200, 140, 9], [20, 12, 9], 4, 2, d, page, BF16, mask, "cpu")
    want_clean = None
    for b in range(3):
        n, count = int(c["lens"][b]), c["counts"][b]
        for j, value, channel in ((3, float("nan"), slice(None)), (5, float("inf"), slice(2, 3)),
                                  (7, -float("inf"), slice(0, 2))):
            t = n - count + j
            page_of = int(c["table"][b][t // page])
            c["kv"][page_of, t % page, :, d:][:, channel] = value
    assert want_clean is None
    g = tc.to(c, dev)
    out, lse = check(g)
    want = tc.attention(c)[0][: c["rows"]]
    assert torch.equal(out[: c["rows"]].double().cpu().isfinite(), want.isfinite())
    assert (~want.isfinite()).any() == (mask != "none")
    assert want.isfinite().any()
    # an unseen key may be NaN too
    sees = [tc.seen(c, b)[0] for b in range(3)]
    hidden = [(b, t) for b in range(3) for t in range(sees[b].shape[1]) if not sees[b][:, t].any()]
    for b, t in hidden:
        c["kv"][int(c["table"][b][t // page]), t % page] = float("nan")
    again, _ = call(tc.to(c, dev))
    assert torch.equal(again[: c["rows"]].view(torch.int16), out[: c["rows"]].view(torch.int16))


def test_nan_keys_of_seen_tokens_reach_their_rows_only(dev):
    c = tc.make(7, [300], [12], 8, 2, 128, 16, BF16, "tree", "cpu")
    t = 300 - 12 + 4
    c["kv"][int(c["table"][0][t // 16]), t % 16, 1, :128] = float("nan")
    out, lse = call(tc.to(c, dev))
    sees = c["mask"][:12, 4]
    bad = out.float().isnan().any(-1).cpu()
    assert torch.equal(bad[:, 4:], sees[:, None].expand(-1, 4)) and not bad[:, :4].any()
    assert torch.equal(lse.isnan().cpu(), bad)


@pytest.mark.parametrize("page,d", [(16, 128), (64, 64), (5, 64)])
def test_unmapped_pages_and_tables_that_end_early(dev, page, d):
    c = tc.make(8, [500, 260, 100], [6, 3, 5], 8, 2, d, page, BF16, "tree", "cpu")
    c["table"][0, 1] = -1
    c["table"][1, 2] = c["kv"].shape[0]
    c["table"][1, 0] = 2**31 - 1
    check(tc.to(c, dev))
    c["table"] = c["table"][:, : 300 // page].contiguous()
    check(tc.to(c, dev))                  # the first request's drafts are out of reach
    c["table"][:] = -1
    out, lse = check(tc.to(c, dev))       # nothing is
    assert (out[: c["rows"]] == 0).all() and (lse[: c["rows"]] == -torch.inf).all()


@pytest.mark.parametrize("page", [16, 3])
def test_empty_requests_rows_and_lengths(dev, page):
    """No rows, no tokens, more rows than tokens, rows that see nothing, padding."""
    c = tc.make(9, [0, 64, 3, 0, 10], [2, 0, 5, 0, 10], 4, 2, 64, page, BF16, "random", dev, pad=4)
    check(c)
    c["mask"][:] = False
    c["lens"].copy_(torch.tensor([2, 64, 5, 0, 10], dtype=torch.int32))
    out, lse = check(c)
    assert (out[: c["rows"]] == 0).all() and (lse[: c["rows"]] == -torch.inf).all()
    c["mask"] = c["mask"][:, :0]
    check(c)
    none = dict(c, q=c["q"][:0], mask=None, rows=0)
    assert call(none)[0].shape[0] == 0


def test_first_rows_of_no_request(dev):
    c = tc.make(10, [100, 60], [4, 4], 8, 2, 128, 16, BF16, "chain", dev)
    c["start"] = torch.tensor([2, 4, 8], dtype=torch.int32, device=dev)
    c["counts"] = [2, 4]
    check(c)


@pytest.mark.parametrize("fused,q_shift", [(False, 0), (True, 8), (True, 3), (False, 5)])
def test_strides_and_alignment(dev, fused, q_shift):
    """Heads before slots, query views with gaps or at odd offsets, outputs with gaps at odd
    offsets."""
    c = tc.make(11, [300, 129], [9, 4], 8, 2, 64, 16, F16, "tree", dev, fused=fused,
                q_shift=q_shift, poison=False)
    want, lse = check(c)
    for shift in (1, 8):
        buf = torch.full((c["q"].shape[0], 10, 64 + 2 * shift), 3.0, dtype=F16, device=dev)
        out = buf[:, 1:9, shift:64 + shift]
        z = torch.full((c["q"].shape[0], 11), 3.0, device=dev)
        call(c, out=out, lse=z[:, 2:10])
        assert torch.equal(out, want) and torch.equal(z[:, 2:10], lse)
        buf[:, 1:9, shift:64 + shift] = 3
        z[:, 2:10] = 3
        assert (buf == 3).all() and (z == 3).all()


@pytest.mark.parametrize("hint", [1, 4, 1000])
@pytest.mark.parametrize("mask", ["chain", "random"])
def test_max_query_len_is_a_hint(dev, hint, mask):
    """A wrong hint moves the work's split, not what is computed: within twice the bound, as
    both results are within it."""
    c = tc.make(12, [700, 90], [60, 17], 8, 1, 128, 16, BF16, mask, dev)
    check(c, max_query_len=hint)


def test_splits_of_long_contexts(dev):
    """One request over many blocks of the work split, and batches whose units are cut at
    uneven places."""
    for lens, counts, hq, hkv, d, page in (([20011], [3], 8, 1, 128, 16),
                                           ([9000, 5, 3001, 12000], [2, 2, 1, 4], 4, 2, 64, 64),
                                           ([6007] * 7, [17] * 7, 8, 1, 128, 64)):
        check(tc.make(sum(lens), lens, counts, hq, hkv, d, page, BF16, "tree", dev, spread=1.2,
                      poison=False))


@pytest.mark.parametrize("requests,hq,hkv,d,page,most,mask", [
    (700, 4, 2, 64, 16, 2, "chain"),     # more requests than the split scans at once
    (150, 16, 8, 128, 16, 3, "random"),
    (90, 8, 1, 128, 64, 40, "tree"),     # two row tiles
    (60, 32, 1, 64, 8, 40, "random"),    # cohorts
])
def test_many_small_units(dev, requests, hq, hkv, d, page, most, mask):
    """Many units to a block, most of a tile or two, some without rows, some without tokens."""
    g = torch.Generator().manual_seed(requests)
    lens = torch.randint(0, 300, (requests,), generator=g).tolist()
    counts = torch.randint(0, most + 1, (requests,), generator=g).tolist()
    c = tc.make(requests, lens, counts, hq, hkv, d, page, BF16, mask, dev, spread=1.2)
    _, lse = check(c)
    lse = torch.nan_to_num(lse, nan=0.0, neginf=-torch.inf)
    w = torch.rand(requests, hkv, 290, generator=g).to(dev)
    factors = (torch.rand(c["q"].shape[0], generator=g) < 0.5).float().to(dev)
    want, tol = tc.weights(c, lse, w, factors)
    got = accumulate(c, lse, w, torch.zeros_like(w), row_factors=factors)
    for b, n in enumerate(lens):
        n = min(n, 290)
        tc.compare(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"request {b}")


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes and 2^31 elements, its pages at both ends used."""
    page, hkv, d = 64, 8, 128
    blocks = 17500  # x 64 x 8 x 256 = 2.3e9 elements
    kv = torch.zeros(blocks, page, hkv, 2 * d, dtype=BF16, device=dev)
    c = tc.make(13, [190, 100], [4, 2], 16, 8, d, page, BF16, "tree", "cpu", poison=False)
    where = torch.tensor([0, 17499, 17498, 8000, 1, 17400, 9, 12000, 16500])[: c["kv"].shape[0]]
    small = c["kv"]
    out0, lse0 = call(tc.to(c, dev))
    kv[where.to(dev)] = small.to(dev)
    big = tc.to(c, dev)
    big.update(k=kv[..., :d], v=kv[..., d:], table=where[c["table"].long()].to(torch.int32).to(dev))
    out, lse = call(big)
    assert torch.equal(out, out0) and torch.equal(lse, lse0)
    w = torch.zeros(2, 8, 190, device=dev)
    from qsa_vllm_b200.eviction import accumulate_attention_weights as acc
    more = dict(max_query_len=4, tree_mask=big["mask"])
    a = acc(big["q"], big["k"], big["table"], big["lens"], big["start"], lse, w, w.clone(), **more)
    s = tc.to(c, dev)
    b = acc(s["q"], s["k"], s["table"], s["lens"], s["start"], lse, w, w.clone(), **more)
    assert torch.equal(a, b) and a.any()


def test_repeats_are_bitwise_and_streams_do_not_meet(dev):
    """Calls at once on two streams, each with its own workspace, and the same call again."""
    cs = [tc.make(14 + i, [3000, 2500], [8, 16], 16, 2, 128, 16, BF16, "tree", dev, poison=False)
          for i in range(2)]
    alone = [call(c) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(c))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, alone[i][0]) and torch.equal(lse, alone[i][1])


def test_captured_graphs_that_share_a_workspace(dev):
    """Two captured calls replayed in turn over one workspace, with lengths that change between
    replays; captured with the longest lengths in mind, replayed with shorter ones."""
    from qsa_vllm_b200.tree_attention import tree_attention_workspace_bytes
    cs = [tc.make(20, [3000, 2500], [8, 16], 16, 2, 128, 16, BF16, "tree", dev, poison=False),
          tc.make(21, [4000], [5], 8, 8, 64, 64, F16, "tree", dev, poison=False)]
    need = max(tree_attention_workspace_bytes(c["q"].shape[0], len(c["lens"]), c["q"].shape[1],
                                              c["hkv"], c["d"], c["most"]) for c in cs)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    graphs, outs = [], []
    for c in cs:
        out = torch.zeros_like(c["q"])
        lse = torch.zeros(c["q"].shape[:2], device=dev)
        call(c, out=out, lse=lse, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c, out=out, lse=lse, workspace=ws)
        graphs.append(g)
        outs.append((out, lse))
    for less in (0, 700, 1999):
        for c in cs:
            c["lens"].sub_(less)
        for g in graphs:
            g.replay()
        for c, (out, lse) in zip(cs, outs):
            want, tol, z, ztol = tc.attention(c)
            tc.compare(out, want, tol, "out")
            tc.compare(lse, z, ztol, "lse")
        for c in cs:
            c["lens"].add_(less)


# ------------------------------------------------------------------------------------ weights

def accumulate(c, lse, w, out=None, **more):
    from qsa_vllm_b200.eviction import accumulate_attention_weights
    more.setdefault("max_query_len", c["most"])
    return accumulate_attention_weights(c["q"], c["k"], c["table"], c["lens"], c["start"], lse, w,
                                        out, tree_mask=c["mask"], **more)


@pytest.mark.parametrize("lens,counts,hq,hkv,d,page,dtype,mask", CASES)
@pytest.mark.parametrize("apart", [False, True])
def test_weights_match_definition(dev, lens, counts, hq, hkv, d, page, dtype, mask, apart):
    from qsa_vllm_b200 import _lib
    c = tc.make(sum(lens) + d, lens, counts, hq, hkv, d, page, dtype, mask, dev, spread=1.5, pad=2)
    _, lse = call(c)
    lse = torch.nan_to_num(lse, nan=0.0, neginf=-torch.inf)
    g = torch.Generator().manual_seed(1)
    cap = max(lens) + 5 if apart else max(max(lens) - 3, 1)
    w = torch.rand(len(lens), hkv, cap, generator=g).to(dev)
    factors = None
    if apart:
        factors = (torch.rand(c["q"].shape[0], generator=g) < 0.6).float().to(dev)
        factors *= torch.rand(c["q"].shape[0], generator=g).to(dev) + 0.5
    want, tol = tc.weights(c, lse, w, factors)
    out = torch.full_like(w, -3.0) if apart else None
    before = w.clone()
    got = accumulate(c, lse, w, out, row_factors=factors)
    assert got is (out if apart else w)
    for b, n in enumerate(lens):
        n = min(n, cap)
        tc.compare(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"request {b}")
        assert torch.equal(got[b, :, n:], out[b, :, n:] if apart else before[b, :, n:])
        if apart:
            assert (got[b, :, n:] == -3).all() and torch.equal(w, before)
    assert _lib.device_error_poll() == 0


@pytest.mark.parametrize("page,d", [(16, 128), (64, 64), (5, 64)])
def test_weights_of_unmapped_pages_and_rows_left_out(dev, page, d):
    """Rejected rows may hold anything; unmapped tokens receive nothing; weights add up to the
    counted rows."""
    c = tc.make(30, [500, 260, 100], [6, 3, 5], 8, 2, d, page, BF16, "tree", "cpu")
    c["table"][0, 1] = -1
    c["table"][1, 2] = c["kv"].shape[0]
    c["q"][2] = float("nan")
    c = tc.to(c, dev)
    _, lse = call(c)
    factors = torch.ones(14, device=dev)
    factors[2] = 0
    factors[10] = 0
    lse[10] = float("nan")
    w = accumulate(c, lse, torch.zeros(3, 2, 500, device=dev), row_factors=factors)
    clean = dict(c, q=torch.nan_to_num(c["q"], 0.0))
    want, tol = tc.weights(clean, torch.nan_to_num(lse, 0.0), torch.zeros(3, 2, 500), factors)
    tc.compare(w, want, tol, "weights")
    assert (w[0, :, page:2 * page] == 0).all()
    rows = torch.tensor([5, 3, 4]) * 4.0  # counted rows x heads of a group
    assert (w.sum(-1).cpu() - rows[:, None]).abs().max() < 1e-3


@pytest.mark.parametrize("value", [-1.5, float("inf"), 1e-30, 3e38])
@pytest.mark.parametrize("page", [16, 5])
def test_weights_take_any_factor(dev, value, page):
    c = tc.make(33, [300, 150], [9, 4], 8, 2, 64, page, BF16, "random", dev, poison=False)
    _, lse = call(c)
    lse = torch.nan_to_num(lse, neginf=-torch.inf)
    factors = torch.ones(13, device=dev)
    factors[[2, 11]] = value
    got = accumulate(c, lse, torch.zeros(2, 2, 300, device=dev), row_factors=factors)
    want, tol = tc.weights(c, lse, torch.zeros(2, 2, 300), factors)
    fine = want.isfinite()
    assert torch.equal(got.isfinite().cpu(), fine & (want.abs() < 3.4e38))
    fine &= want.abs() < 3.4e38
    tc.compare(torch.where(fine.to(dev), got, 0.0), torch.where(fine, want, 0.0),
               torch.where(fine, tol, 0.0), "weights")


def test_weights_without_rows_copy(dev):
    c = tc.make(31, [64, 30], [0, 0], 4, 2, 64, 16, BF16, "chain", dev)
    w = torch.rand(2, 2, 64, device=dev)
    out = torch.full_like(w, -1.0)
    accumulate(c, torch.empty(0, 4, device=dev), w, out)
    assert torch.equal(out[0], w[0]) and torch.equal(out[1, :, :30], w[1, :, :30])
    assert (out[1, :, 30:] == -1).all()


def test_weights_captured_add_up(dev):
    c = tc.make(32, [900, 1200], [4, 7], 8, 2, 128, 16, BF16, "tree", dev, poison=False)
    _, lse = call(c)
    w = torch.zeros(2, 2, 1200, device=dev)
    accumulate(c, lse, w)
    once = w.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accumulate(c, lse, w)
    w.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, once)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.allclose(w, 2 * once, rtol=2.0 ** -20)


@pytest.mark.parametrize("page,d", [(16, 128), (64, 64), (5, 64)])
@pytest.mark.parametrize("factored", [False, True])
def test_weights_of_rows_with_heads_left_out(dev, page, d, factored):
    """A head whose log-sum-exp is -inf gives nothing, whatever it holds; the row's other heads
    give what they give, whichever of them it is.  More rows than a pass takes."""
    c = tc.make(34, [700, 260, 90], [70, 3, 5], 8, 2, d, page, BF16, "tree", dev, poison=False)
    _, lse = call(c)
    lse[:, 0] = -torch.inf           # the first head of the first group, of every row
    lse[3:60:7, 4:7] = -torch.inf    # all but the last head of the second
    lse[5] = lse[71] = -torch.inf    # whole rows
    lse[9, 5] = -torch.inf
    c["q"][9, 5] = float("nan")
    factors = torch.linspace(0.25, 2, 78).to(dev) if factored else None
    if factored:
        factors[8::9] = 0
    got = accumulate(c, lse, torch.ones(3, 2, 700, device=dev), row_factors=factors)
    clean = dict(c, q=torch.nan_to_num(c["q"], 0.0))
    want, tol = tc.weights(clean, lse, torch.ones(3, 2, 700), factors)
    tc.compare(got, want, tol, "weights")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,count,at", [(64, 1, 0), (128, 1, 0), (128, 16, 70001), (64, 40, 0),
                                        (128, 40, 0)])
def test_many_light_tokens_beside_a_heavy_one(dev, dtype, d, count, at):
    """131072 tokens, of which one holds almost all of the weight: what the others give together
    is seen although each is far below the heavy one, down to 2^-24.6.

    The light tokens' values are 1 and the heavy one's 0, so an output is n p / (1 + n p).  p is
    rounded to the type (half a step, and no finer than 2^-32 of the heavy token's in fp16);
    sums are chains of at most n / 16 products of 16 tokens, each to 2^-23, and of 64 + n / 128
    exponentials, each to 2^-24; the output is rounded once."""
    n, batch, hkv, group, page = 131072, 64, 4, 8, 64
    kv = torch.zeros(n // page, page, hkv, 2 * d, dtype=dtype, device=dev)
    kv[at // page, at % page, :, 0] = 17.0625
    gap = float(kv[at // page, at % page, 0, 0])  # as the type holds it
    kv[..., d:] = 1
    kv[at // page, at % page, :, d:] = 0
    q = torch.zeros(batch * count, hkv * group, d, dtype=dtype, device=dev)
    part = torch.tensor([1.0, 0.75] * (hkv * group // 2), dtype=torch.float64)
    q[..., 0] = part.to(dtype).to(dev)
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(batch, -1).contiguous()
    start = torch.arange(batch + 1, dtype=torch.int32, device=dev) * count
    lens = torch.full((batch,), n, dtype=torch.int32, device=dev)
    from qsa_vllm_b200.tree_attention import tree_paged_attention
    lse = torch.empty(batch * count, hkv * group, device=dev)
    out = tree_paged_attention(q, kv[..., :d], kv[..., d:], table, lens, start,
                               max_query_len=count, scale=1.0, lse=lse)
    light = (n - count + torch.arange(count).double())[:, None]  # seen, without the heavy one
    p = (-gap * part).exp()[None]
    want = light * p / (1 + light * p)
    eps = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -32 if dtype == F16 else 0.0
    tol = want * (eps + n / 16 * 2.0 ** -23 + (64 + n / 128) * 2.0 ** -24 + 2.0 ** -18) \
        + light * tiny / (1 + light * p)
    tol = tol + eps * (want + tol)
    off = (out.double().cpu().view(batch, count, -1, d) - want[..., None]).abs()
    assert (off <= tol[..., None]).all(), (off / want[..., None]).amax((0, 1, 3))
    z = gap * part + torch.log1p(light * p)
    assert ((lse.double().cpu().view(batch, count, -1) - z).abs() <= 2.0 ** -13).all()
