"""The serving operators around a paged cache, case by case: rotary positions (with and
without the store to the cache), attention of a tree of drafted tokens, the attention weight
that each cached token has received, the eviction that goes by it, and the compaction that
commits an accepted path.

``run`` is one pass through one of them: with ``own`` false from elementary torch operations in
32 bits, with ``own`` true through ``qsa_vllm_b200``.  ``exact`` is the definition in 64 bits.
Every operator writes to buffers apart from what it reads, so a pass can be repeated.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda"


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token of each of 64 requests before a decode step: a few hundred kilobytes, so
        # the call's own latency is what counts
        dict(name="rotary_decode", op="rotary", tokens=64, hq=32, hkv=4, d=128, rot=64,
             interleaved=False, inverse=False, scaling="none", far=32768, dtype="bf16"),
        # the projections of a chunked prefill step of 2 x 4096 tokens, whole head rotated,
        # positions stretched for a long context, keys and values stored to scattered pages
        dict(name="rotary_store_prefill", op="store", tokens=8192, hq=16, hkv=2, d=128, rot=128,
             interleaved=True, scaling="yarn", far=131072, page=16, dtype="bf16"),
        # four requests of 2048 tokens that verify 8 drafted tokens each: the small end
        dict(name="tree_small", op="tree", batch=4, ctx=2048, tree=8, hq=16, hkv=2, d=128,
             page=16, even=True, dtype="bf16"),
        # the serving point: 64 requests of 8k to 32k tokens, trees of 16 nodes
        dict(name="tree_serving", op="tree", batch=64, ctx=32768, tree=16, hq=32, hkv=4, d=128,
             page=64, even=False, dtype="bf16"),
        # few requests with very long contexts and wide trees (64 nodes x 8 query heads per
        # KV head): the heaviest verification step
        dict(name="tree_long", op="tree", batch=8, ctx=131072, tree=64, hq=32, hkv=4, d=128,
             page=64, even=True, dtype="bf16"),
        # one row per request, odd lengths, head size 64, no grouping of query heads: a plain
        # decode step of a dense layer
        dict(name="tree_single", op="tree", batch=61, ctx=4099, tree=1, hq=8, hkv=8, d=64,
             page=32, even=False, dtype="fp16"),
        # weights of one decoded token per request over short contexts
        dict(name="weights_small", op="weights", batch=4, ctx=2048, tree=1, hq=16, hkv=2, d=128,
             page=16, even=True, dtype="bf16"),
        # weights of the accepted rows of the serving point's verification step
        dict(name="weights_serving", op="weights", batch=64, ctx=32768, tree=16, hq=32, hkv=4,
             d=128, page=64, even=False, dtype="bf16"),
        # 256 requests kept at 2048 tokens: each has grown by up to 64 since the last time
        dict(name="evict_steady", op="evict", batch=256, ctx=2112, budget=2048, sinks=4,
             recent=512, hq=16, hkv=2, d=128, page=16, even=True, dtype="bf16"),
        # long prompts cut to 8192 tokens once they have been read
        dict(name="evict_prompt", op="evict", batch=8, ctx=131072, budget=8192, sinks=16,
             recent=1024, hq=32, hkv=4, d=128, page=64, even=False, dtype="bf16"),
        # the accepted path of a 16-node tree, at most 5 tokens, for 64 requests
        dict(name="compact_commit", op="compact", batch=64, ctx=4096, count=5, spread=16,
             start=3001, hq=32, hkv=4, d=128, page=64, dtype="bf16"),
        # half of a 16k passage dropped from the middle of 16 contexts
        dict(name="compact_passage", op="compact", batch=16, ctx=32768, count=8191, spread=16384,
             start=7777, hq=32, hkv=4, d=128, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "store", "tree", "tree", "weights", "evict", "compact"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 7, 8, 16])
    hq = hq if hq <= 64 else 8 * hkv
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("rotary", "store"):
        tokens = _log(rng, 1, 8192)
        case = dict(op=op, tokens=tokens, hq=min(hq, 32), hkv=min(hkv, 4), d=d,
                    rot=rng.choice([32, 64, d, d - 16]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    far=_log(rng, 64, 1 << 20), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        case["hq"] -= case["hq"] % case["hkv"]
        if op == "rotary":
            case["inverse"] = rng.random() < 0.3
        else:
            case["page"] = page
        return case
    ctx = _log(rng, 17, 65536)
    most = 1 << 20  # cached tokens in all
    batch = min(_log(rng, 1, 128), max(1, most // ctx))
    even = rng.random() < 0.5
    base = dict(op=op, batch=batch, ctx=ctx, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype)
    if op in ("tree", "weights"):
        tree = min(_log(rng, 1, 64), ctx)
        while batch * ctx * tree * hq > (1 << 20) * 64 * 16 and tree > 1:
            tree = tree // 2
        return dict(base, tree=tree, even=even)
    if op == "evict":
        budget = rng.randint(max(1, ctx // 8), ctx)
        sinks = rng.randint(0, min(16, budget))
        recent = rng.randint(0, (budget - sinks) // 2)
        return dict(base, budget=budget, sinks=sinks, recent=recent, even=even)
    spread = _log(rng, 1, max(1, ctx // 2))
    start = rng.randint(0, ctx - spread)
    return dict(base, count=rng.randint(1, spread), spread=spread, start=start)


# ---------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(DTYPES[dtype])


def _lengths(case, seed):
    """Cached tokens per request, evenly from a quarter of the context to all of it (their sum
    is the same for every seed), or all at the context's end."""
    batch, ctx = case["batch"], case["ctx"]
    low = ctx if case.get("even", True) else max(min(ctx, case.get("tree", 1)), ctx // 4)
    steps = torch.linspace(ctx, low, batch, dtype=torch.float64).round().to(torch.int32)
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(seed))
    return steps[order].to(DEVICE)


def _cache(case, g, more=0):
    """A pool of pages in one buffer, keys and values side by side, and each request's pages,
    scattered over it; ``more``: pages of each request's second table."""
    batch, page = case["batch"], case["page"]
    width = -(-case["ctx"] // page)
    total = batch * (width + more)
    kv = torch.empty(total, page, case["hkv"], 2 * case["d"], dtype=DTYPES[case["dtype"]],
                     device=DEVICE)
    kv.normal_(generator=g)
    pages = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    first = pages[: batch * width].view(batch, width)
    return kv, first, pages[batch * width:].view(batch, more)


def _trees(batch, tree, seed):
    """[batch, tree, tree]: node i sees itself and its ancestors; each node's parent is one of
    the eight nodes before it, or the end of the context."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros(batch, tree, tree, dtype=torch.bool)
    each = torch.arange(batch)
    for i in range(tree):
        parent = i - 1 - torch.randint(0, min(i, 8) + 1, (batch,), generator=g)
        mask[:, i] = torch.where((parent >= 0)[:, None], mask[each, parent.clamp(min=0)], False)
        mask[:, i, i] = True
    return mask


def _frequencies(case):
    """Angle per position of each pair of dimensions, and the factor on the rotated values."""
    half, base, reach = case["rot"] // 2, 10000.0, 4.0
    i = torch.arange(half, dtype=torch.float64)
    if case["scaling"] == "ntk":
        base = base * reach ** (case["rot"] / max(case["rot"] - 2, 1))
    f = base ** (-i / half)
    if case["scaling"] == "linear":
        f = f / reach
    if case["scaling"] == "yarn":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f / reach * (1 - keep) + f * keep, 0.1 * math.log(reach) + 1
    return f, 1.0


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = dict(op=op)
    if op in ("rotary", "store"):
        n, d = case["tokens"], case["d"]
        f, s["factor"] = _frequencies(case)
        s["frequencies"] = f.to(DEVICE)
        s["interleaved"] = case["interleaved"]
        s["inverse"] = case.get("inverse", False)
        s["positions"] = torch.randint(0, case["far"], (n,), generator=g, device=DEVICE)
        # one projection's output, split into heads as a layer splits it
        qkv = _normal(g, (n, (case["hq"] + 2 * case["hkv"]) * d), case["dtype"])
        parts = qkv.split([case["hq"] * d, case["hkv"] * d, case["hkv"] * d], dim=1)
        s["q"], s["k"], s["v"] = (p.unflatten(1, (-1, d)) for p in parts)
        s["q_out"] = torch.empty(n, case["hq"], d, dtype=s["q"].dtype, device=DEVICE)
        if op == "rotary":
            s["k_out"] = torch.empty(n, case["hkv"], d, dtype=s["q"].dtype, device=DEVICE)
        else:
            blocks = -(-n // case["page"]) + 3
            s["kv"] = torch.zeros(blocks, case["page"], case["hkv"], 2 * d, dtype=s["q"].dtype,
                                  device=DEVICE)
            s["slots"] = torch.randperm(blocks * case["page"], generator=g, device=DEVICE)[:n]
        return s
    d, hkv, batch = case["d"], case["hkv"], case["batch"]
    s["d"] = d
    if op in ("tree", "weights"):
        tree = case["tree"]
        s["max_query_len"] = tree
        s["seq_lens"] = _lengths(case, seed)
        # trees end early for some requests
        rows = (tree - torch.arange(batch) % 3).clamp(min=1)
        start = torch.cat([torch.zeros(1, dtype=torch.int64), rows.cumsum(0)]).to(torch.int32)
        total = int(start[-1])
        s["query_start_loc"] = start.to(DEVICE)
        s["kv"], s["block_table"], _ = _cache(case, g)
        s["q"] = _normal(g, (total, case["hq"], d), case["dtype"], 1.5)
        of = torch.repeat_interleave(torch.arange(batch), rows)
        s["tree_mask"] = _trees(batch, tree, seed)[of, torch.arange(total) - start[of]].to(DEVICE)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(total, case["hq"], dtype=torch.float32, device=DEVICE)
        if op == "weights":
            # the log-sum-exp that the attention left, and the rows that were accepted
            s["lse"] = _plain_tree(s, 1.0 / math.sqrt(d))[1]
            s["factors"] = (torch.rand(total, generator=g, device=DEVICE) < 0.4).float()
            s["weights"] = torch.rand(batch, hkv, case["ctx"], generator=g, device=DEVICE)
            s["weights"] *= torch.arange(case["ctx"], device=DEVICE) < s["seq_lens"][:, None, None]
            s["weights_out"] = torch.zeros_like(s["weights"])
        return s
    s["pages_out"] = -(-(case["budget"] if op == "evict" else case["ctx"]) // case["page"])
    s["kv"], s["block_table"], s["out_table"] = _cache(case, g, s["pages_out"])
    if op == "evict":
        s["seq_lens"] = _lengths(case, seed)
        s["budget"], s["sinks"], s["recent"] = case["budget"], case["sinks"], case["recent"]
        # what accumulates: a few heavy tokens, many light ones, some never attended
        w = (2.0 * torch.randn(batch, hkv, case["ctx"], generator=g, device=DEVICE)).exp()
        seen = torch.rand(batch, hkv, case["ctx"], generator=g, device=DEVICE) < 0.8
        s["weights"] = torch.where(seen, w, 0.0)
        s["weights_out"] = torch.zeros_like(w)
        s["kept"] = torch.empty(batch, hkv, case["budget"], dtype=torch.int32, device=DEVICE)
    else:
        at = torch.rand(batch, case["spread"], generator=g, device=DEVICE).argsort(1)
        at = at[:, : case["count"]].sort(1).values + case["start"]
        s["indices"] = at.to(torch.int32)
        s["starts"] = torch.full((batch,), case["start"], dtype=torch.int32, device=DEVICE)
    return s


# -------------------------------------------------------------------------------- the passes

def _turn(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    a, rest = x[..., :rot].float(), x[..., rot:]
    if interleaved:
        p, q = a[..., 0::2], a[..., 1::2]
        turned = torch.stack([p * cos - q * sin, q * cos + p * sin], dim=-1).flatten(-2)
    else:
        p, q = a.chunk(2, dim=-1)
        turned = torch.cat([p * cos - q * sin, q * cos + p * sin], dim=-1)
    return torch.cat([turned.to(x.dtype), rest], dim=-1)


def _plain_rotary(s):
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    sin = -sin if s["inverse"] else sin
    return (_turn(s["q"], cos, sin, s["interleaved"]), _turn(s["k"], cos, sin, s["interleaved"]))


def _plain_store(s):
    q, k = _plain_rotary(s)
    rows = s["kv"].flatten(0, 1)
    rows[s["slots"]] = torch.cat([k, s["v"]], dim=-1)
    return q, s["kv"]


def _padded(s):
    """Rows of each request side by side: their numbers, and which are rows at all."""
    start = s["query_start_loc"].long()
    at = start[:-1, None] + torch.arange(s["max_query_len"], device=start.device)
    return at.clamp(max=s["q"].shape[0] - 1), at < start[1:, None]


def _plain_scores(s, scale):
    """Scaled scores [batch, kv head, row, head of group, token], -inf where not to be seen."""
    d = s["d"]
    at, real = _padded(s)
    q = s["q"][at].float() * scale
    batch, rows, hq = q.shape[:3]
    hkv = s["kv"].shape[2]
    k = s["kv"][..., :d][s["block_table"].long()].flatten(1, 2).float()
    q = q.view(batch, rows, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)
    score = torch.matmul(q.reshape(batch, hkv, -1, d), k.permute(0, 2, 3, 1))
    score = score.view(batch, hkv, rows, hq // hkv, -1)
    token = torch.arange(score.shape[-1], device=score.device)
    length = s["seq_lens"].long()
    count = s["query_start_loc"].diff().long()
    node = token - (length - count)[:, None]
    width = s["tree_mask"].shape[1]
    seen = s["tree_mask"][at].gather(2, node.clamp(0, width - 1)[:, None].expand(-1, rows, -1))
    seen = (seen | (node < 0)[:, None]) & (token < length[:, None])[:, None]
    return score.masked_fill_(~seen[:, None, :, None], float("-inf")), at, real


def _plain_tree(s, scale):
    d = s["d"]
    score, at, real = _plain_scores(s, scale)
    batch, hkv, rows, group, n = score.shape
    high = score.amax(-1, keepdim=True)
    high = torch.where(high.isinf(), 0.0, high)
    p = score.sub_(high).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["kv"][..., d:][s["block_table"].long()].flatten(1, 2).float().permute(0, 2, 1, 3)
    o = torch.matmul(p.flatten(2, 3), v).view(batch, hkv, rows, group, d)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (high + total.log()).squeeze(-1)
    out, lse_out = torch.zeros_like(s["out"]), torch.full_like(s["lse"], float("-inf"))
    out[at[real]] = o.permute(0, 2, 1, 3, 4).flatten(2, 3)[real].to(out.dtype)
    lse_out[at[real]] = lse.permute(0, 2, 1, 3).flatten(2, 3)[real]
    return out, lse_out


def _plain_weights(s, scale):
    score, at, real = _plain_scores(s, scale)
    batch, hkv, rows, group, n = score.shape
    lse = s["lse"][at].view(batch, rows, hkv, group).permute(0, 2, 1, 3)
    factor = torch.where(real, s["factors"][at], 0.0)
    p = score.sub_(lse[..., None]).exp_() * factor[:, None, :, None, None]
    return s["weights"] + p.sum((2, 3))[..., : s["weights"].shape[-1]]


def _slots(table, token, page):
    """Slots of tokens [batch, heads, n] in the pool (0 for a token below 0)."""
    token = token.clamp(min=0).long()
    return table.long()[:, None].expand(-1, token.shape[1], -1).gather(2, token // page) * page \
        + token % page


def _plain_move(kv, table, out_table, source, target, moved):
    """Rows of each head from the tokens ``source`` to the tokens ``target``."""
    page, heads = kv.shape[1], kv.shape[2]
    head = torch.arange(heads, device=kv.device)[:, None].expand_as(source)[moved]
    rows = kv.flatten(0, 1)
    rows[_slots(out_table, target, page)[moved], head] = \
        rows[_slots(table, source, page)[moved], head]


def _plain_evict(s):
    w, length = s["weights"], s["seq_lens"].long()[:, None, None]
    token = torch.arange(w.shape[-1], device=w.device)
    kept_anyway = (token < s["sinks"]) | (token >= length - s["recent"])
    rank = torch.where(kept_anyway, float("inf"), w)
    rank = torch.where(token < length, rank, -1.0)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., : s["budget"]]
    count = length.clamp(max=s["budget"])
    here = torch.arange(order.shape[-1], device=w.device) < count
    order = torch.where(here, order, w.shape[-1]).sort(-1).values
    kept = torch.where(here, order, -1)
    out = torch.zeros_like(w)
    out[..., : order.shape[-1]] = torch.where(here, w.gather(2, kept.clamp(min=0)), 0.0)
    target = torch.arange(order.shape[-1], device=w.device).expand_as(kept)
    _plain_move(s["kv"], s["block_table"], s["out_table"], kept, target, here.expand_as(kept))
    return kept.to(torch.int32), count.flatten().to(torch.int32), out, s["kv"]


def _plain_compact(s):
    source = s["indices"].long()[:, None].expand(-1, s["kv"].shape[2], -1)
    target = s["starts"].long()[:, None, None] \
        + torch.arange(source.shape[2], device=source.device).expand_as(source)
    _plain_move(s["kv"], s["block_table"], s["out_table"], source, target, source >= 0)
    return s["kv"]


def run(s):
    op = s["op"]
    if not own:
        if op == "rotary":
            return _plain_rotary(s)
        if op == "store":
            return _plain_store(s)
        if op == "tree":
            return _plain_tree(s, 1.0 / math.sqrt(s["d"]))
        if op == "weights":
            return _plain_weights(s, 1.0 / math.sqrt(s["d"]))
        return _plain_evict(s) if op == "evict" else _plain_compact(s)
    if op == "rotary":
        from qsa_vllm_b200.rotary import rotary_embed
        return rotary_embed(s["q"], s["k"], s["positions"], s["frequencies"],
                            interleaved=s["interleaved"], inverse=s["inverse"],
                            factor=s["factor"], q_out=s["q_out"], k_out=s["k_out"])
    d = s["q"].shape[-1] if op == "store" else s["d"]
    k_cache, v_cache = s["kv"][..., :d], s["kv"][..., d:]
    if op == "store":
        from qsa_vllm_b200.rotary import rotary_store
        q = rotary_store(s["q"], s["k"], s["v"], s["positions"], s["frequencies"], k_cache,
                         v_cache, s["slots"], interleaved=s["interleaved"], factor=s["factor"],
                         q_out=s["q_out"])
        return q, s["kv"]
    if op == "tree":
        from qsa_vllm_b200.tree_attention import tree_paged_attention
        out = tree_paged_attention(s["q"], k_cache, v_cache, s["block_table"], s["seq_lens"],
                                   s["query_start_loc"], s["out"], lse=s["lse"],
                                   max_query_len=s["max_query_len"], tree_mask=s["tree_mask"])
        return out, s["lse"]
    if op == "weights":
        from qsa_vllm_b200.eviction import accumulate_attention_weights
        return accumulate_attention_weights(
            s["q"], k_cache, s["block_table"], s["seq_lens"], s["query_start_loc"], s["lse"],
            s["weights"], s["weights_out"], max_query_len=s["max_query_len"],
            tree_mask=s["tree_mask"], row_factors=s["factors"])
    from qsa_vllm_b200.eviction import cache_compact, cache_evict
    if op == "evict":
        kept, count = cache_evict(s["weights"], s["seq_lens"], s["block_table"], k_cache, v_cache,
                                  s["budget"], sinks=s["sinks"], recent=s["recent"],
                                  out_table=s["out_table"], weights_out=s["weights_out"],
                                  kept=s["kept"])
        return kept, count, s["weights_out"], s["kv"]
    cache_compact(k_cache, v_cache, s["block_table"], s["indices"], s["starts"],
                  out_table=s["out_table"])
    return s["kv"]


# ------------------------------------------------------------------------------ what it takes

def _rows_of(case):
    return sum(max(1, case["tree"] - b % 3) for b in range(case["batch"]))


def _pairs_of(case):
    """Sum over requests of rows x cached tokens, and of cached tokens."""
    batch, ctx = case["batch"], case["ctx"]
    low = ctx if case.get("even", True) else max(min(ctx, case.get("tree", 1)), ctx // 4)
    tokens = batch * (ctx + low) / 2
    return tokens * _rows_of(case) / batch if "tree" in case else 0, tokens


def work(case):
    op, d, size = case["op"], case["d"], BYTES[case["dtype"]]
    if op in ("rotary", "store"):
        n, heads = case["tokens"], case["hq"] + case["hkv"] * (2 if op == "store" else 1)
        return {"bytes": 2.0 * n * heads * d * size + 8 * n * (2 if op == "store" else 1),
                "flops": 3.0 * n * (case["hq"] + case["hkv"]) * case["rot"]}
    row = case["hkv"] * d * size
    if op in ("tree", "weights"):
        pairs, tokens = _pairs_of(case)
        rows = _rows_of(case)
        ends = rows * case["hq"] * 4 + rows * case["tree"]
        if op == "tree":
            return {"bytes": 2.0 * tokens * row + 2 * rows * case["hq"] * d * size + ends,
                    "flops": 4.0 * pairs * case["hq"] * d}
        return {"bytes": tokens * (row + 8.0 * case["hkv"]) + rows * case["hq"] * d * size + ends,
                "flops": 2.0 * pairs * case["hq"] * d}
    if op == "evict":
        _, tokens = _pairs_of(case)
        kept = case["batch"] * min(case["budget"], case["ctx"])
        return {"bytes": 4.0 * kept * row + case["hkv"] * (4 * tokens + 8 * kept), "flops": 0.0}
    moved = case["batch"] * case["count"]
    return {"bytes": 4.0 * moved * row + 4 * moved, "flops": 0.0}


# ----------------------------------------------------------------------------- the definition

def _exact_rotated(x, positions, f, factor, interleaved, inverse):
    y = x.double().clone()
    half = f.numel()
    turn = torch.polar(torch.full_like(f, factor).expand(positions.numel(), half),
                       positions.double()[:, None] * f * (-1 if inverse else 1))[:, None]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(y[..., one], y[..., two]) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_attention(s, of_request):
    """Calls of_request(request, rows, kv head, probabilities' log [row, head of group, token],
    pages) for each request and KV head, in 64 bits."""
    d, hkv = s["d"], s["kv"].shape[2]
    group = s["q"].shape[1] // hkv
    start, lens = s["query_start_loc"].tolist(), s["seq_lens"].tolist()
    page = s["kv"].shape[1]
    for b, n in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        count = hi - lo
        pages = s["kv"][s["block_table"][b, : -(-n // page)].long()].flatten(0, 1)[:n].double()
        may = torch.ones(count, n, dtype=torch.bool, device=pages.device)
        may[:, n - count:] = s["tree_mask"][lo:hi, :count]
        for h in range(hkv):
            q = s["q"][lo:hi, h * group:(h + 1) * group].double()
            score = (q.reshape(-1, d) @ pages[:, h, :d].T).view(count, group, n) / math.sqrt(d)
            score[~may[:, None].expand_as(score)] = float("-inf")
            of_request(b, slice(lo, hi), slice(h * group, (h + 1) * group), h, score,
                       pages[:, h, d:])


def _exact_moved(s, source_of, starts):
    """The pool after the moves, and nothing else changed; source_of(request, head) lists them."""
    kv, page = s["kv"].clone(), s["kv"].shape[1]
    for b in range(s["block_table"].shape[0]):
        for h in range(kv.shape[2]):
            source = source_of(b, h)
            target = starts[b] + torch.arange(source.numel(), device=source.device)
            kv[s["out_table"][b][target // page].long(), target % page, h] = \
                s["kv"][s["block_table"][b][source // page].long(), source % page, h]
    return kv.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("rotary", "store"):
        f = s["frequencies"]
        q, k = (_exact_rotated(s[x], s["positions"], f, s["factor"], s["interleaved"],
                               s["inverse"]) for x in ("q", "k"))
        if op == "rotary":
            return q, k
        kv, page = s["kv"].double(), s["kv"].shape[1]
        kv[s["slots"] // page, s["slots"] % page] = torch.cat([k, s["v"].double()], -1)
        return q, kv
    if op == "tree":
        out = torch.zeros_like(s["out"], dtype=torch.float64)
        lse = torch.zeros_like(s["lse"], dtype=torch.float64)

        def attend(b, rows, heads, h, score, values):
            lse[rows, heads] = score.logsumexp(-1)
            p = (score - lse[rows, heads][..., None]).exp()
            out[rows, heads] = (p.flatten(0, 1) @ values).view(p.shape[0], p.shape[1], -1)

        _exact_attention(s, attend)
        return out, lse
    if op == "weights":
        got = s["weights"].double()

        def add(b, rows, heads, h, score, values):
            p = (score - s["lse"][rows, heads].double()[..., None]).exp()
            p = p * s["factors"][rows].double()[:, None, None]
            got[b, h, : score.shape[-1]] += p.sum((0, 1))

        _exact_attention(s, add)
        return got
    if op == "evict":
        lens, w = s["seq_lens"].tolist(), s["weights"]
        kept = torch.full_like(s["kept"], -1)
        out = torch.zeros_like(w, dtype=torch.float64)

        def choose(b, h):
            n, first, last = lens[b], s["sinks"], s["recent"]
            if n <= s["budget"]:
                at = torch.arange(n, device=w.device)
            else:
                middle = w[b, h, first:n - last].double()
                best = (-middle).sort(stable=True).indices[: s["budget"] - first - last]
                at = torch.cat([torch.arange(first, device=w.device), best.sort().values + first,
                                torch.arange(n - last, n, device=w.device)])
            kept[b, h, : at.numel()] = at.to(torch.int32)
            out[b, h, : at.numel()] = w[b, h, at].double()
            return at

        kv = _exact_moved(s, choose, [0] * len(lens))
        return kept, torch.tensor([min(n, s["budget"]) for n in lens], dtype=torch.int32), out, kv
    source = s["indices"].long()
    return _exact_moved(s, lambda b, h: source[b], s["starts"].tolist())
