"""Inputs, 64-bit definition and error bounds of the tree attention operators.

Bounds.  A score is a 32-bit sum of d products: off by at most d 2^-24 sum|q k| scale, and the
exponent's argument by a step of it, 2^-24 (|s| + |lse|) log2 e; the exponential by 2^-22.  That is
``delta``, the relative error of one weight p; the sum of n weights adds n 2^-24, in the
denominator as in the product with v.  p is rounded to the tensors' type before that product
(eps/2; below the smallest normal fp16 number by 2^-25 absolute, against a sum of at least 1),
and the output once more (eps/2).
"""

import math

import torch

BF16, F16 = torch.bfloat16, torch.float16


def make(seed, lens, counts, hq, hkv, d, page, dtype, mask="tree", dev="cpu", spread=1.0, pad=0,
         width=None, poison=True, fused=True, q_shift=0):
    """One batch.  mask: "tree", "chain", "random" (any pattern, some rows empty among the
    drafts), "none" (drafted tokens see nothing of one another)."""
    g = torch.Generator().manual_seed(seed)
    batch = len(lens)
    cols = max(1, max(-(-n // page) for n in lens))
    cols = cols if width is None else width
    blocks = batch * cols + 3
    if fused:
        kv = torch.randn(blocks, page, hkv, 2 * d, generator=g).to(dtype)
        if poison:
            kv = kv.clone()
    else:
        kv = torch.randn(blocks, hkv, page, 2 * d, generator=g).to(dtype).transpose(1, 2)
    table = torch.randperm(blocks, generator=g)[: batch * cols].view(batch, cols).to(torch.int32)
    rows = sum(counts)
    q = (torch.randn(rows + pad, hq, d + q_shift, generator=g) * spread).to(dtype)[..., q_shift:]
    start = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    tm = None
    most = max(max(counts), 1)
    if mask != "chain":
        tm = torch.zeros(rows + pad, most, dtype=torch.bool)
        for b, n in enumerate(counts):
            for i in range(n):
                row = int(start[b]) + i
                if mask == "tree":
                    parent = i - 1 - int(torch.randint(0, min(i, 4) + 1, (1,), generator=g))
                    if parent >= 0:
                        tm[row] = tm[int(start[b]) + parent]
                    tm[row, i] = True
                elif mask == "random":
                    if int(torch.randint(0, 4, (1,), generator=g)):
                        tm[row, :n] = torch.rand(n, generator=g) < 0.5
    if poison:  # what no row may read: tokens past the lengths, pages of no request
        page_of = torch.arange(cols * page) // page
        for b, n in enumerate(lens):
            at = torch.arange(min(n, cols * page), cols * page)
            kv[table[b][page_of[at]].long(), at % page] = float("nan")
        kv[[x for x in range(blocks) if x not in set(table.flatten().tolist())]] = float("inf")
    c = dict(q=q, kv=kv, k=kv[..., :d], v=kv[..., d:], table=table,
             lens=torch.tensor(lens, dtype=torch.int32), start=start, mask=tm, d=d, hkv=hkv,
             page=page, most=most, counts=counts, rows=rows)
    return to(c, dev)


def to(c, dev):
    got = {}
    for name, x in c.items():
        got[name] = x.to(dev) if isinstance(x, torch.Tensor) else x
    got["k"], got["v"] = got["kv"][..., : c["d"]], got["kv"][..., c["d"]:]
    return got


def seen(c, b):
    """[rows of b, tokens]: what each row sees, of the tokens that the table reaches."""
    n, count = int(c["lens"][b]), int(c["start"][b + 1] - c["start"][b])
    lo = int(c["start"][b])
    reach = min(n, c["table"].shape[1] * c["page"])
    t = torch.arange(reach)
    node = t - (n - count)
    if c["mask"] is None:
        ok = node[None] <= torch.arange(count)[:, None]
    else:
        m = c["mask"][lo:lo + count].bool().cpu()
        width = m.shape[1]
        ok = (node < 0)[None] | (m[:, node.clamp(0, max(width - 1, 0))] & (node < width)[None]
                                 if width else torch.zeros(count, reach, dtype=torch.bool))
    pages = c["table"][b].cpu()[t // c["page"]].long() if reach else t
    ok = ok & ((pages >= 0) & (pages < c["kv"].shape[0]))[None]
    return ok, pages, t % c["page"]


def each(c, scale):
    """(request, rows, kv head, scores [rows, group, tokens], |q||k| sums, values, seen)."""
    q, kv, d, hkv = c["q"].double().cpu(), c["kv"].double().cpu(), c["d"], c["hkv"]
    group = q.shape[1] // hkv
    for b in range(len(c["lens"])):
        lo, hi = int(c["start"][b]), int(c["start"][b + 1])
        if hi == lo:
            continue
        ok, pages, at = seen(c, b)
        rows = kv[pages.clamp(0, kv.shape[0] - 1), at]
        for h in range(hkv):
            x = q[lo:hi, h * group:(h + 1) * group]
            k, v = rows[:, h, :d], rows[:, h, d:]
            s = torch.einsum("igd,td->igt", x, torch.nan_to_num(k, 0, 0, 0)) * scale
            a = torch.einsum("igd,td->igt", x.abs(), torch.nan_to_num(k, 0, 0, 0).abs()) * scale
            yield b, slice(lo, hi), slice(h * group, (h + 1) * group), h, s, a, v, \
                ok[:, None].expand_as(s)


def attention(c, scale=None):
    """(out, its bound, lse, its bound); rows of no request hold NaN."""
    d = c["d"]
    scale = d ** -0.5 if scale is None else scale
    eps = torch.finfo(c["q"].dtype).eps / 2
    tiny = 2.0 ** -25 if c["q"].dtype == F16 else 0.0
    shape = tuple(c["q"].shape)
    out, tol = torch.full(shape, math.nan, dtype=torch.float64), torch.zeros(shape).double()
    lse = torch.full(shape[:2], math.nan, dtype=torch.float64)
    ltol = torch.zeros(shape[:2]).double()
    for b, rows, heads, h, s, a, v, ok in each(c, scale):
        n = s.shape[2]
        s = s.masked_fill(~ok, -math.inf)
        z = s.logsumexp(-1) if n else torch.full(s.shape[:2], -math.inf, dtype=torch.float64)
        p = (s - z.masked_fill(z.isinf(), 0)[..., None]).exp()
        delta = d * 2.0 ** -24 * a.masked_fill(~ok, 0).amax(-1) if n else torch.zeros_like(z)
        finite = z.masked_fill(z.isinf(), 0).abs()
        big = torch.where(ok, s, 0.0).abs().amax(-1) if n else finite
        delta = delta + 1.5 * 2.0 ** -23 * (big + finite) + 2.0 ** -21
        lse[rows, heads], ltol[rows, heads] = z, delta + n * 2.0 ** -24 + 2.0 ** -22 * (1 + finite)
        # an unseen token gives nothing, whatever its value holds
        seen_v = torch.where(ok[..., None], v, 0.0)
        out[rows, heads] = torch.einsum("igt,igtd->igd", p, seen_v)
        weight = torch.einsum("igt,igtd->igd", p, seen_v.abs())
        most = seen_v.abs().sum(2) * tiny
        tol[rows, heads] = weight * (eps + 2 * delta[..., None] + n * 2.0 ** -23) + most
        tol[rows, heads] += eps * (out[rows, heads].abs() + tol[rows, heads]) + tiny
    return out, tol, lse, ltol


def weights(c, lse, before, factors=None, scale=None):
    """(weights, bound) from the given log-sum-exps."""
    d = c["d"]
    scale = d ** -0.5 if scale is None else scale
    got = before.double().cpu().clone()
    tol = torch.zeros_like(got)
    lse = lse.double().cpu()
    for b, rows, heads, h, s, a, v, ok in each(c, scale):
        z = lse[rows, heads]
        f = torch.ones(s.shape[0]).double() if factors is None else factors.double().cpu()[rows]
        use = ok & ~z.isinf()[..., None] & (f != 0)[:, None, None]
        e = torch.where(use, s - z.masked_fill(z.isinf(), 0)[..., None], -math.inf).exp()
        # an unseen token gets nothing, of an infinite factor either
        e = torch.where(use, e * f[:, None, None], 0.0)
        n = min(s.shape[2], got.shape[2])
        delta = d * 2.0 ** -24 * a + 1.5 * 2.0 ** -23 * (
            s.abs() + z.masked_fill(z.isinf(), 0).abs()[..., None]) + 2.0 ** -21
        got[b, h, :n] += e.sum((0, 1))[:n]
        terms = s.shape[0] * s.shape[1]
        tol[b, h, :n] = ((e.abs() * (delta + terms * 2.0 ** -24)).sum((0, 1))
                         + 2.0 ** -23 * e.abs().sum((0, 1)))[:n]
        tol[b, h, :n] += 2.0 ** -23 * got[b, h, :n].abs()
    return got, tol


def compare(got, want, tol, what):
    got = got.double().cpu()
    off = (got - want).abs()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | (off <= tol))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} "
                           f"+- {tol[bad][0]}")
