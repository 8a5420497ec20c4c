"""Rotary positions and the store to the paged cache against the definition in 64 bits.

Bound of one output y of the pair (x1, x2): half a step of its type, eps/2 |y|, and the 32-bit
arithmetic before it: the reduced angle is off by at most pi 2^-24 (half a turn rounded to 32
bits), sine and cosine by one step (2^-24), the factor's product, the two products and the sum by
half a step each, in all below 8 * 2^-24 * factor * (|x1| + |x2|).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def turned(x, positions, freq, factor, interleaved, inverse):
    """(values, bound without the last rounding) in 64 bits, on the CPU."""
    x = x.double().cpu()
    a = positions.double().cpu()[:, None] * freq.double().cpu()
    cos, sin = a.cos()[:, None], a.sin()[:, None] * (-1 if inverse else 1)
    half = freq.numel()
    y, slack = x.clone(), torch.zeros_like(x)
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    x1, x2 = x[..., one], x[..., two]
    y[..., one] = factor * (x1 * cos - x2 * sin)
    y[..., two] = factor * (x2 * cos + x1 * sin)
    for part in (one, two):
        slack[..., part] = 8 * 2.0 ** -24 * factor * (x1.abs() + x2.abs())
    return y, slack


def near(got, want, slack):
    got = got.double().cpu()
    # subnormal results of the 16-bit types are spaced by their smallest step
    tiny = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}
    eps = torch.finfo(near.dtype).eps / 2
    bound = slack + eps * (want.abs() + slack) + tiny[near.dtype]
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of bounds"


def inputs(dev, tokens, hq, hkv, d, dtype, seed, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, (hq + 2 * hkv) * d, generator=g).to(dtype).to(dev)
    q, k, v = (p.unflatten(1, (-1, d)) for p in qkv.split([hq * d, hkv * d, hkv * d], 1))
    pos = torch.randint(0, far, (tokens,), generator=g).to(dev)
    return q, k, v, pos


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot", [
    (1, 1, 1, 2, 2), (1, 16, 2, 128, 128), (7, 4, 4, 64, 64), (33, 32, 4, 128, 64),
    (5, 3, 1, 96, 32), (9, 5, 5, 80, 20), (3, 2, 1, 37, 10), (257, 7, 1, 64, 48),
    (2, 2, 2, 256, 256), (4, 1, 1, 1024, 1024)])
def test_embed_matches_definition(dev, dtype, interleaved, tokens, hq, hkv, d, rot):
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    q, k, _, pos = inputs(dev, tokens, hq, hkv, d, dtype, tokens + d)
    freq, factor = rotary_frequencies(rot, scaling="yarn", scaling_factor=4.0,
                                      original_length=4096, device=dev)
    near.dtype = dtype
    for inverse in (False, True):
        qo, ko = rotary_embed(q, k, pos, freq, interleaved=interleaved, inverse=inverse,
                              factor=factor)
        for got, x in ((qo, q), (ko, k)):
            near(got, *turned(x, pos, freq, factor, interleaved, inverse))
            assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_in_place_views_and_odd_offsets(dev, shift):
    """Views of one projection, turned in place; a start that is not 16-byte aligned takes the
    element-wise path; the values between the heads' rows are left alone."""
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    tokens, hq, hkv, d, rot = 19, 6, 2, 64, 32
    g = torch.Generator().manual_seed(5)
    buf = torch.randn(tokens, (hq + hkv) * d + 8 + shift, generator=g).to(BF16).to(dev)
    before = buf.clone()
    q = buf[:, shift:shift + hq * d].unflatten(1, (-1, d))
    k = buf[:, shift + hq * d:shift + (hq + hkv) * d].unflatten(1, (-1, d))
    pos = torch.arange(2 * tokens, device=dev)[::2]
    freq, _ = rotary_frequencies(rot, device=dev)
    want = [turned(x, pos, freq, 1.0, False, False) for x in (q, k)]
    qo, ko = rotary_embed(q, k, pos, freq, q_out=q, k_out=k)
    assert qo is q and ko is k
    near.dtype = BF16
    near(q, *want[0])
    near(k, *want[1])
    assert torch.equal(buf[:, :shift], before[:, :shift])
    assert torch.equal(buf[:, shift + (hq + hkv) * d:], before[:, shift + (hq + hkv) * d:])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot,page,fused", [
    (1, 4, 1, 64, 64, 16, True), (65, 16, 2, 128, 64, 16, True), (40, 8, 8, 64, 32, 1, False),
    (23, 3, 3, 72, 24, 5, False), (300, 32, 4, 128, 128, 64, True)])
def test_store_writes_named_slots_only(dev, dtype, tokens, hq, hkv, d, rot, page, fused):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.rotary import rotary_frequencies, rotary_store
    q, k, v, pos = inputs(dev, tokens, hq, hkv, d, dtype, tokens, far=5000)
    blocks = -(-tokens // page) + 3
    g = torch.Generator().manual_seed(9)
    if fused:
        kv = torch.randn(blocks, page, hkv, 2 * d, generator=g).to(dtype).to(dev)
        kc, vc = kv[..., :d], kv[..., d:]
    else:  # heads before slots, values apart
        kc = torch.randn(blocks, hkv, page, d, generator=g).to(dtype).to(dev).transpose(1, 2)
        vc = torch.randn(blocks, page, hkv, d, generator=g).to(dtype).to(dev)
    kc0, vc0 = kc.clone(), vc.clone()
    slots = torch.randperm(blocks * page, generator=g)[:tokens].to(dev)
    slots[::7] = -1
    freq, factor = rotary_frequencies(rot, scaling="linear", scaling_factor=2.0, device=dev)
    qo = rotary_store(q, k, v, pos, freq, kc, vc, slots, interleaved=True, factor=factor)
    near.dtype = dtype
    near(qo, *turned(q, pos, freq, factor, True, False))
    want, slack = turned(k, pos, freq, factor, True, False)
    on = (slots >= 0).cpu()
    at = slots[slots >= 0]
    got_k, got_v = kc[at // page, at % page], vc[at // page, at % page]
    near(got_k, want[on], slack[on])
    assert torch.equal(got_v, v[slots >= 0])
    kc0[at // page, at % page] = got_k
    vc0[at // page, at % page] = got_v
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)
    assert _lib.device_error_poll() == 0


def test_slot_past_the_cache_is_skipped_and_reported(dev):
    from qsa_vllm_b200 import _lib
    from qsa_vllm_b200.rotary import rotary_frequencies, rotary_store
    _, k, v, pos = inputs(dev, 3, 1, 2, 64, BF16, 1)
    kv = torch.zeros(2, 16, 2, 128, dtype=BF16, device=dev)
    slots = torch.tensor([5, 32, 1 << 40], device=dev)
    freq, _ = rotary_frequencies(64, device=dev)
    assert rotary_store(None, k, v, pos, freq, kv[..., :64], kv[..., 64:], slots) is None
    assert _lib.device_error_poll() == 2
    assert torch.equal(kv[0, 5, :, 64:], v[0])
    kv[0, 5] = 0
    assert not kv.any()


def test_far_positions_and_round_trip(dev):
    """Positions up to 2^40 keep the definition's angles; turning back returns the input to
    within the two roundings."""
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    g = torch.Generator().manual_seed(3)
    q = torch.randn(64, 2, 128, generator=g).to(dev)
    # up to 2^30 the definition's own angle is within 2^-22 radians in 64 bits
    pos = torch.randint(0, 1 << 30, (64,), generator=g).to(dev)
    freq, _ = rotary_frequencies(128, device=dev)
    y, _ = rotary_embed(q, None, pos, freq)
    want, slack = turned(q, pos, freq, 1.0, False, False)
    near.dtype = F32
    near(y, want, slack * 2)
    back, _ = rotary_embed(y, None, pos, freq, inverse=True)
    assert (back - q).abs().max() <= 32 * 2.0 ** -24 * q.abs().max()
    neg, _ = rotary_embed(q, None, -pos, freq)
    inv, _ = rotary_embed(q, None, pos, freq, inverse=True)
    assert torch.equal(neg, inv)


def test_inverse_is_the_gradient(dev):
    """The inverse against the derivative of a scalar of the outputs, by the formula and by
    differences (the map is linear, so a central difference is exact but for rounding)."""
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    g = torch.Generator().manual_seed(11)
    x = torch.randn(3, 2, 32, generator=g).to(dev)
    dy = torch.randn(3, 2, 32, generator=g).to(dev)
    pos = torch.tensor([0, 17, 4099], device=dev)
    freq, factor = rotary_frequencies(24, scaling="yarn", scaling_factor=8.0,
                                      original_length=512, device=dev)
    for interleaved in (False, True):
        dx, _ = rotary_embed(dy, None, pos, freq, interleaved=interleaved, inverse=True,
                             factor=factor)
        for at in [(0, 0, 0), (1, 1, 5), (2, 0, 13), (2, 1, 23), (1, 0, 31)]:
            e = torch.zeros_like(x)
            e[at] = 0.5
            hi, _ = rotary_embed(x + e, None, pos, freq, interleaved=interleaved, factor=factor)
            lo, _ = rotary_embed(x - e, None, pos, freq, interleaved=interleaved, factor=factor)
            slope = ((hi.double() - lo.double()) * dy.double()).sum()
            if at[-1] >= 24:  # passes through
                assert dx[at] == dy[at]
                continue
            assert abs(slope - dx[at].double()) <= 64 * 2.0 ** -24 * factor * 4
        leaf = x.double().cpu().requires_grad_()
        y, _ = _double_turn(leaf, pos, freq, factor, interleaved)
        (y * dy.double().cpu()).sum().backward()
        assert (leaf.grad - dx.double().cpu()).abs().max() <= 16 * 2.0 ** -24 * factor * 4


def _double_turn(x, positions, freq, factor, interleaved):
    a = positions.double().cpu()[:, None] * freq.double().cpu()
    cos, sin = a.cos()[:, None] * factor, a.sin()[:, None] * factor
    half = freq.numel()
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        p, q = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([p * cos - q * sin, q * cos + p * sin], -1).flatten(-2)
    else:
        p, q = rot[..., :half], rot[..., half:]
        y = torch.cat([p * cos - q * sin, q * cos + p * sin], -1)
    return torch.cat([y, rest], -1), None


def test_captured_and_replayed_on_another_stream(dev):
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    q, k, _, pos = inputs(dev, 12, 8, 2, 128, BF16, 4)
    freq, _ = rotary_frequencies(64, device=dev)
    qo, ko = torch.empty(12, 8, 128, dtype=BF16, device=dev), torch.empty(12, 2, 128, dtype=BF16,
                                                                           device=dev)
    rotary_embed(q, k, pos, freq, q_out=qo, k_out=ko)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary_embed(q, k, pos, freq, q_out=qo, k_out=ko)
    pos.add_(1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    want = rotary_embed(q, k, pos, freq)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_positions_past_what_64_bits_hold_exactly(dev):
    """Positions up to 2^52, against angles reduced with 60 decimal digits: a turn is off by at
    most 2^-54 of the position (two products and the constant 1 / 2 pi, each rounded to 2^-53 of
    position / 2 pi) and by 2^-25 for its 32-bit form; sine and cosine by 2 pi times that and two
    units of their own; y1 and y2 are a sum of two products of values up to 1."""
    import math
    from decimal import Decimal, getcontext
    from qsa_vllm_b200.rotary import rotary_embed, rotary_frequencies
    getcontext().prec = 60
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781")
    freq, _ = rotary_frequencies(32)
    pos = torch.tensor([1, 3, 4095, 2**20 + 1, 2**30 - 1, 2**33 + 5, 2**40 - 3, 2**45 + 77, 2**52])
    pos = torch.cat([pos, -pos])
    q = torch.ones(pos.numel(), 1, 32, device=dev)
    y, _ = rotary_embed(q, None, pos.to(dev), freq.to(dev))
    y = y.double().cpu()[:, 0]
    for n, at in enumerate(pos.tolist()):
        for i, f in enumerate(freq.tolist()):
            turns = Decimal(at) * Decimal(f) / two_pi
            a = 2 * math.pi * float(turns - turns.to_integral_value())
            off = 2 * math.pi * (abs(at) * f * 2.0 ** -54 + 2.0 ** -25) + 2 * 2.0 ** -24
            c, s = math.cos(a), math.sin(a)
            assert abs(y[n, i] - (c - s)) <= 2 * off + 3 * 2.0 ** -24, (at, i)
            assert abs(y[n, i + 16] - (c + s)) <= 2 * off + 3 * 2.0 ** -24, (at, i)
