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
