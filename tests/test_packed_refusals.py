"""Arguments that the packed operators refuse, in Python and at the C entries; nothing here reaches a device."""
import math

import pytest
import torch

from tagan_amd import _lib, packed

I32 = torch.int32


def _qkv(n=6, hq=4, hk=2, d=16, dtype=torch.float32):
    return torch.zeros(n, hq, d, dtype=dtype), torch.zeros(n, hk, d, dtype=dtype), torch.zeros(n, hk, d, dtype=dtype)


def _offs(*v):
    return torch.tensor(v, dtype=I32)


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(6, 4, 16, dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros(6, 2, 16, dtype=torch.bfloat16)), TypeError),
    (dict(q=torch.zeros(6, 64)), ValueError),
    (dict(q=torch.zeros(6, 3, 16)), ValueError),                          # 3 heads over 2 key heads
    (dict(q=torch.zeros(6, 4, 24)), ValueError),                          # other head size than k
    (dict(v=torch.zeros(6, 2, 8)), ValueError),
    (dict(offsets=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(offsets=torch.zeros(0, dtype=I32)), ValueError),
    (dict(offsets=torch.zeros(1, 2, dtype=I32)), ValueError),
    (dict(offsets_k=_offs(0, 3, 6)), ValueError),                         # another number of sequences
    (dict(k=torch.zeros(7, 2, 16), v=torch.zeros(7, 2, 16)), ValueError),   # needs offsets_k
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.inf), ValueError),
    (dict(scale=math.nan), ValueError),
])
def test_attention_refuses(change, error):
    q, k, v = _qkv()
    args = dict(q=q, k=k, v=v, offsets=_offs(0, 6))
    args.update(change)
    with pytest.raises(error):
        packed.attention(**args)


@pytest.mark.parametrize("d", [0, 4, 12, 20, 136, 256])
def test_attention_refuses_head_sizes(d):
    q, k, v = _qkv(d=d)
    with pytest.raises(ValueError):
        packed.attention(q, k, v, _offs(0, 6))


def test_no_cpu_path():
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="HIP device"):
        packed.attention(q, k, v, _offs(0, 6))
    with pytest.raises(RuntimeError, match="HIP device"):
        packed.rotary(q, k, torch.arange(6), packed.rotary_frequencies(16)[0])
    c = torch.zeros(1, 8, 2, 16)
    with pytest.raises(RuntimeError, match="HIP device"):
        packed.cached_attention(q[None], c, c, _offs(6))
    with pytest.raises(RuntimeError, match="HIP device"):
        packed.rotary_append(q[None], k[None], v[None], c, c.clone(), _offs(0), packed.rotary_frequencies(16)[0])


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(6, 4, 16, dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros(5, 2, 16)), ValueError),
    (dict(k=torch.zeros(6, 2, 8)), ValueError),
    (dict(q=torch.zeros(6, 0, 16)), ValueError),
    (dict(positions=torch.arange(5)), ValueError),
    (dict(positions=torch.arange(6).short()), TypeError),
    (dict(inv_freq=torch.ones(9, dtype=torch.float64)), ValueError),     # more pairs than the head has
    (dict(inv_freq=torch.ones(0, dtype=torch.float64)), ValueError),
    (dict(inv_freq=torch.ones(8, dtype=torch.bfloat16)), TypeError),
    (dict(scale=math.nan), ValueError),
])
def test_rotary_refuses(change, error):
    q, k, _ = _qkv()
    args = dict(q=q, k=k, positions=torch.arange(6), inv_freq=torch.ones(8, dtype=torch.float64))
    args.update(change)
    with pytest.raises(error):
        packed.rotary(**args)


@pytest.mark.parametrize("kw", [dict(dim=3), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.5),
                                dict(dim=8, scaling="twice"), dict(dim=2, scaling="base", factor=2.0),
                                dict(dim=8, scaling="parts", fast=1.0, slow=1.0)])
def test_rotary_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        packed.rotary_frequencies(**kw)


def test_rotary_frequencies_formulas():
    f, s = packed.rotary_frequencies(8)
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(packed.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    b, _ = packed.rotary_frequencies(8, scaling="base", factor=4.0)
    assert b[0] == 1 and abs(float(b[-1] * 4 / f[-1]) - 1) < 1e-12
    p, s = packed.rotary_frequencies(64, scaling="parts", factor=8.0, original_len=4096)
    f, _ = packed.rotary_frequencies(64)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and abs(s - (0.1 * math.log(8) + 1)) < 1e-15
    assert torch.allclose(p[turns <= 1], f[turns <= 1] / 8, rtol=1e-14, atol=0)
    assert bool(((p <= f) & (p >= f / 8 * (1 - 1e-14))).all())


@pytest.mark.parametrize("change, error", [
    (dict(k_cache=torch.zeros(1, 8, 2, 16, dtype=torch.bfloat16)), TypeError),
    (dict(k_cache=torch.zeros(8, 2, 16)), ValueError),
    (dict(k_cache=torch.zeros(2, 8, 2, 16), v_cache=torch.zeros(2, 8, 2, 16)), ValueError),
    (dict(v_cache=torch.zeros(1, 9, 2, 16)), ValueError),
    (dict(lens=_offs(0, 0)), ValueError), (dict(lens=torch.zeros(1)), TypeError),
    (dict(k_cache=torch.zeros(1, 8, 2, 16, requires_grad=True)), ValueError),
    (dict(k_cache=torch.zeros(1, 8, 16, 2).transpose(2, 3)), ValueError),
])
def test_cache_operators_refuse(change, error):
    q, k, v = (t[None] for t in _qkv())
    args = dict(q=q, k=k, v=v, k_cache=torch.zeros(1, 8, 2, 16), v_cache=torch.zeros(1, 8, 2, 16), lens=_offs(0),
                inv_freq=torch.ones(8, dtype=torch.float64))
    args.update(change)
    with pytest.raises(error):
        packed.rotary_append(**args)
    for name in ("k", "v", "inv_freq"):
        args.pop(name)
    with pytest.raises(error):
        packed.cached_attention(**args)


def test_append_refuses_shared_cache_rows():
    q, k, v = (t[None].expand(2, -1, -1, -1) for t in _qkv())
    shared = torch.zeros(1, 8, 2, 16).expand(2, -1, -1, -1)
    with pytest.raises(ValueError, match="shared"):
        packed.rotary_append(q, k, v, shared, shared, _offs(0, 0), torch.ones(8, dtype=torch.float64))


# ----------------------------------------------------------------------------- C entries: refused before any launch
A = 0x10000   # a pointer that is never followed


def _fwd(L, dtype=0, n_seq=1, nq=4, nk=4, heads=4, kv=2, d=16, q=A, tok=64, head=16, offs=A, scale=0.25, ws=None, size=0):
    return L.tagan_packed_attn_fwd(dtype, n_seq, nq, nk, heads, kv, d, q, tok, head, A, 32, 16, A, 32, 16, offs, offs,
                                   1, scale, A, 64, 16, None, None, ws, size, None)


@pytest.mark.parametrize("kw, status", [
    (dict(dtype=2), -2), (dict(d=12), -2), (dict(d=136), -2), (dict(heads=5), -1), (dict(kv=0), -1),
    (dict(heads=1026, kv=2), -1), (dict(scale=0.0), -1), (dict(nq=-1), -1), (dict(nk=1 << 31), -1), (dict(n_seq=-1), -1),
    (dict(q=None), -1), (dict(q=A + 4), -1), (dict(tok=66), -1), (dict(tok=8), -1), (dict(tok=1 << 23), -1),
    (dict(offs=None), -1), (dict(nq=0, q=None), 0), (dict(nk=4000), -4), (dict(nk=4000, ws=A + 8, size=1 << 30), -4),
])
def test_packed_fwd_entry(kw, status):
    assert _fwd(_lib.lib(), **kw) == status


def _bwd(L, ws=A, size=None, lse=A, head=16, heads=4):
    size = L.tagan_packed_attn_bwd_workspace(4, heads) if size is None else size
    return L.tagan_packed_attn_bwd(0, 1, 4, 4, heads, 2, 16, A, 64, head, A, 32, 16, A, 32, 16, A, A, 1, 0.25, A, 64,
                                   16, lse, None, A, 64, 16, A, 64, 16, A, 32, 16, A, 32, 16, ws, size, None)


@pytest.mark.parametrize("kw, status", [(dict(size=4 * 4 * 8 - 1), -4), (dict(ws=None), -4), (dict(lse=None), -4),
                                        (dict(head=1 << 28), -2), (dict(heads=3), -1)])
def test_packed_bwd_entry(kw, status):
    assert _bwd(_lib.lib(), **kw) == status


def test_cached_entry():
    L = _lib.lib()
    need = L.tagan_cached_attn_workspace(2, 1, 4096, 8, 2, 64)
    assert need > 0 and L.tagan_cached_attn_workspace(0, 1, 4096, 8, 2, 64) == 0

    def call(ws=A, size=need, lens=A, cap=4096, batch=2):
        return L.tagan_cached_attn(0, batch, 1, cap, 8, 2, 64, A, 512, 512, 64, A, 1 << 20, 128, 64, A, 1 << 20, 128,
                                   64, lens, 0.125, A, 512, 512, 64, ws, size, None)
    assert call(size=need - 1) == -4 and call(ws=None) == -4 and call(lens=None) == -1 and call(cap=-1) == -1
    assert call(batch=0) == 0


def test_rotary_entry():
    L = _lib.lib()

    def call(dtype=0, n=4, heads=4, kv=2, d=16, rot=16, pos=A, kind=0, scale=1.0, q=A):
        return L.tagan_rotary(dtype, n, heads, kv, d, rot, q, 64, 16, A, 32, 16, pos, kind, A, scale, 0, 0, A, 64, 16,
                              A, 32, 16, None)
    for kw, status in [(dict(dtype=3), -2), (dict(rot=3), -1), (dict(rot=18), -1), (dict(rot=0), -1), (dict(d=258), -2),
                       (dict(heads=0, kv=0), -1), (dict(pos=None), -1), (dict(kind=4), -2), (dict(q=None), -1),
                       (dict(scale=math.inf), -1), (dict(n=-1), -1), (dict(n=0), 0)]:
        assert call(**kw) == status, kw
