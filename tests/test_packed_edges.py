"""Edges of the packed operators: bounds that a wrong result cannot pass, caches past their capacity, infinities, limits.

Inputs are made on the CPU, so that the checks of the bounds themselves run without a device: a bound has to refuse a
planted mistake (in the 64-bit reference).  Bounds, with W = 2^-24 and u half a step of the storage type:
  scores   |ds| <= (d + 4) W scale |q||k|; the exponent's argument (at most 8 powers of two above the maximum's) and
           exp2 add (|s - m| + 16) W: a relative error e of each unnormalised weight, 2 e of each normalised one
  out      the sum over S keys adds (S + 8) W, the join of at most 512 splits 2 (512 + 8) W (its weights and its sum):
           |do| <= (u' + 2 e + (S + 8 + 2 * 520) W) P|V| + u |o|, u' = u for bf16 (each probability is rounded), else 0
"""
import math
import os
import subprocess
import sys

import pytest
import torch

from tagan_amd import _lib, packed

DEV = "cuda"
W = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]
I32 = torch.int32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def _rows(q, k, v, see, scale, dtype):
    """softmax(scale q kᵀ) v of the keys that `see` [R, S] shows, in 64 bits: out [R, d], its bound and the weights."""
    q, k, v = q.double(), k.double(), v.double()
    u, u1, d, S = UNIT[dtype], UNIT[dtype] if dtype == torch.bfloat16 else 0.0, q.shape[1], k.shape[0]
    s = ((q @ k.T) * scale).masked_fill(~see, -math.inf)
    m = s.amax(1, keepdim=True) if S else torch.zeros(q.shape[0], 1, dtype=torch.float64)
    m = torch.where(torch.isfinite(m), m, 0.0)
    P = torch.exp(s - m)
    total = P.sum(1, keepdim=True)
    P = P / torch.where(total > 0, total, 1.0)
    sab = (q.abs() @ k.abs().T) * scale
    e = ((d + 4) * W * sab + ((s - m).abs() + 16) * W).masked_fill(~see, 0.0)
    e = e.amax(1, keepdim=True) if S else torch.zeros_like(m)
    o = P @ v
    return o, (u1 + 2 * e + (S + 8 + 2 * 520) * W) * (P @ v.abs()) * (1 + u) + u * o.abs(), P


def _cached_want(q, kc, vc, lens, scale=None):
    """cached_attention and its bound on the CPU: query i sees rows j < lens - L + 1 + i of the cache."""
    B, L, hq, d = q.shape
    cap, hk = kc.shape[1:3]
    G, scale = hq // hk, d ** -0.5 if scale is None else scale
    out, tol = torch.zeros(B, L, hq, d, dtype=torch.float64), torch.zeros(B, L, hq, d, dtype=torch.float64)
    for b, n in enumerate(lens):
        S = max(0, min(n, cap))
        end = torch.tensor([n - L + 1 + i for i in range(L) for _ in range(G)])
        see = torch.arange(S)[None] < end[:, None]
        for h in range(hk):
            sl = slice(h * G, (h + 1) * G)
            o, t, _ = _rows(q[b, :, sl].reshape(L * G, d), kc[b, :S, h], vc[b, :S, h], see, scale, q.dtype)
            out[b, :, sl], tol[b, :, sl] = o.view(L, G, d), t.view(L, G, d)
    return out, tol


def _within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    over = (got - want).abs() - tol
    assert not bool((over > 0).any()), "%s: %d of %d beyond their bound, worst by %.3g" % (
        what, int((over > 0).sum()), over.numel(), float(over.max()))


def _dev(*tensors):
    return [t.to(DEV) for t in tensors]


# ----------------------------------------------------------------------------- a cache whose lengths pass its capacity
PAST = [(50, 5, [52, 50, 54, 55, 56, 2 ** 31 - 1, 45, 3, -2 ** 31], 8, 2, 64), (3000, 3, [3002, 3001, 3000, 3500], 4, 1, 128),
        (20, 40, [25, 59, 60, 7], 4, 2, 16), (0, 2, [0, 2, 9], 2, 1, 32)]


def _past(cap, L, lens, hq, hk, d, dtype):
    gen = _gen(21)
    q = _randn(gen, len(lens), L, hq, d, dtype=dtype)
    return q, *(_randn(gen, len(lens), cap, hk, d, dtype=dtype) for _ in range(2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap, L, lens, hq, hk, d", PAST)
def test_lengths_past_the_capacity_keep_the_window(dtype, cap, L, lens, hq, hk, d):
    """The rows that did not fit are missing, but each query still sees what lies before it."""
    q, kc, vc = _past(cap, L, lens, hq, hk, d, dtype)
    got = packed.cached_attention(*_dev(q, kc, vc, torch.tensor(lens, dtype=I32)))
    _within(got, *_cached_want(q, kc, vc, lens), "capacity %d, new %d" % (cap, L))


@pytest.mark.gpu
def test_append_past_the_capacity_then_attend():
    """Three of five new tokens fit: each of them sees its own key, and so do those that follow."""
    gen, cap, L, hq, hk, d = _gen(22), 50, 5, 4, 2, 32
    q, k, v = (_randn(gen, 1, L, h, d) for h in (hq, hk, hk))
    kc, vc = _dev(_randn(gen, 1, cap, hk, d), _randn(gen, 1, cap, hk, d))
    freq, _ = packed.rotary_frequencies(d, device=DEV)
    lens = torch.tensor([47], dtype=I32, device=DEV)
    qn = packed.rotary_append(*_dev(q, k, v), kc, vc, lens, freq)
    lens += L
    got = packed.cached_attention(qn, kc, vc, lens)
    assert torch.equal(vc[0, 47:].cpu(), v[0, :3])
    _within(got, *_cached_want(qn.cpu(), kc.cpu(), vc.cpu(), [52]), "after the last row")


# ----------------------------------------------------------------------------- infinities that a row sees
def _hidden_weight(n, hk, d, at, bad, gen):
    """Keys 0 to 511 weigh nothing in fp32 (their scores lie 120 below the others'); one of their values is `bad`."""
    k, v = _randn(gen, n, hk, d), _randn(gen, n, hk, d)
    k[:, :, 0] = 0
    k[:512, :, 0] = -120 * d ** 0.5
    v[at, :, 3] = bad
    return k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d", [16, 128])
def test_what_a_row_sees_reaches_it_whatever_its_weight(dtype, bad, d):
    """In one pass over the keys and in splits of them, packed and cached: no finite result hides such a value."""
    gen, n, at = _gen(23), 6000, 70
    k, v = (t.to(dtype) for t in _hidden_weight(n, 1, d, at, bad, gen))
    q = torch.zeros(n, 2, d, dtype=dtype)
    q[:, :, 0] = 1
    k, v, q = _dev(k, v, q)
    offs = [torch.tensor([0, m], dtype=I32, device=DEV) for m in (1, 3, n)]

    def seen(out, rows):
        assert not bool(torch.isfinite(out[rows, :, 3]).any())
        assert bool(torch.isfinite(out[rows][..., [0, 1, 2, *range(4, d)]]).all())
    assert packed.lib().tagan_packed_attn_fwd_workspace(1, 1, n, 2, 1, d) > 0
    seen(packed.attention(q[:1], k, v, offs[0], offs[2]), slice(0, 1))
    seen(packed.attention(q[:3], k, v, offs[1], offs[2], causal=False), slice(0, 3))
    out = packed.attention(q[:900], k[:900], v[:900], torch.tensor([0, 900], dtype=I32, device=DEV))
    assert bool(torch.isfinite(out[:at]).all())
    seen(out, slice(at, 900))
    one = packed.cached_attention(q[None, :2], k[None], v[None], torch.tensor([n], dtype=I32, device=DEV))
    seen(one[0], slice(0, 2))


# ----------------------------------------------------------------------------- C entries: refused before any launch
A = 0x10000   # a pointer that is never followed


def test_cached_entry_leaves_room_behind_the_last_key():
    """A tile's end is counted in 31 bits: the capacity stays a tile and more below 2^31, as packed keys do."""
    L = _lib.lib()
    for cap, status in ((0x7fffffff, -1), (0x7fffffff - 1023, -1), (-1, -1)):
        got = L.tagan_cached_attn(0, 1, 1, cap, 2, 1, 8, A, 16, 16, 8, A, 0, 8, 8, A, 0, 8, 8, A, 0.25, A, 16, 16, 8, A,
                                  1 << 40, None)
        assert got == status, cap


@pytest.mark.parametrize("nq, heads", [(1 << 31, 1 << 30), (1 << 62, 1 << 30), (1 << 30, 1 << 30), (1 << 40, 8)])
def test_forward_workspace_of_impossible_sizes(nq, heads):
    """Sizes that no call takes need no workspace; their products do not overflow into a division by zero."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.path.insert(0, '.')\nfrom tagan_amd import _lib\n"
            "print(_lib.lib().tagan_packed_attn_fwd_workspace(1, %d, (1 << 31) - 4096, %d, %d, 16))" % (nq, heads, heads))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=root)
    assert r.returncode == 0 and r.stdout.strip() == "0", (r.returncode, r.stderr[-300:])


def test_entries_refuse_impossible_sizes():
    L, n = _lib.lib(), 1 << 30
    assert L.tagan_packed_attn_fwd(0, 1, n, n, n, n, 16, A, 16, 0, A, 16, 0, A, 16, 0, A, A, 1, 0.25, A, 16, 0, None, None,
                                   A, 1 << 60, None) == -2
    assert L.tagan_packed_attn_bwd(0, 1, n, n, n, n, 16, A, 16, 0, A, 16, 0, A, 16, 0, A, A, 1, 0.25, A, 16, 0, A, None, A,
                                   16, 0, A, 16, 0, A, 16, 0, A, 16, 0, A, 1 << 60, None) == -2
    assert L.tagan_cached_attn(0, n, 1 << 12, 64, n, n, 16, A, 0, 16, 0, A, 0, 16, 0, A, 0, 16, 0, A, 0.25, A, 0, 16, 0, A,
                               1 << 60, None) == -2
    assert L.tagan_cached_attn_workspace(n, 1 << 12, 64, n, n, 16) == 0


@pytest.mark.parametrize("heads, kv", [((1 << 28) + 1, 1), (1, (1 << 28) + 1), (0x7fffffff, 0)])
def test_rotary_entries_count_heads_in_31_bits(heads, kv):
    """A block counts the heads of four tokens, and the steps behind the last, in 31 bits."""
    L = _lib.lib()
    assert L.tagan_rotary(0, 1, heads, kv, 2, 2, A, 2, 2, A, 2, 2, A, 0, A, 1.0, 0, 0, A, 2, 2, A, 2, 2, None) == -2
    if kv:
        assert L.tagan_rotary_append(0, 1, 1, heads, kv, 2, 2, A, 2, 2, 2, A, 2, 2, 2, A, 2, 2, 2, A, A, 1.0, 0, A, 2, 2,
                                     2, A, 2, 2, 2, A, 2, 2, 2, 8, None) == -2


# ----------------------------------------------------------------------------- caches and autograd
@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_append_to_a_cache_that_a_backward_still_reads(which):
    """The rows that attention kept for its backward were overwritten: it has to say so, not to use them."""
    gen, cap, hq, hk, d = _gen(24), 8, 4, 2, 16
    q = _randn(gen, 4, hq, d).to(DEV).requires_grad_(True)
    caches = _dev(_randn(gen, 1, cap, hk, d), _randn(gen, 1, cap, hk, d))
    kept = [c[0, :4] if i == which else c[0, :4].clone() for i, c in enumerate(caches)]
    freq, _ = packed.rotary_frequencies(d, device=DEV)
    out = packed.attention(q, *kept, torch.tensor([0, 4], dtype=I32, device=DEV))
    new = _dev(*(_randn(gen, 1, 2, h, d) for h in (hq, hk, hk)))
    packed.rotary_append(*new, *caches, torch.tensor([1], dtype=I32, device=DEV), freq)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_append_refuses_one_tensor_as_both_caches():
    q, k, v = (torch.zeros(2, 1, h, 16) for h in (4, 2, 2))
    c, both = torch.zeros(2, 8, 2, 16), torch.zeros(2, 8, 2, 2, 16)
    freq, lens = torch.ones(8, dtype=torch.float64), torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match="one tensor"):
        packed.rotary_append(q, k, v, c, c, lens, freq)
    for pair in ((c, c.clone()), both.unbind(2)):          # accepted up to the device
        with pytest.raises(RuntimeError, match="HIP device"):
            packed.rotary_append(q, k, v, *pair, lens, freq)


# ----------------------------------------------------------------------------- cached attention within a narrow bound
CACHED = [(6, L, 333, [0, 1, 2, 64, 332, 333], *h) for L in (1, 3)
          for h in ((1, 1, 8), (8, 2, 64), (8, 1, 128), (12, 4, 96))]
CACHED += [(2, 1, 9000, [9000, 4001], 8, 2, 128), (1, 40, 700, [690], 8, 2, 64), (3, 5, 30, [2, 5, 30], 64, 1, 16),
           (60, 1, 70, [(7 * i) % 71 for i in range(60)], 2, 1, 16)]


def _cache_inputs(B, L, cap, hq, hk, d, sharp=1.0, dtype=torch.float32):
    gen = _gen(25)
    return (_randn(gen, B, L, hq, d) * sharp).to(dtype), *(_randn(gen, B, cap, hk, d, dtype=dtype) for _ in range(2))


@pytest.mark.gpu
@pytest.mark.parametrize("B, L, cap, lens, hq, hk, d", CACHED)
def test_cached_attention_in_32_bits(B, L, cap, lens, hq, hk, d):
    q, kc, vc = _cache_inputs(B, L, cap, hq, hk, d)
    got = packed.cached_attention(*_dev(q, kc, vc, torch.tensor(lens, dtype=I32)))
    _within(got, *_cached_want(q, kc, vc, lens), "%d x %d on %s" % (B, L, lens[:6]))


@pytest.mark.parametrize("B, L, cap, lens, hq, hk, d", CACHED)
def test_the_bound_refuses_zeros_and_a_missing_key(B, L, cap, lens, hq, hk, d):
    """For every history with a key (two, where one is left out): zeros, the newest key left out, a tenth of them."""
    q, kc, vc = _cache_inputs(B, L, cap, hq, hk, d)
    want, tol = _cached_want(q, kc, vc, lens)

    def caught(got, least):
        bad = ((got - want).abs() > tol).flatten(1).any(1)
        assert all(bool(bad[b]) for b, n in enumerate(lens) if n >= least)
    caught(torch.zeros_like(want), 1)
    caught(_cached_want(q, kc, vc, [n - 1 for n in lens])[0], max(2, L))
    late = [max(0, n - n // 10) for n in lens]
    caught(_cached_want(q, kc, vc, late)[0], max(20, L))


def _boundary_values(n, hk, d):
    """Values at the ends of every run of 64 keys and at the last key only, all positive: each is a part of every sum."""
    gen = _gen(26)
    v = torch.zeros(n, hk, d)
    at = sorted({j for m in range(0, n, 64) for j in (m - 1, m) if j >= 0} | {n - 1})
    v[at] = _randn(gen, len(at), hk, d).abs() + 0.5
    return v, at


@pytest.mark.parametrize("n, hq, hk, d", [(9000, 8, 2, 128), (4001, 4, 1, 64)])
def test_the_bound_refuses_any_key_at_a_boundary(n, hq, hk, d):
    q, kc, _ = _cache_inputs(1, 1, n, hq, hk, d, 0.1)
    v, at = _boundary_values(n, hk, d)
    G = hq // hk
    for h in range(hk):
        o, tol, P = _rows(q[0, 0, h * G:(h + 1) * G], kc[0, :, h], v[:, h], torch.ones(G, n, dtype=torch.bool), d ** -0.5,
                          torch.float32)
        gone = P[:, at, None] * v[at, h].double()[None]         # what the result lacks without that key: [G, at, d]
        assert bool((gone > tol[:, None]).any(2).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n, hq, hk, d", [(9000, 8, 2, 128), (4001, 4, 1, 64)])
def test_keys_at_every_boundary_of_a_split_count(n, hq, hk, d):
    q, kc, _ = _cache_inputs(1, 1, n, hq, hk, d, 0.1)
    v, _ = _boundary_values(n, hk, d)
    want, tol = _cached_want(q, kc, v[None], [n])
    got = packed.cached_attention(*_dev(q, kc, v[None], torch.tensor([n], dtype=I32)))
    _within(got, want, tol, "cached")
    offs = _dev(torch.tensor([0, 1], dtype=I32), torch.tensor([0, n], dtype=I32))
    got = packed.attention(*_dev(q[0], kc[0], v), *offs)
    _within(got, want[0], tol[0], "packed")


@pytest.mark.gpu
@pytest.mark.parametrize("step", [1, 5])
def test_serving_in_32_bits(step):
    """Every step of three histories against the caches as they then are."""
    gen, hq, hk, d, cap = _gen(27), 4, 2, 32, 64
    kc, vc = (torch.full((3, cap, hk, d), math.nan, device=DEV) for _ in range(2))
    lens = torch.tensor([0, 7, 19], dtype=I32, device=DEV)
    for c in (kc, vc):
        for b, n in enumerate(lens.tolist()):
            c[b, :n] = _randn(gen, n, hk, d).to(DEV)
    freq, _ = packed.rotary_frequencies(16, device=DEV)
    for _ in range(40 // step):
        qn = packed.rotary_append(*_dev(*(_randn(gen, 3, step, h, d) for h in (hq, hk, hk))), kc, vc, lens, freq)
        lens += step
        got = packed.cached_attention(qn, kc, vc, lens)
        _within(got, *_cached_want(qn.cpu(), kc.cpu(), vc.cpu(), lens.tolist()), "lengths %s" % lens.tolist())


# ----------------------------------------------------------------------------- bf16: what the output's rounding took away
# All scores are equal (q or k is zero), so the forward's probabilities are ones before the division and lose nothing as
# bf16 operands.  Values are multiples of 1/2 near 64: a sum of 5000 stays below 2^23 halves and is exact in fp32, in any
# order and in splits (their weights are ones too).  So out and its rest together are within 2^-16 (two roundings) and 8 W
# (the division) of the mean.  With their large common part dP - rowsum(dO O) is a small difference of large terms, and
# the output's own rounding (2^-8) would drown it; q, k and dO have a common part, so that
# no sum over keys or rows averages it away.
REST = [([3, 2, 4], [3, 2, 4], True), ([65], [65], True), ([90, 2], [90, 2], False), ([2, 1], [4000, 900], True),
        ([150], [5000], False)]


def _equal_scores(lens, klens, zero, hk=2, G=2, d=64):
    gen = _gen(28)
    n, nk = sum(lens), sum(klens)
    q, k, do = (_randn(gen, m, h, d, dtype=torch.bfloat16) for m, h in ((n, hk * G), (nk, hk), (n, hk * G)))
    v = ((_randn(gen, nk, hk, d) * 2).round() / 2 + 64).to(torch.bfloat16)
    q, k, do = q + 1, k + 1, do + 1
    (q if zero == "q" else k).zero_()
    offs = [torch.tensor([0, *torch.tensor(x).cumsum(0).tolist()], dtype=I32) for x in (lens, klens)]
    return q, k, v, do, *offs


def _equal_want(q, k, v, do, offs, koffs, causal, lost=0.0):
    """out, dq, dk and their bounds in 64 bits; `lost` 1 takes rowsum(dO O) from the rounded output (a planted mistake)."""
    n, hq, d = q.shape
    nk, hk = k.shape[:2]
    G, scale, u = hq // hk, d ** -0.5, UNIT[torch.bfloat16]
    o, to = (torch.zeros(n, hq, d, dtype=torch.float64) for _ in range(2))
    dq, tq = torch.zeros_like(o), torch.zeros_like(o)
    dk, tk = (torch.zeros(nk, hk, d, dtype=torch.float64) for _ in range(2))
    Q, K, V, D = (t.double() for t in (q, k, v, do))
    for a, b, ka, kb in zip(offs.tolist(), offs.tolist()[1:], koffs.tolist(), koffs.tolist()[1:]):
        lq, lk = b - a, kb - ka
        see = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            see = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + lk - lq
        P = see.double() / see.sum(1, keepdim=True)
        for h in range(hq):
            x, y, z, g = Q[a:b, h], K[ka:kb, h // G], V[ka:kb, h // G], D[a:b, h]
            oh = P @ z
            toh = (2.0 ** -16 + 8 * W) * (P @ z.abs())
            o[a:b, h], to[a:b, h] = oh, toh
            dP = g @ z.T
            kept = oh + lost * (oh.to(torch.bfloat16).double() - oh)
            delta = (g * kept).sum(1, keepdim=True)
            dS = P * (dP - delta)
            dd = (g.abs() * toh).sum(1, keepdim=True) + (d + 4) * W * (g.abs() * oh.abs()).sum(1, keepdim=True)
            # P again from the log-sum-exp: log2 of the count and exp2, a few W of up to 13
            tS = P * ((d + 4) * W * (g.abs() @ z.abs().T) + dd + 4 * W * (dP.abs() + delta.abs())) + 32 * W * dS.abs()
            tS = tS * (1 + u) + u * dS.abs()
            dq[a:b, h] = dS @ y * scale
            tq[a:b, h] = (tS @ y.abs() + (lk + 8) * W * (dS.abs() @ y.abs())) * scale * (1 + u) + u * dq[a:b, h].abs()
            dk[ka:kb, h // G] += dS.T @ x * scale
            tk[ka:kb, h // G] += (tS.T @ x.abs() + (lq * G + 8) * W * (dS.abs().T @ x.abs())) * scale * (1 + u)
    return o, to, dq, tq, dk, tk + u * dk.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("lens, klens, causal", REST)
@pytest.mark.parametrize("zero", ["q", "k"])
def test_the_rest_of_the_rounding_is_kept_and_used(lens, klens, causal, zero):
    split = sum(klens) > 4000
    assert (packed.lib().tagan_packed_attn_fwd_workspace(len(lens), sum(lens), sum(klens), 4, 2, 64) > 0) == split
    q, k, v, do, offs, koffs = _equal_scores(lens, klens, zero)
    leaves = [t.requires_grad_(True) for t in _dev(q, k, v)]
    out = packed.attention(*leaves, *_dev(offs, koffs), causal=causal)
    o, to, dq, tq, dk, tk = _equal_want(q, k, v, do, offs, koffs, causal)
    assert torch.equal(out.grad_fn.saved_tensors[3], out)
    rest = out.grad_fn.saved_tensors[5]
    _within(out.detach().double() + rest.double(), o, to, "out and its rest")
    grads = torch.autograd.grad(out, leaves, do.to(DEV))
    _within(grads[0], dq, tq, "dq")
    _within(grads[1], dk, tk, "dk")


@pytest.mark.parametrize("lens, klens, causal", REST)
def test_the_bound_refuses_a_rest_of_zeros(lens, klens, causal):
    for zero, which in (("q", 2), ("k", 4)):
        args = _equal_scores(lens, klens, zero)
        want, lost = _equal_want(*args, causal), _equal_want(*args, causal, lost=1.0)
        assert bool(((lost[which] - want[which]).abs() > want[which + 1]).any()), zero
        assert bool(((want[0].to(torch.bfloat16).double() - want[0]).abs() > want[1]).any())


@pytest.mark.parametrize("scale", [3e38, 1e39, 2.0 ** 127 * 1.0001, 1e-39, 1e-46])
def test_scales_beyond_the_range_of_fp32_are_refused(scale):
    q, k, offs = torch.zeros(6, 4, 16), torch.zeros(6, 2, 16), torch.tensor([0, 6], dtype=I32)
    with pytest.raises(ValueError, match="scale"):
        packed.attention(q, k, k, offs, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        packed.cached_attention(q[:, None], k[:, None], k[:, None], torch.ones(6, dtype=I32), scale=scale)
    assert _lib.lib().tagan_packed_attn_fwd(0, 1, 6, 6, 4, 2, 16, A, 64, 16, A, 32, 16, A, 32, 16, A, A, 1, scale, A, 64, 16,
                                            None, None, None, 0, None) == -1


# ----------------------------------------------------------------------------- bf16: short histories
# Up to 64 keys to an average history each probability and each dS enters as two bf16 operands (2^-16): out and its rest are
# within (2^-16 + 2 e + (S + 8) W) P|V| + 2^-16 |o|, rowsum(dO O) is as exact, and the gradients have their own rounding (u)
# and those terms only.  Values with a large common part show the forward's share: the probabilities' bf16 rounding alone
# (2^-8 each) would move the mean, and with it every dP - rowsum(dO O) of the row; values without one show the backward's.
FINE = [([1, 2, 3, 4] * 8, None, 2, 2, 16, True), ([5, 20, 40, 64], None, 2, 1, 64, True), ([16, 9, 30], None, 16, 2, 32, True),
        ([50, 50], None, 2, 2, 128, False), ([3, 1, 0], [40, 9, 90], 4, 2, 96, True)]


def _short(lens, klens, hq, hk, d, common):
    gen, klens = _gen(29), klens or lens
    assert sum(klens) <= 64 * len(klens)
    q, k, do = (_randn(gen, sum(x), h, d, dtype=torch.bfloat16) for x, h in ((lens, hq), (klens, hk), (lens, hq)))
    v = (_randn(gen, sum(klens), hk, d) + common).to(torch.bfloat16)
    if common:                                           # so that no sum averages a row's error away
        q, k, do = q / 2 + 0.5, k / 2 + 0.5, do + 1
    return q, k, v, do, *(torch.tensor([0, *torch.tensor(x).cumsum(0).tolist()], dtype=I32) for x in (lens, klens))


def _short_want(q, k, v, do, offs, koffs, causal, planted=None):
    """out, dq, dk, dv and their bounds in 64 bits.  Planted: one bf16 operand for the forward's or the backward's."""
    n, hq, d = q.shape
    nk, hk = k.shape[:2]
    G, scale, u, u2 = hq // hk, d ** -0.5, UNIT[torch.bfloat16], 2.0 ** -16
    res = [torch.zeros(m, h, d, dtype=torch.float64) for m, h in ((n, hq),) * 4 + ((nk, hk),) * 4]
    o, to, dq, tq, dk, tk, dv, tv = res
    Q, K, V, D = (t.double() for t in (q, k, v, do))
    for a, b, ka, kb in zip(offs.tolist(), offs.tolist()[1:], koffs.tolist(), koffs.tolist()[1:]):
        lq, S = b - a, kb - ka
        if lq == 0:
            continue
        see = torch.ones(lq, S, dtype=torch.bool)
        if causal:
            see = torch.arange(S)[None] <= torch.arange(lq)[:, None] + S - lq
        for h in range(hq):
            x, y, z, g = Q[a:b, h], K[ka:kb, h // G], V[ka:kb, h // G], D[a:b, h]
            s = ((x @ y.T) * scale).masked_fill(~see, -math.inf)
            w = torch.exp(s - s.amax(1, keepdim=True))
            total = w.sum(1, keepdim=True)
            P = w / total
            e = ((d + 4) * W * (x.abs() @ y.abs().T) * scale + ((s - s.amax(1, keepdim=True)).abs() + 16) * W)
            e = e.masked_fill(~see, 0.0).amax(1, keepdim=True)
            oh = ((w.to(torch.bfloat16).double() if planted == "forward" else w) @ z) / total
            toh = (u2 + 2 * e + (S + 8) * W) * (P @ z.abs()) + u2 * oh.abs()
            o[a:b, h], to[a:b, h] = oh, toh
            dP, delta = g @ z.T, (g * oh).sum(1, keepdim=True)
            dS = P * (dP - delta)
            dd = (g.abs() * toh).sum(1, keepdim=True) + (d + 4) * W * (g.abs() * oh.abs()).sum(1, keepdim=True)
            tS = P * ((d + 4) * W * (g.abs() @ z.abs().T) + dd + 4 * W * (dP.abs() + delta.abs()))
            tS = (tS + (2 * e + 32 * W) * dS.abs()) * (1 + u2) + u2 * dS.abs()
            Pb = P
            if planted == "backward":
                dS, Pb = dS.to(torch.bfloat16).double(), P.to(torch.bfloat16).double()
            dv[ka:kb, h // G] += Pb.T @ g
            tv[ka:kb, h // G] += (u2 + 2 * e.amax() + 32 * W + (lq * G + 8) * W) * (P.T @ g.abs()) * (1 + u)
            dq[a:b, h] = dS @ y * scale
            tq[a:b, h] = (tS @ y.abs() + (S + 8) * W * (dS.abs() @ y.abs())) * scale * (1 + u) + u * dq[a:b, h].abs()
            dk[ka:kb, h // G] += dS.T @ x * scale
            tk[ka:kb, h // G] += (tS.T @ x.abs() + (lq * G + 8) * W * (dS.abs().T @ x.abs())) * scale * (1 + u)
    tk += u * dk.abs()
    tv += u * dv.abs()
    return res


def _over_one_rounding(got, want):
    """The error's norm over that of rounding the exact result once.  N elements' own roundings leave it within 5 / sqrt(N)
    of 1 (five deviations); independent roundings of the same size in every term of its sums bring it to sqrt(2)."""
    return float((got.detach().cpu().double() - want).norm() / (want.to(torch.bfloat16).double() - want).norm())


@pytest.mark.gpu
@pytest.mark.parametrize("common", [0, 64])
@pytest.mark.parametrize("lens, klens, hq, hk, d, causal", FINE)
def test_short_histories_lose_nothing_to_the_operands(lens, klens, hq, hk, d, causal, common):
    q, k, v, do, offs, koffs = _short(lens, klens, hq, hk, d, common)
    leaves = [t.requires_grad_(True) for t in _dev(q, k, v)]
    out = packed.attention(*leaves, *_dev(offs, koffs), causal=causal)
    o, to, dq, tq, dk, tk, dv, tv = _short_want(q, k, v, do, offs, koffs, causal)
    _within(out.detach().double() + out.grad_fn.saved_tensors[5].double(), o, to, "out and its rest")
    grads = torch.autograd.grad(out, leaves, do.to(DEV))
    _within(grads[0], dq, tq, "dq")
    _within(grads[1], dk, tk, "dk")
    _within(grads[2], dv, tv, "dv")
    if common == 0:
        assert q.numel() > 625 and k.numel() > 2500
        assert _over_one_rounding(grads[0], dq) < 1.2 and _over_one_rounding(grads[1], dk) < 1.2
        assert _over_one_rounding(grads[2], dv) < 1.1
    assert torch.equal(packed.attention(*(t.detach() for t in leaves), *_dev(offs, koffs), causal=causal), out)


@pytest.mark.parametrize("lens, klens, hq, hk, d, causal", FINE)
def test_the_bound_refuses_rounded_operands(lens, klens, hq, hk, d, causal):
    args = _short(lens, klens, hq, hk, d, 64)
    want, got = _short_want(*args, causal), _short_want(*args, causal, planted="forward")
    for which in (0, 2, 4):
        assert bool(((got[which] - want[which]).abs() > want[which + 1]).any()), which
    args = _short(lens, klens, hq, hk, d, 0)
    want, got = _short_want(*args, causal), _short_want(*args, causal, planted="backward")
    for which, least in ((2, 1.2), (4, 1.2), (6, 1.1)):
        assert _over_one_rounding(got[which].to(torch.bfloat16), want[which]) > least, which


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_short_histories_keep_infinities(causal):
    """A visible infinity is that infinity, not NaN, though the second operand's weights are zeros and negative ones too."""
    gen, n = _gen(30), 50
    q, k, v = (_randn(gen, n, h, 16, dtype=torch.bfloat16) for h in (4, 2, 2))
    v[7, :, 3], v[9, :, 5] = math.inf, -math.inf
    out = packed.attention(*_dev(q, k, v, torch.tensor([0, 20, 50], dtype=I32)), causal=causal).cpu()
    rows = slice(9, 20) if causal else slice(0, 20)
    assert bool((out[rows, :, 3] == math.inf).all()) and bool((out[rows, :, 5] == -math.inf).all())
    assert bool(torch.isfinite(out[20:]).all()) and bool(torch.isfinite(out[rows][..., [0, 1, 2, 4, *range(6, 16)]]).all())
    assert not causal or bool(torch.isfinite(out[:7]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[700] + [1] * 20, [1] * 10 + [128, 129, 3], [127, 2, 0, 0, 0, 400] + [5] * 10], ids=str)
@pytest.mark.parametrize("hq, hk, d", [(2, 2, 16), (4, 1, 128)])
def test_a_long_history_among_short_ones(lens, hq, hk, d):
    """The batch's average is short; each history goes by its own keys."""
    from test_gpu_packed import _attend
    assert sum(lens) <= 64 * len(lens)
    _attend(lens, lens, hq, hk, d, torch.bfloat16)
    _attend(lens, lens, hq, hk, d, torch.bfloat16, causal=False)


# ----------------------------------------------------------------------------- infinities and gradients
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, d", [([40, 30, 9], 16), ([300, 200, 77], 128), ([20, 5, 900], 64)])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_gradients_of_other_histories_keep_their_bits(dtype, lens, d, which):
    """NaN and infinities in one history reach gradients of that history only."""
    gen, n = _gen(31), sum(lens)
    t = {x: _randn(gen, n, h, d, dtype=dtype) for x, h in (("q", 4), ("k", 2), ("v", 2), ("dout", 4))}
    offs = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=I32).to(DEV)

    def grads():
        leaves = [x.to(DEV).requires_grad_(True) for x in (t["q"], t["k"], t["v"])]
        return torch.autograd.grad(packed.attention(*leaves, offs), leaves, t["dout"].to(DEV))
    want = grads()
    at = lens[0] + 3
    t[which][at, :, 2], t[which][at + 1, :, 5] = math.nan, math.inf
    others = [*range(lens[0]), *range(lens[0] + lens[1], n)]
    for got, w in zip(grads(), want):
        assert torch.equal(got[others], w[others])
