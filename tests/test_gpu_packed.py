"""Packed attention, rotary positions and cached attention against plain 64-bit formulas.

Tolerances are worked out per element from the roundings that the operators make.  u is half a step of the storage
type (2^-8 for bf16, 2^-24 for fp32), w = 2^-24 that of the fp32 sums.
  scores   a product sum of d terms and its scale: |ds| <= (d + 4) w s |q||k|, and exp2's argument and result add
           (|s - m| + 4) w: together a relative error e of each unnormalised weight, 2 e of each probability
  out      each probability is rounded to storage (u), the sum of L terms adds L w, the result is rounded (u):
           |do| <= (u' + 2 e + (L + 8) w) P|V| + u |o|, with u' = u for bf16 and 0 for fp32
  dV       the same with Pᵀ|dO|; the group's rows are the terms
  dS       P (dP - D): e as above on |dS|, dP's sum (d + 4) w |dO||V|, D from the rounded output; then rounded (u')
  dQ, dK   that through |K|, |Q|, plus u of the result and (terms) w of the sum
"""
import math

import pytest
import torch

import tagan_amd  # noqa: F401
from tagan_amd import packed

pytestmark = pytest.mark.gpu
DEV = "cuda"
W = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F64 = torch.float64


def _offs(lens, first=0):
    got = [first]
    for n in lens:
        got.append(got[-1] + n)
    return torch.tensor(got, dtype=torch.int32, device=DEV)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _one(q, k, v, causal, scale, do=None, dtype=torch.float32):
    """One sequence and one key head in 64 bits: rows [R = L * G, d] with their tokens, and bounds of every result."""
    lq, G, d = q.shape
    lk = k.shape[0]
    u, u1 = UNIT[dtype], (UNIT[dtype] if dtype == torch.bfloat16 else 0.0)
    Q = q.reshape(lq * G, d)
    tok = torch.arange(lq, device=q.device).repeat_interleave(G)
    res = {"o": torch.zeros_like(Q), "to": torch.zeros_like(Q)}
    if lk == 0 or lq == 0:
        if do is not None:
            for n, like in (("dq", Q), ("dk", k), ("dv", k)):
                res[n], res["t" + n] = torch.zeros_like(like), torch.zeros_like(like)
        return res
    see = torch.ones(lq * G, lk, dtype=torch.bool, device=q.device)
    if causal:
        see = torch.arange(lk, device=q.device)[None] <= tok[:, None] + lk - lq
    s = (Q @ k.T) * scale
    sm = s.masked_fill(~see, -math.inf)
    m = sm.max(1, keepdim=True).values
    m = torch.where(torch.isfinite(m), m, 0.0)
    P = torch.exp(sm - m)
    tot = P.sum(1, keepdim=True)
    P = P / torch.where(tot > 0, tot, 1.0)
    o = P @ v
    sab = (Q.abs() @ k.abs().T) * scale
    e = ((d + 4) * W * sab + ((s - m).abs() + 4) * W).masked_fill(~see, 0.0).max(1, keepdim=True).values
    rel = u1 + 2 * e + (lk + 8) * W
    to = rel * (P @ v.abs())
    res["o"], res["to"] = o, to * (1 + u) + u * o.abs()
    if do is None:
        return res
    D = do.reshape(lq * G, d)
    dP = D @ v.T
    delta = (D * o).sum(1, keepdim=True)
    dS = P * (dP - delta)
    ddelta = (D.abs() * res["to"]).sum(1, keepdim=True) + d * W * (D.abs() * o.abs()).sum(1, keepdim=True)
    tS = P * ((d + 4) * W * (D.abs() @ v.abs().T) + ddelta + 4 * W * (dP.abs() + delta.abs())) + 2 * e * dS.abs()
    tS = tS * (1 + u1) + u1 * dS.abs()
    R = lq * G
    res["dq"] = dS @ k * scale
    res["tdq"] = (tS @ k.abs() + (lk + 8) * W * (dS.abs() @ k.abs())) * scale * (1 + u) + u * res["dq"].abs()
    res["dk"] = dS.T @ Q * scale
    res["tdk"] = (tS.T @ Q.abs() + (R + 8) * W * (dS.abs().T @ Q.abs())) * scale * (1 + u) + u * res["dk"].abs()
    res["dv"] = P.T @ D
    tP = P * (u1 + 2 * e)
    res["tdv"] = (tP.T @ D.abs() + (R + 8) * W * (P.T @ D.abs())) * (1 + u) + u * res["dv"].abs()
    return res


def _reference(q, k, v, offs, koffs, causal, scale, do=None):
    """(out, dq, dk, dv) and their bounds in 64 bits, zero outside the sequences."""
    n, hq, d = q.shape
    hk = k.shape[1]
    G = hq // hk
    dt = q.dtype
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    do = do.double() if do is not None else None
    names = [("o", q), ("dq", q), ("dk", k), ("dv", k)][:4 if do is not None else 1]
    out = {}
    for name, like in names:
        out[name], out["t" + name] = torch.zeros_like(like), torch.zeros_like(like)
    offs, koffs = offs.tolist(), koffs.tolist()
    for a, b, ka, kb in zip(offs, offs[1:], koffs, koffs[1:]):
        for h in range(hk):
            sl = slice(h * G, (h + 1) * G)
            r = _one(q[a:b, sl], k[ka:kb, h], v[ka:kb, h], causal, scale, None if do is None else do[a:b, sl], dt)
            for name in r:
                if name.endswith("o") or name.endswith("dq"):
                    out[name][a:b, sl] = r[name].reshape(b - a, G, d)
                else:
                    out[name][ka:kb, h] = r[name]
    return out


def _check(got, want, tol, what):
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got.float()).all()), what + " is not finite"
    over = (got.double() - want).abs() - tol
    bad = over > 0
    assert not bool(bad.any()), "%s: %d of %d beyond their bound, worst by %.3g (error %.3g)" % (
        what, int(bad.sum()), bad.numel(), float(over.max()), float((got.double() - want).abs().max()))


def _attend(lens, klens, hq, hk, d, dtype, causal=True, scale=None, seed=0, first=0, tail=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    offs, koffs = _offs(lens, first), _offs(klens, first)
    n, nk = int(offs[-1]) + tail, int(koffs[-1]) + tail
    q, k, v, do = (_randn(gen, m, h, d, dtype=dtype) for m, h in ((n, hq), (nk, hk), (nk, hk), (n, hq)))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = packed.attention(q, k, v, offs, koffs if klens is not lens else (None if n == nk else koffs),
                           causal=causal, scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), do)
    ref = _reference(q, k, v, offs, koffs, causal, d ** -0.5 if scale is None else scale, do)
    what = "lens %s/%s heads %d/%d d %d %s causal %d" % (lens[:6], klens[:6], hq, hk, d, dtype, causal)
    _check(out.detach(), ref["o"], ref["to"], "out, " + what)
    for name, g in zip(("dq", "dk", "dv"), grads):
        _check(g, ref[name], ref["t" + name], name + ", " + what)
    return q, k, v, out, grads


DTYPES = [torch.float32, torch.bfloat16]
LENS = [[1], [0, 1, 2, 0, 3], [31, 32, 33], [63, 64, 65, 127, 128, 129], [300, 0, 5]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("hq, hk, d", [(1, 1, 8), (8, 2, 64), (4, 4, 16), (7, 1, 32), (6, 2, 128)])
def test_lengths_and_heads(dtype, lens, hq, hk, d):
    _attend(lens, lens, hq, hk, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 24, 40, 72, 96, 104, 120])
def test_head_sizes_between_tiles(dtype, d):
    _attend([70, 9], [70, 9], 2, 1, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens, klens", [([5, 40, 1], [105, 300, 64]), ([100, 7], [30, 1]), ([3, 50], [0, 200]),
                                         ([0, 200], [17, 130]), ([1, 1, 1], [129, 1, 64])], ids=str)
def test_more_or_fewer_keys_than_queries(dtype, causal, lens, klens):
    """Fewer keys than queries leaves the first rows without a key; no keys leaves all of them."""
    _attend(lens, klens, 4, 2, 32, dtype, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_few_queries_on_many_keys(dtype, causal, d):
    """The key axis is split over workgroups and joined: one-wave and four-wave blocks, empty sequences, empty tails."""
    assert packed.lib().tagan_packed_attn_fwd_workspace(4, 12, 6301, 4, 2, d) > 0
    assert packed.lib().tagan_packed_attn_fwd_workspace(2, 150, 5000, 4, 2, d) > 0
    _attend([1, 8, 0, 3], [3000, 700, 600, 2001], 4, 2, d, dtype, causal, first=0, tail=0)
    _attend([130, 20], [4000, 1000], 4, 2, d, dtype, causal)
    _attend([5, 1], [1500, 0], 2, 2, d, dtype, causal, first=9, tail=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [([2, 0, 5, 1], [9000, 300, 4100, 1]), ([300], [2300]), ([1100, 1], [1100, 2500])])
def test_long_keys_for_few_blocks(dtype, lens):
    """Axes long enough to be split in both types: one-wave blocks, one history of many rows, uneven ones."""
    assert packed.lib().tagan_packed_attn_fwd_workspace(len(lens[0]), sum(lens[0]), sum(lens[1]), 2, 1, 64) > 0
    _attend(*lens, 2, 1, 64, dtype, True, first=0, tail=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_groups(dtype):
    _attend([20, 3], [45, 3], 100, 1, 16, dtype)
    _attend([2], [5], 512, 1, 8, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences(dtype):
    _attend([1500, 700], [1500, 700], 4, 2, 128 if dtype == torch.bfloat16 else 64, dtype)
    _attend([900], [900], 2, 2, 64, dtype, causal=False, scale=0.3)


def test_many_short_sequences():
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 9, (700,), generator=gen).tolist()
    _attend(lens, lens, 2, 1, 16, torch.float32)
    _attend(lens, lens, 2, 1, 16, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_outside_every_sequence(dtype):
    q, k, v, out, (dq, dk, dv) = _attend([40, 100], [40, 100], 4, 2, 32, dtype, first=37, tail=70)
    for t in (out, dq, dk, dv):
        assert not bool(t[:37].any()) and not bool(t[37 + 140:].any())
    # no sequence at all
    o = packed.attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert o.shape == q.shape and float(o.abs().max()) == 0
    # no token at all, and offsets past the tokens
    e = packed.attention(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=DEV))
    assert e.shape == (0, 4, 32)
    far = packed.attention(q[:50], k[:50], v[:50], torch.tensor([0, 2 ** 30], dtype=torch.int32, device=DEV))
    assert torch.equal(far, packed.attention(q[:50], k[:50], v[:50], _offs([50])))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs(dtype):
    """Slices of one fused projection, head-major tensors, an expanded output gradient, an odd storage offset."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    n, h, d = 150, 4, 32
    offs = _offs([60, 90])
    qkv = _randn(gen, n, 3, h, d, dtype=dtype).requires_grad_(True)
    out = packed.attention(*qkv.unbind(1), offs)
    want = packed.attention(*(t.detach().contiguous() for t in qkv.unbind(1)), offs)
    assert torch.equal(out, want)
    out.sum().backward()                               # an expanded (stride 0) gradient
    leaves = [t.detach().contiguous().requires_grad_(True) for t in qkv.unbind(1)]
    packed.attention(*leaves, offs).backward(torch.ones(n, h, d, dtype=dtype, device=DEV))
    for i, t in enumerate(leaves):
        assert torch.equal(qkv.grad[:, i], t.grad)
    major = [t.detach().transpose(0, 1).contiguous().transpose(0, 1) for t in qkv.unbind(1)]
    assert torch.equal(packed.attention(*major, offs), want)
    flat = torch.empty(n * h * d + 3, dtype=dtype, device=DEV)
    odd = flat[3:].view(n, h, d).copy_(qkv.detach()[:, 0])
    assert torch.equal(packed.attention(odd, *(t.detach() for t in qkv.unbind(1)[1:]), offs), want)
    wide = torch.zeros(n, h, 2 * d, dtype=dtype, device=DEV)[..., ::2].copy_(qkv.detach()[:, 0])
    assert torch.equal(packed.attention(wide, *(t.detach() for t in qkv.unbind(1)[1:]), offs), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d, at", [(16, 50), (128, 70), (128, 199)])
def test_what_is_not_seen_does_not_reach_a_row(dtype, bad, d, at):
    """Infinities and NaN in k and v from a token on: earlier rows keep their bits, and neighbours too."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    lens = [200, 30]
    offs = _offs(lens)
    q, k, v = (_randn(gen, 230, h, d, dtype=dtype) for h in (4, 2, 2))
    want = packed.attention(q, k, v, offs)
    kb, vb = k.clone(), v.clone()
    vb[at:at + 9] = bad
    got = packed.attention(q, k, vb, offs)
    keep = [*range(at), *(range(200, 230) if at + 9 <= 200 else ())]   # from 199 on the neighbour's own are bad too
    assert torch.equal(got[keep], want[keep])
    assert not bool(torch.isfinite(got[at:200]).any())
    if math.isinf(bad):
        assert bool((got[at:200].float() == bad).all())
    kb[at:at + 9] = bad
    got = packed.attention(q, kb, vb, offs)
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores far apart, all equal, and of the type's lowest value: the running maximum carries them."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    offs = _offs([150])
    q, k, v = (_randn(gen, 150, 2, 32, dtype=dtype) for _ in range(3))
    ref = _reference(q * 100, k, v, offs, offs, True, 32 ** -0.5)
    _check(packed.attention(q * 100, k, v, offs), ref["o"], ref["to"], "scores of some hundreds")
    same = packed.attention(torch.zeros_like(q), k, v, offs)
    mean = v.double().cumsum(0) / torch.arange(1, 151, device=DEV).double()[:, None, None]
    tol = (2 * UNIT[dtype] + 200 * W) * (v.double().abs().cumsum(0) / torch.arange(1, 151, device=DEV)[:, None, None]) \
        + UNIT[dtype] * mean.abs()
    _check(same, mean, tol, "equal scores")
    low = k.clone()
    low[1:] = torch.finfo(dtype).min / 256      # q . k near the lowest fp32 value: only the first key counts
    one = packed.attention(torch.ones_like(q), low, v, offs)
    assert torch.equal(one, v[:1].expand(150, -1, -1))


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit formula by central differences: error h^2 / 6 times the third derivative
    (estimated from a second step size) plus the gradients' own bounds."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    lens, hq, hk, d = [40, 9], 4, 2, 16
    offs = _offs(lens)
    q, k, v = (_randn(gen, 49, h, d, dtype=torch.float32).requires_grad_(True) for h in (hq, hk, hk))
    do = _randn(gen, 49, hq, d, dtype=torch.float32)
    out = packed.attention(q, k, v, offs)
    grads = torch.autograd.grad(out, (q, k, v), do)
    ref = _reference(q, k, v, offs, offs, True, d ** -0.5, do)
    for i, (g, name) in enumerate(zip(grads, ("dq", "dk", "dv"))):
        x = [t.detach().double() for t in (q, k, v)]
        way = _randn(gen, *g.shape, dtype=F64)

        def f(h):
            y = list(x)
            y[i] = y[i] + h * way
            return float((_reference(*y, offs, offs, True, d ** -0.5)["o"] * do.double()).sum())
        _UNIT64 = UNIT.setdefault(F64, 2.0 ** -53)
        d1, d2 = ((f(h) - f(-h)) / (2 * h) for h in (1e-3, 2e-3))
        slack = abs(d2 - d1) + 1e-9 * abs(f(0.0)) / 1e-3 + float((ref["t" + name] * way.abs()).sum())
        assert abs(float((g.double() * way).sum()) - d1) <= slack, (name, _UNIT64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_again_and_on_another_stream(dtype):
    a = _attend([500, 33], [500, 33], 8, 2, 64, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = packed.attention(a[0], a[1], a[2], _offs([500, 33]))
        grads = torch.autograd.grad(out, a[:3], torch.ones_like(out))
    torch.cuda.current_stream().wait_stream(side)
    out2 = packed.attention(a[0], a[1], a[2], _offs([500, 33]))
    grads2 = torch.autograd.grad(out2, a[:3], torch.ones_like(out2))
    assert torch.equal(out, a[3]) and torch.equal(out2, a[3])
    assert all(torch.equal(x, y) for x, y in zip(grads, grads2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_groups_wider_than_a_tile(dtype, d):
    """A token's rows take several tiles of the key blocks, the last one part empty; short sequences too."""
    _attend([9, 2], [14, 2], 100, 1, d, dtype)
    _attend([1, 0, 1, 2] * 10, [1, 0, 1, 2] * 10, 40, 1, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_sequences_than_a_wave_ranks(dtype):
    lens = [60 + (37 * i) % 80 for i in range(75)]
    _attend(lens, lens, 2, 1, 16, dtype)
    _attend(lens[:62], lens[:62], 2, 1, 64, dtype)
    _attend(lens[:63], lens[:63], 2, 1, 64, dtype, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_sequence_of_a_hundred_thousand(dtype):
    """Some rows of a sequence whose scores would not fit anywhere."""
    gen = torch.Generator(device=DEV).manual_seed(12)
    n, d = 100003, 16
    q, k, v, do = (_randn(gen, n, 1, d, dtype=dtype) for _ in range(4))
    v.requires_grad_(True)
    do[: n - 40] = 0                          # the last rows alone give dv
    offs = _offs([n])
    out = packed.attention(q, k, v, offs)
    dv, = torch.autograd.grad(out, v, do)
    want = torch.zeros(n, 1, d, dtype=F64, device=DEV)
    tol = torch.zeros_like(want)
    for i in (0, 1, 777, 50000, n - 40, n - 1):
        r = _one(q[i:i + 1].double(), k[:i + 1, 0].double(), v.detach()[:i + 1, 0].double(), True, d ** -0.5, dtype=dtype)
        _check(out.detach()[i], r["o"], r["to"], "row %d" % i)
    r = _one(q[n - 40:].double(), k[:, 0].double(), v.detach()[:, 0].double(), True, d ** -0.5, do[n - 40:].double(), dtype)
    want[:, 0], tol[:, 0] = r["dv"], r["tdv"]
    _check(dv, want, tol, "dv")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_broadcast_and_head_major_inputs(dtype):
    """One key head seen as four, heads outermost, k and v of other strides, and a gradient for v alone."""
    gen = torch.Generator(device=DEV).manual_seed(13)
    n, d = 90, 32
    offs = _offs([50, 40])
    q, do = (_randn(gen, n, 4, d, dtype=dtype) for _ in range(2))
    k1, v1 = (_randn(gen, n, 1, d, dtype=dtype).requires_grad_(True) for _ in range(2))
    out = packed.attention(q, k1.expand(-1, 4, -1), v1.expand(-1, 4, -1), offs)
    grads = torch.autograd.grad(out, (k1, v1), do)
    k4, v4 = (t.detach().expand(-1, 4, -1).contiguous().requires_grad_(True) for t in (k1, v1))
    out4 = packed.attention(q, k4, v4, offs)
    assert torch.equal(out, out4)
    for g, g4 in zip(grads, torch.autograd.grad(out4, (k4, v4), do)):
        assert torch.equal(g, g4.sum(1, keepdim=True))      # the expansion's own sum
    ref = [torch.autograd.grad(packed.attention(a, k4, v4, offs), (a, k4, v4), do)
           for a in (q.detach().requires_grad_(True),)][0]
    major = [t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True) for t in (q, k4)]
    got = torch.autograd.grad(packed.attention(*major, v4, offs), (*major, v4),
                              do.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    alone, = torch.autograd.grad(packed.attention(q, k4.detach(), v4, offs), v4, do)
    assert torch.equal(alone, ref[2])


def test_no_second_derivative():
    q = torch.randn(5, 1, 8, device=DEV, requires_grad=True)
    out = packed.attention(q, q, q, _offs([5]))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


def test_second_derivative_of_a_turn():
    """The turn is linear: the gradient of a gradient's square is twice the scale's square times the weights."""
    q = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    w = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    freq, _ = packed.rotary_frequencies(8, device=DEV)
    out, _ = packed.rotary(q, None, torch.arange(5, device=DEV), freq, scale=1.5)
    g, = torch.autograd.grad((out * w).sum(), q, create_graph=True)
    h, = torch.autograd.grad((g * g).sum(), w)
    # two turns of 12 W of a pair's sum each, and the factors
    bound = 2 * 1.5 * 1.5 * 40 * W * w.detach().double().abs().sum(-1, keepdim=True)
    _check(h, 2 * 1.5 ** 2 * w.detach().double(), bound.expand_as(h), "second derivative")


# ----------------------------------------------------------------------------- rotary
def _turned(x, pos, freq, interleaved, scale, sign=1.0):
    r = 2 * freq.numel()
    x = x.detach().double()
    t = (pos.double()[:, None] * freq.double())[:, None]
    c, s = t.cos() * scale, sign * t.sin() * scale
    y = x.clone()
    i0, i1 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
    # angle remainder pi 2^-25, sinpi / cospi 4 ulp, two products and their sum; then the storage rounding
    pair = scale * (x[..., i0].abs() + x[..., i1].abs())
    tol = torch.zeros_like(y)
    tol[..., i0] = tol[..., i1] = pair * 12 * W
    return y, tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n, hq, hk, d, rot", [(1, 1, 1, 2, 2), (5, 3, 1, 7, 4), (33, 8, 2, 64, 64), (17, 4, 4, 96, 48),
                                               (9, 2, 1, 256, 256), (9000, 2, 1, 128, 64), (9001, 1, 1, 6, 2)])
def test_rotary(dtype, interleaved, n, hq, hk, d, rot):
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, gq, gk = (_randn(gen, n, h, d, dtype=dtype) for h in (hq, hk, hq, hk))
    q.requires_grad_(True), k.requires_grad_(True)
    freq, scale = packed.rotary_frequencies(rot, scaling="parts", factor=4.0, device=DEV)
    pos = torch.randint(-50, 1 << 20, (n,), generator=gen, device=DEV)
    outs = packed.rotary(q, k, pos, freq, interleaved=interleaved, scale=scale)
    grads = torch.autograd.grad(outs, (q, k), (gq, gk))
    for x, got, sign in ((q, outs[0], 1), (k, outs[1], 1), (gq, grads[0], -1), (gk, grads[1], -1)):
        want, tol = _turned(x, pos, freq, interleaved, scale, sign)
        _check(got.detach(), want, tol * 1.01 + UNIT[dtype] * want.abs(), "rotary")
        assert torch.equal(got[..., rot:], x.detach()[..., rot:])
    for p in (pos.int(), pos.float(), pos.double()):
        again = packed.rotary(q.detach(), None, p, freq, interleaved=interleaved, scale=scale)
        assert again[1] is None and torch.equal(again[0], outs[0].detach())


def test_rotary_strides_types_and_partial_gradients():
    gen = torch.Generator(device=DEV).manual_seed(7)
    n, d = 40, 32
    freq, _ = packed.rotary_frequencies(d, device=DEV)
    pos = torch.arange(n, device=DEV)
    qkv = _randn(gen, n, 3, 4, d, dtype=torch.bfloat16)
    q, k, _ = qkv.unbind(1)
    want = packed.rotary(q.contiguous(), k.contiguous(), pos, freq)
    for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k),
                 (torch.empty(n, 4, 2 * d, dtype=q.dtype, device=DEV)[..., ::2].copy_(q), k),
                 (torch.empty(n * 4 * d + 1, dtype=q.dtype, device=DEV)[1:].view(n, 4, d).copy_(q), k)):
        got = packed.rotary(a, b, pos, freq)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(packed.rotary(q, k, pos, freq.float())[0][:1], want[0][:1])   # position 0: no turn at all
    e = packed.rotary(q[:0], k[:0], pos[:0], freq)
    assert e[0].shape == (0, 4, d)
    # a gradient through one of the two only, and an expanded one
    ql, kl = q.float().requires_grad_(True), k.float().requires_grad_(True)
    out = packed.rotary(ql, kl, pos, freq)
    gk, = torch.autograd.grad(out[1].sum(), kl, retain_graph=True)
    want, tol = _turned(torch.ones_like(kl), pos, freq, False, 1.0, -1.0)
    _check(gk, want, tol * 1.01 + W * want.abs(), "dk alone")
    gq, = torch.autograd.grad(out[0].sum(), ql)
    assert torch.equal(gq, gk)


# ----------------------------------------------------------------------------- serving
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B, L, cap, hq, hk, d, rot", [(1, 1, 1, 1, 1, 8, 8), (5, 1, 100, 8, 2, 64, 64),
                                                       (3, 7, 20, 6, 3, 32, 16), (2, 5, 9, 2, 1, 6, 4)])
def test_rotary_append(dtype, interleaved, B, L, cap, hq, hk, d, rot):
    gen = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = (_randn(gen, B, L, h, d, dtype=dtype) for h in (hq, hk, hk))
    kc, vc = (_randn(gen, B, cap, hk, d, dtype=dtype) for _ in range(2))
    lens = torch.randint(0, cap - L + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    if B > 2:
        lens[1], lens[2] = cap - L + (1 if L > 1 else 1), -1      # a row that does not fit; a row before the cache
    freq, _ = packed.rotary_frequencies(rot, device=DEV)
    k0, v0 = kc.clone(), vc.clone()
    out = packed.rotary_append(q, k, v, kc, vc, lens, freq, interleaved=interleaved, scale=1.5)
    for b, n in enumerate(lens.tolist()):
        pos = torch.arange(n, n + L, device=DEV)
        want, tol = _turned(q[b], pos, freq, interleaved, 1.5)
        _check(out[b], want, tol * 1.01 + UNIT[dtype] * want.abs(), "q of %d" % b)
        wk, tol = _turned(k[b], pos, freq, interleaved, 1.5)
        for i in range(L):
            if 0 <= n + i < cap:
                _check(kc[b, n + i], wk[i], tol[i] * 1.01 + UNIT[dtype] * wk[i].abs(), "k of %d" % b)
                assert torch.equal(vc[b, n + i], v[b, i])
        rest = [j for j in range(cap) if not n <= j < n + L]
        assert torch.equal(kc[b, rest], k0[b, rest]) and torch.equal(vc[b, rest], v0[b, rest])


def _cached(B, L, cap, lens, hq, hk, d, dtype, seed=0, scale=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = _randn(gen, B, L, hq, d, dtype=dtype)
    kc, vc = (_randn(gen, B, cap, hk, d, dtype=dtype) for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for b, x in enumerate(lens):      # behind the end: anything
        kc[b, max(0, min(x, cap)):], vc[b, max(0, min(x, cap)):] = math.nan, math.inf
    out = packed.cached_attention(q, kc, vc, n, scale=scale)
    for b, x in enumerate(lens):
        x = max(0, min(x, cap))
        z = torch.tensor([0, L], dtype=torch.int32), torch.tensor([0, x], dtype=torch.int32)
        ref = _reference(q[b], kc[b, :x], vc[b, :x], *z, True, d ** -0.5 if scale is None else scale)
        # the join of the splits adds a product and a sum for each of at most 256 of them
        _check(out[b], ref["o"], ref["to"] + 520 * W * ref["to"] / UNIT[dtype], "cached %d of %s" % (b, lens))
    return q, kc, vc, n, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, hk, d", [(1, 1, 8), (8, 2, 64), (8, 1, 128), (5, 5, 32), (12, 4, 96)])
@pytest.mark.parametrize("L", [1, 3])
def test_cached_attention(dtype, hq, hk, d, L):
    _cached(6, L, 333, [0, 1, 2, 64, 332, 333], hq, hk, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cached_attention_long_and_wide(dtype):
    _cached(2, 1, 9000, [9000, 4001], 8, 2, 128, dtype)
    _cached(1, 40, 700, [690], 8, 2, 64, dtype)           # more rows than one wave takes
    _cached(3, 5, 30, [2, 5, 30], 64, 1, 16, dtype)       # fewer rows than new tokens: the first see nothing
    _cached(2, 1, 50, [99, -4], 4, 2, 32, dtype)          # outside the capacity
    _cached(300, 1, 70, [(7 * i) % 71 for i in range(300)], 2, 1, 16, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_caches_with_heads_outermost_and_slices(dtype):
    """[B, heads, capacity, d] caches seen as [B, capacity, heads, d], and a slice of the batch and of the capacity."""
    gen = torch.Generator(device=DEV).manual_seed(14)
    B, cap, hk, d = 3, 200, 2, 64
    q, k, v = (_randn(gen, B, 2, h, d, dtype=dtype) for h in (4, hk, hk))
    dense = [_randn(gen, B, cap, hk, d, dtype=dtype) for _ in range(2)]
    lens = torch.tensor([0, 77, 198], dtype=torch.int32, device=DEV)
    freq, _ = packed.rotary_frequencies(d, device=DEV)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense]
    wide = [torch.zeros(B + 2, cap + 50, hk, d, dtype=dtype, device=DEV) for _ in range(2)]
    for w, t in zip(wide, dense):
        w[1:B + 1, 20:20 + cap] = t
    parts = [w[1:B + 1, 20:20 + cap] for w in wide]
    res = []
    for kc, vc in (dense, major, parts):
        qn = packed.rotary_append(q, k, v, kc, vc, lens, freq)
        res.append((qn, kc, vc, packed.cached_attention(qn, kc, vc, lens + 2)))
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))
    for w in wide:
        assert not bool(w[0].any()) and not bool(w[-1].any()) and not bool(w[:, :20].any()) and not bool(w[:, 220:].any())
    with pytest.raises(RuntimeError, match="16 bytes"):
        flat = torch.zeros(B * cap * hk * d + 1, dtype=dtype, device=DEV)[1:].view(B, cap, hk, d)
        packed.cached_attention(q, flat, flat, lens)


def test_two_calls_at_once():
    """The same operators on two streams with nothing between them: each has its own workspace."""
    gen = torch.Generator(device=DEV).manual_seed(15)
    q = [_randn(gen, 4, 1, 8, 64, dtype=torch.bfloat16) for _ in range(2)]
    caches = [[_randn(gen, 4, 3000, 2, 64, dtype=torch.bfloat16) for _ in range(2)] for _ in range(2)]
    lens = torch.tensor([3000, 1, 1500, 64], dtype=torch.int32, device=DEV)
    want = [packed.cached_attention(a, *c, lens) for a, c in zip(q, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(packed.cached_attention(q[i], *caches[i], lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_cached_attention_empty():
    z = torch.zeros
    i32 = torch.int32
    assert packed.cached_attention(z(0, 1, 2, 8, device=DEV), z(0, 5, 1, 8, device=DEV), z(0, 5, 1, 8, device=DEV),
                                   z(0, dtype=i32, device=DEV)).shape == (0, 1, 2, 8)
    assert packed.cached_attention(z(2, 0, 2, 8, device=DEV), z(2, 5, 1, 8, device=DEV), z(2, 5, 1, 8, device=DEV),
                                   z(2, dtype=i32, device=DEV)).shape == (2, 0, 2, 8)
    o = packed.cached_attention(torch.ones(2, 1, 2, 8, device=DEV), z(2, 0, 1, 8, device=DEV),
                                z(2, 0, 1, 8, device=DEV), z(2, dtype=i32, device=DEV))
    assert float(o.abs().max()) == 0


def test_cached_attention_beyond_32_bit_offsets():
    """Rows 4 MB apart: row 1300 lies 5.4 GB into the cache."""
    rows, step, d = 1300, 1 << 21, 128
    flat = torch.empty((rows - 1) * step + 2 * d, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(9)
    kc, vc = (flat[i * d:].as_strided((1, rows, 1, d), (rows * step, step, d, 1)) for i in range(2))
    kd, vd = (_randn(gen, 1, rows, 1, d, dtype=torch.bfloat16) for _ in range(2))
    kc.copy_(kd), vc.copy_(vd)
    q = _randn(gen, 1, 1, 4, d, dtype=torch.bfloat16)
    lens = torch.tensor([rows], dtype=torch.int32, device=DEV)
    assert torch.equal(packed.cached_attention(q, kc, vc, lens), packed.cached_attention(q, kd, vd, lens))


@pytest.mark.parametrize("dtype", DTYPES)
def test_serving_agrees_with_training(dtype):
    """The operators together: turn, attend and differentiate packed histories; then serve the same histories token by
    token, and in blocks, from a cache, and get the same rows."""
    gen = torch.Generator(device=DEV).manual_seed(10)
    lens, hq, hk, d = [12, 3, 40], 4, 2, 32
    n, cap = sum(lens), 64
    offs = _offs(lens)
    q, k, v, do = (_randn(gen, n, h, d, dtype=dtype) for h in (hq, hk, hk, hq))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    freq, scale = packed.rotary_frequencies(16, scaling="base", factor=2.0, device=DEV)
    pos = torch.cat([torch.arange(m, device=DEV) for m in lens])
    qt, kt = packed.rotary(q, k, pos, freq, scale=scale)
    out = packed.attention(qt, kt, v, offs)
    grads = torch.autograd.grad(out, leaves, do)
    ref = _reference(qt, kt, v, offs, offs, True, d ** -0.5, do)
    _check(out.detach(), ref["o"], ref["to"], "out")
    _check(grads[2], ref["dv"], ref["tdv"], "dv")
    for g, name, x in ((grads[0], "dq", q), (grads[1], "dk", k)):
        back, _ = _turned(ref[name].float(), pos, freq, False, scale, -1.0)
        # the turned gradient was rounded once more on its way; a turn mixes two features' bounds
        bound = ref["t" + name]
        mix = (bound.sum(-1, keepdim=True) + ref[name].abs().amax(-1, keepdim=True) * 2 * UNIT[dtype])
        _check(g, back, mix + 2 * UNIT[dtype] * back.abs(), name)
    ref = _reference(qt, kt, v, offs, offs, True, d ** -0.5)
    starts = offs.tolist()
    for step in (1, 5):
        kc, vc = (torch.full((3, cap, hk, d), math.nan, dtype=dtype, device=DEV) for _ in range(2))
        count = torch.zeros(3, dtype=torch.int32, device=DEV)
        for t in range(0, 40, step):
            rows = torch.tensor([[min(starts[b] + t + i, n - 1) for i in range(step)] for b in range(3)], device=DEV)
            qn = packed.rotary_append(q.detach()[rows], k.detach()[rows], v.detach()[rows], kc, vc, count, freq,
                                      scale=scale)
            count += step
            got = packed.cached_attention(qn, kc, vc, count)
            for b in range(3):
                for i in range(step):
                    if t + i < lens[b]:
                        at = starts[b] + t + i
                        _check(got[b, i], ref["o"][at], ref["to"][at] * (1 + 520 * W / UNIT[dtype]),
                               "step %d, history %d, token %d" % (step, b, t + i))


def test_captured_training_and_serving():
    """One HIP graph of turn, attention and backward, and one of a serving step, each replayed with eager work between
    and checked against the eager result every time."""
    gen = torch.Generator(device=DEV).manual_seed(11)
    lens, hq, hk, d = [70, 1, 0, 200], 8, 2, 64
    n, dtype = sum(lens), torch.bfloat16
    offs = _offs(lens)
    freq, _ = packed.rotary_frequencies(d, device=DEV)
    pos = torch.cat([torch.arange(m, device=DEV) for m in lens])

    def fresh():
        return [_randn(gen, n, h, d, dtype=dtype) for h in (hq, hk, hk, hq)]

    def step(q, k, v, do):
        out = packed.attention(*packed.rotary(q, k, pos, freq), v, offs)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))

    held = fresh()
    for t in held[:3]:
        t.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*held)

    B, cap = 5, 300
    kc, vc = (_randn(gen, B, cap, hk, d, dtype=dtype) for _ in range(2))
    sq, sk, sv = (_randn(gen, B, 1, h, d, dtype=dtype) for h in (hq, hk, hk))
    count = torch.tensor([0, 1, 63, 64, 250], dtype=torch.int32, device=DEV)

    def serve(kc, vc, count):
        qn = packed.rotary_append(sq, sk, sv, kc, vc, count, freq)
        count.add_(1)
        return packed.cached_attention(qn, kc, vc, count)

    serve(kc.clone(), vc.clone(), count.clone())
    ke, ve, ce = kc.clone(), vc.clone(), count.clone()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        res2 = serve(kc, vc, count)
    for _ in range(4):
        new = fresh()
        with torch.no_grad():
            for t, x in zip(held, new):
                t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*[x.requires_grad_(True) if i < 3 else x for i, x in enumerate(new)])
        assert all(torch.equal(a, b) for a, b in zip(res, want))
        for x in (sq, sk, sv):
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        graph2.replay()
        want = serve(ke, ve, ce)
        torch.cuda.synchronize()
        assert torch.equal(res2, want) and torch.equal(kc, ke) and torch.equal(vc, ve) and torch.equal(count, ce)
