"""Attention over packed histories with rotary positions: the cases that are timed and their plain forms.

Four operators of ``tagan_amd.packed``: ``rotary`` (training), ``attention`` (packed sequences of different lengths,
causal, grouped heads; forward, and forward with backward), and for serving ``rotary_append`` (new tokens into a cache)
and ``cached_attention`` (new tokens against the cache).  ``run`` computes the plain form in 32 bits (angles in 64)
with elementary torch operations, or calls the framework where ``own`` is set; ``exact`` states each definition once
more in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ----------------------------------------------------------------------------------------------------- the cases
def _rotary(tokens, heads, kv_heads, dim, rot, dtype, *, train=False, interleaved=False, far=0, factor=1.0):
    return {"op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "dtype": dtype, "train": train, "interleaved": interleaved, "far": far, "factor": factor}


def _append(batch, new, capacity, heads, kv_heads, dim, rot, dtype, *, interleaved=False):
    return {"op": "append", "batch": batch, "new": new, "capacity": capacity, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "dtype": dtype, "interleaved": interleaved}


def _attention(seqs, low, high, heads, kv_heads, dim, dtype, *, train=False, past=0, causal=True):
    return {"op": "attention", "seqs": seqs, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "train": train, "past": past, "causal": causal}


def _cached(batch, new, low, high, heads, kv_heads, dim, dtype):
    return {"op": "cached", "batch": batch, "new": new, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def listed():
    return [
        # a training batch of packed histories: a part of each head rotated, neighbouring pairs, there and back
        dict(_rotary(24001, 32, 8, 128, 64, "bf16", train=True, interleaved=True), name="rotary_train"),
        # event times far beyond the trained range, frequencies stretched by parts, fp32
        dict(_rotary(8003, 16, 16, 96, 96, "f32", far=1000000, factor=8.0), name="rotary_far_f32"),
        # one new event for each of 48 histories: rotate q and k, write k and v behind each history's end
        dict(_append(48, 1, 2048, 32, 8, 128, 128, "bf16"), name="append_step"),
        # a block of events for each of 5 histories, half of each head rotated, fp32
        dict(_append(5, 130, 1500, 8, 4, 64, 32, "f32", interleaved=True), name="append_block_f32"),
        # the framework's own width (H = 128, 8 heads of 16) on 1200 node histories of 1 to 64 events, fp32 training
        dict(_attention(1200, 1, 64, 8, 8, 16, "f32", train=True), name="nodes_train_f32"),
        # medium histories, every head with its own keys, training; 100 earlier events that only serve as keys
        dict(_attention(48, 17, 512, 12, 12, 64, "bf16", train=True, past=100), name="train_64"),
        # long ragged histories, four query heads to a key head, training
        dict(_attention(6, 900, 4096, 16, 4, 128, "bf16", train=True), name="train_long"),
        # one very long history read in whole before serving, eight query heads to a key head
        dict(_attention(1, 16384, 16384, 16, 2, 128, "bf16"), name="prompt_long"),
        # a batch of prompts of very different lengths, forward
        dict(_attention(13, 5, 2500, 32, 8, 128, "bf16"), name="prompt_ragged"),
        # one event of one history: the smallest serving call
        dict(_cached(1, 1, 777, 777, 8, 2, 64, "bf16"), name="cached_one"),
        # a full serving batch, ragged histories, grouped heads
        dict(_cached(64, 1, 11, 8000, 32, 8, 128, "bf16"), name="cached_batch"),
        # three events at once against two very long histories with one key head, fp32
        dict(_cached(2, 3, 40001, 70000, 8, 1, 128, "f32"), name="cached_long_f32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ranges; sizes are spread over their logarithm and bounded by the listed cost."""
    dtype = rng.choice(["bf16", "bf16", "f32"])
    dim = rng.choice([16, 32, 64, 64, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 8 else [1, 2, 4])
    op = rng.choice(["rotary", "append", "attention", "attention", "attention", "cached", "cached"])
    if op == "rotary":
        return _rotary(_log(rng, 1, 24000), heads, kv_heads, dim, dim if rng.random() < 0.5 else dim // 2, dtype,
                       train=rng.random() < 0.6, interleaved=rng.random() < 0.5,
                       far=rng.choice([0, 200000, 1000000]), factor=rng.choice([1.0, 4.0, 8.0]))
    if op == "append":
        new = _log(rng, 1, 130)
        return _append(_log(rng, 1, 64), new, new + _log(rng, 10, 1000), heads, kv_heads, dim,
                       dim if rng.random() < 0.5 else dim // 2, dtype, interleaved=rng.random() < 0.5)
    if op == "attention":
        train = rng.random() < 0.6
        high = _log(rng, 1, 4096)
        # the padded scores of the plain form bound the cost: at most 2^30 of them (2^28 in fp32, whose matrix rate
        # is a sixteenth)
        most = (1 << (28 if dtype == "f32" else 30)) // (heads * high * high)
        return _attention(_log(rng, 1, max(1, min(most, 800))), max(1, high // rng.choice([1, 3, 50])), high, heads,
                          kv_heads, dim, dtype, train=train, past=rng.choice([0, 0, 33, 200]) if high < 2000 else 0,
                          causal=rng.random() < 0.8)
    high = _log(rng, 3, 60000)
    most = (1 << 26) // (high * kv_heads)   # tokens times key heads of one cache
    return _cached(_log(rng, 1, max(1, min(most, 100))), rng.choice([1, 1, 1, 2, 5]), max(1, high // 7), high, heads,
                   kv_heads, dim, dtype)


def _lengths(count, low, high):
    """`count` lengths from `low` to `high`, spread evenly in an order without a trend; the last is the longest."""
    got = [low + int((high - low) * math.fmod(0.6180339887498949 * (i + 1), 1.0)) for i in range(count)]
    got[-1] = high
    return got


def _offsets(lens):
    got = [0]
    for n in lens:
        got.append(got[-1] + n)
    return got


def _frequencies(rot, factor):
    """base^(-2i/rot), divided by `factor` where a turn is long against 4096 positions, kept where it is short, and a
    linear ramp between one and 32 turns."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / factor * (1 - keep)


# ----------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    s = dict(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["tokens"]
        s["q"], s["k"] = normal(n, hq, d), normal(n, hk, d)
        if case["far"]:
            s["pos"] = torch.randint(0, case["far"], (n,), generator=gen, device="cuda")
        else:
            s["pos"] = torch.arange(n, device="cuda") % 777 + seed % 100
        s["freq"] = _frequencies(case["rot"], case["factor"]).cuda()
        s["scale"] = 0.1 * math.log(case["factor"]) + 1.0
        if case["train"]:
            s["dq"], s["dk"] = normal(n, hq, d), normal(n, hk, d)
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
    elif case["op"] == "append":
        b, new, cap = case["batch"], case["new"], case["capacity"]
        s["q"], s["k"], s["v"] = normal(b, new, hq, d), normal(b, new, hk, d), normal(b, new, hk, d)
        s["k_cache"], s["v_cache"] = normal(b, cap, hk, d), normal(b, cap, hk, d)
        s["lens"] = torch.randint(0, cap - new + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        s["freq"] = _frequencies(case["rot"], 1.0).cuda()
    elif case["op"] == "attention":
        lens = _lengths(case["seqs"], case["low"], case["high"])
        klens = [n + case["past"] for n in lens]
        offs, koffs = _offsets(lens), _offsets(klens)
        s["q"], s["k"], s["v"] = normal(offs[-1], hq, d), normal(koffs[-1], hk, d), normal(koffs[-1], hk, d)
        s["offsets"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
        s["offsets_k"] = torch.tensor(koffs, dtype=torch.int32, device="cuda") if case["past"] else None
        s["most"], s["most_k"] = max(lens), max(klens)
        if case["train"]:
            s["dout"] = normal(offs[-1], hq, d)
            for name in ("q", "k", "v"):
                s[name].requires_grad_(True)
    else:
        lens = [max(n, case["new"]) for n in _lengths(case["batch"], case["low"], case["high"])]
        s["q"] = normal(case["batch"], case["new"], hq, d)
        s["k_cache"], s["v_cache"] = (normal(case["batch"], max(lens) + 37, hk, d) for _ in range(2))
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return s


# ----------------------------------------------------------------------------------------------------- plain forms
def _angles(pos, freq, scale):
    a = pos.to(torch.float64)[:, None] * freq
    return (a.cos() * scale).float()[:, None, :], (a.sin() * scale).float()[:, None, :]


def _turned(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] features of each head turned by the angles, the others as they are."""
    r = 2 * cos.shape[-1]
    y = x.float().clone()
    if interleaved:
        a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = y[..., :r // 2].clone(), y[..., r // 2:r].clone()
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    return y.to(x.dtype)


def _plain_rotary(s):
    cos, sin = _angles(s["pos"], s["freq"], s["scale"])
    out = [_turned(s["q"], cos, sin, s["interleaved"]), _turned(s["k"], cos, sin, s["interleaved"])]
    if s["train"]:   # a turn's gradient is the turn back
        out += [_turned(s["dq"], cos, -sin, s["interleaved"]), _turned(s["dk"], cos, -sin, s["interleaved"])]
    return out


def _plain_append(s):
    b, new = s["q"].shape[:2]
    pos = s["lens"].long()[:, None] + torch.arange(new, device="cuda")
    cos, sin = _angles(pos.reshape(-1), s["freq"], 1.0)
    q = _turned(s["q"].reshape(b * new, *s["q"].shape[2:]), cos, sin, s["interleaved"]).view_as(s["q"])
    k = _turned(s["k"].reshape(b * new, *s["k"].shape[2:]), cos, sin, s["interleaved"]).view_as(s["k"])
    row = torch.arange(b, device="cuda")[:, None].expand(b, new)
    s["k_cache"][row, pos] = k
    s["v_cache"][row, pos] = s["v"]
    return [q, s["k_cache"], s["v_cache"]]


def _padded(x, offsets, most):
    """[B, most, heads, dim] in fp32, zero behind each sequence's end, and which places hold a token."""
    at = offsets[:-1, None].long() + torch.arange(most, device="cuda")
    ok = at < offsets[1:, None]
    return torch.where(ok[..., None, None], x[at.clamp(max=x.shape[0] - 1)].float(), 0.0), ok


def _packed(x, offsets, n, like):
    """The tokens of [B, most, heads, dim] behind one another, rounded to the type of `like`."""
    token = torch.arange(n, device="cuda")
    b = torch.searchsorted(offsets[1:].contiguous(), token.to(offsets.dtype), right=True)
    return x[b, token - offsets[b]].to(like.dtype)


def _probabilities(q, k, see):
    """softmax(q k^T) over the visible keys, zero rows where none is: q [B, kv, L*G, d], k [B, kv, S, d],
    see [B, L, S] or [B, 1, S]."""
    p = torch.matmul(q, k.transpose(-1, -2).contiguous())
    v = p.view(p.shape[0], p.shape[1], see.shape[1], -1, p.shape[3])
    v.masked_fill_(~see[:, None, :, None, :], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _plain_attention(s):
    koffs = s["offsets"] if s["offsets_k"] is None else s["offsets_k"]
    qp, qok = _padded(s["q"].detach(), s["offsets"], s["most"])
    kp, kok = _padded(s["k"].detach(), koffs, s["most_k"])
    vp, _ = _padded(s["v"].detach(), koffs, s["most_k"])
    b, lq, hq, d = qp.shape
    lk, hk, g = kp.shape[1], kp.shape[2], hq // kp.shape[2]

    def grouped(x):     # [B, L, hk * g, d] -> [B, hk, L * g, d]
        return x.view(b, lq, hk, g, d).transpose(1, 2).reshape(b, hk, lq * g, d)

    def back(x):
        return x.view(b, hk, lq, g, d).transpose(1, 2).reshape(b, lq, hq, d)

    scale = d ** -0.5
    qh, kh, vh = grouped(qp) * scale, kp.transpose(1, 2).contiguous(), vp.transpose(1, 2).contiguous()
    see = kok[:, None, :] & qok[:, :, None]
    if s["causal"]:     # the last query sees the last key
        past = (koffs[1:] - koffs[:-1] - s["offsets"][1:] + s["offsets"][:-1])[:, None, None]
        see = see & (torch.arange(lk, device="cuda") <= torch.arange(lq, device="cuda")[:, None] + past)
    p = _probabilities(qh, kh, see)
    o = torch.matmul(p, vh)
    out = [_packed(back(o), s["offsets"], s["q"].shape[0], s["q"])]
    if s["train"]:
        do = grouped(_padded(s["dout"], s["offsets"], s["most"])[0])
        dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
        ds = torch.matmul(do, vh.transpose(-1, -2).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
        dq = torch.matmul(ds, kh) * scale
        dk = torch.matmul(ds.transpose(-1, -2).contiguous(), qh)
        n, nk = s["q"].shape[0], s["k"].shape[0]
        out += [_packed(back(dq), s["offsets"], n, s["q"]),
                _packed(dk.transpose(1, 2), koffs, nk, s["k"]), _packed(dv.transpose(1, 2), koffs, nk, s["v"])]
    return out


def _plain_cached(s):
    b, new, hq, d = s["q"].shape
    cap, hk = s["k_cache"].shape[1:3]
    g = hq // hk
    qh = (s["q"].float() * d ** -0.5).view(b, new, hk, g, d).transpose(1, 2).reshape(b, hk, new * g, d)
    end = s["lens"].long()[:, None] - new + 1 + torch.arange(new, device="cuda")
    see = torch.arange(cap, device="cuda") < end[..., None]
    p = _probabilities(qh, s["k_cache"].float().transpose(1, 2).contiguous(), see)
    o = torch.matmul(p, s["v_cache"].float().transpose(1, 2).contiguous())
    return o.view(b, hk, new, g, d).transpose(1, 2).reshape(b, new, hq, d).to(s["q"].dtype)


def run(s):
    if own:
        return _framework(s)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention,
            "cached": _plain_cached}[s["op"]](s)


# ----------------------------------------------------------------------------------------------------- the framework
def _framework(s):
    from tagan_amd import packed
    if s["op"] == "rotary":
        q, k = packed.rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=s["interleaved"], scale=s["scale"])
        if not s["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    if s["op"] == "append":
        q = packed.rotary_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lens"], s["freq"],
                                 interleaved=s["interleaved"])
        return [q, s["k_cache"], s["v_cache"]]
    if s["op"] == "attention":
        out = packed.attention(s["q"], s["k"], s["v"], s["offsets"], s["offsets_k"], causal=s["causal"])
        if not s["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]
    return packed.cached_attention(s["q"], s["k_cache"], s["v_cache"], s["lens"])


# ----------------------------------------------------------------------------------------------------- the floor
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        passes = 2 if case["train"] else 1
        n = case["tokens"]
        return {"bytes": passes * (2 * n * (hq + hk) * d * size + n * 8),
                "flops": passes * 3 * n * (hq + hk) * case["rot"]}
    if case["op"] == "append":
        n = case["batch"] * case["new"]
        return {"bytes": 2 * n * (hq + 2 * hk) * d * size, "flops": 3 * n * (hq + hk) * case["rot"]}
    if case["op"] == "attention":
        lens = _lengths(case["seqs"], case["low"], case["high"])
        past = case["past"]
        pairs = sum(n * past + n * (n + 1) // 2 if case["causal"] else n * (n + past) for n in lens)
        nq, nk = sum(lens), sum(lens) + past * len(lens)
        # two products forward; five backward, for the probabilities are made again and not kept
        flops = 2 * pairs * hq * d * (7 if case["train"] else 2)
        tensors = 2 * nq * hq + 2 * nk * hk
        return {"bytes": size * d * tensors * (2 if case["train"] else 1), "flops": flops}
    lens = [max(n, case["new"]) for n in _lengths(case["batch"], case["low"], case["high"])]
    new = case["new"]
    pairs = sum(new * n - new * (new - 1) // 2 for n in lens)
    return {"bytes": size * d * (2 * sum(lens) * hk + 2 * case["batch"] * new * hq), "flops": 4 * pairs * hq * d}


# ----------------------------------------------------------------------------------------------------- in 64 bits
def _exact_turn(x, pos, freq, scale, interleaved, sign):
    """Each pair as a complex number times scale * exp(i * angle)."""
    n, r = x.shape[0], 2 * freq.numel()
    y = x.detach().double()
    a = sign * pos.double().reshape(n, 1, 1) * freq.double()
    turn = torch.polar(torch.full_like(a, scale), a)
    head = y[..., :r]
    if interleaved:
        z = torch.view_as_complex(head.reshape(n, -1, r // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(n, -1, r)
    else:
        z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, y[..., r:]], -1)


def _exact_heads(q, k, v, causal, do=None):
    """One sequence: q [L, hq, d], k and v [S, hk, d] in 64 bits, head by head."""
    lq, hq, d = q.shape
    lk, hk = k.shape[:2]
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if do is not None else None
    if lq == 0 or lk == 0:
        return o, grads
    hidden = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1) if causal else None
    for h in range(hq):
        kh, vh = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        z = (q[:, h] @ kh.T) / math.sqrt(d)
        if causal:
            z[hidden] = -math.inf
        w = torch.softmax(z, 1).nan_to_num(0.0)
        o[:, h] = w @ vh
        if do is not None:
            g = do[:, h] @ vh.T
            g = w * (g - (g * w).sum(1, keepdim=True)) / math.sqrt(d)
            grads[0][:, h] = g @ kh
            grads[1][:, h // (hq // hk)] += g.T @ q[:, h]
            grads[2][:, h // (hq // hk)] += w.T @ do[:, h]
    return o, grads


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        rest = (s["pos"], s["freq"], s["scale"], case["interleaved"])
        out = [_exact_turn(s["q"], *rest, 1.0), _exact_turn(s["k"], *rest, 1.0)]
        if case["train"]:
            out += [_exact_turn(s["dq"], *rest, -1.0), _exact_turn(s["dk"], *rest, -1.0)]
        return out
    if case["op"] == "append":
        new = case["new"]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        qs = []
        for b, n in enumerate(s["lens"].tolist()):
            pos = torch.arange(n, n + new, device="cuda")
            qs.append(_exact_turn(s["q"][b], pos, s["freq"], 1.0, case["interleaved"], 1.0))
            kc[b, n:n + new] = _exact_turn(s["k"][b], pos, s["freq"], 1.0, case["interleaved"], 1.0)
            vc[b, n:n + new] = s["v"][b].double()
        return [torch.stack(qs), kc, vc]
    if case["op"] == "attention":
        offs = s["offsets"].tolist()
        koffs = offs if s["offsets_k"] is None else s["offsets_k"].tolist()
        q, k, v = (s[x].detach().double() for x in "qkv")
        do = s["dout"].double() if case["train"] else None
        outs, grads = [], []
        for a, e, ka, ke in zip(offs, offs[1:], koffs, koffs[1:]):
            o, g = _exact_heads(q[a:e], k[ka:ke], v[ka:ke], case["causal"], do[a:e] if case["train"] else None)
            outs.append(o)
            grads.append(g)
        return [torch.cat(outs)] + ([torch.cat(x) for x in zip(*grads)] if case["train"] else [])
    outs = []
    for b, n in enumerate(s["lens"].tolist()):
        outs.append(_exact_heads(s["q"][b].double(), s["k_cache"][b, :n].double(), s["v_cache"][b, :n].double(),
                                 True)[0])
    return torch.stack(outs)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
