"""Attention over packed histories with rotary positions (csrc/packed_attn.hip, csrc/rotary.hip).

Beside the rectangular temporal attention of ``kernels.TemporalAttnFn`` ([rows, T], equal heads, T <= 128 on the matrix
cores): histories of different lengths lie behind one another in one token axis, several query heads may share a key
head, and positions enter as turns of the query and key features.

* ``rotary_frequencies`` / ``rotary``        turn q and k by their positions (differentiable)
* ``attention``                              softmax attention inside each packed history (differentiable)
* ``rotary_append`` / ``cached_attention``   serving: write new tokens behind each cached history, attend to it

fp32 or bf16 storage, fp32 statistics and sums.  Everything runs on the current HIP stream of the tensors' device,
allocates from PyTorch's caching allocator only, never waits for the device and can be captured in a HIP graph; offsets
and lengths stay on the device.  Wrong arguments raise TypeError / ValueError before anything is launched.

A captured backward: capture forward and backward together (``graph_step.GraphedStep``) and let no eager graph of the
same leaves live across the capture: such a graph keeps the leaves' gradient accumulation on the eager stream, which a
capture must not touch.
"""
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import check, dtype_code, lib, ptr, require_hip, stream_of

MAX_HEAD_DIM = 128        # attention: multiples of 8 up to this
MAX_ROTARY_DIM = 256
MAX_GROUP = 512           # query heads to a key head
MAX_TOKEN_STRIDE = 1 << 21
_POS_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


# ----------------------------------------------------------------------------- arguments
def _need(ok: bool, text: str, *args) -> None:
    if not ok:
        raise ValueError(text % args)


def _on_device(first: torch.Tensor, *rest) -> None:
    require_hip(first, *rest)
    for t in rest:
        if t is not None and t.device != first.device:
            raise ValueError("tensors on %s and %s" % (first.device, t.device))


def _storage(first: torch.Tensor, *rest) -> None:
    for t in (first,) + rest:
        if t is not None and t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("float32 or bfloat16 is wanted, got %s" % t.dtype)
        if t is not None and t.dtype != first.dtype:
            raise TypeError("tensors of %s and %s" % (first.dtype, t.dtype))


def _index(t: torch.Tensor, name: str, size: Optional[int] = None) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError("%s has to be int32, got %s" % (name, t.dtype))
    _need(t.dim() == 1 and (size is None or t.shape[0] == size), "%s has shape %s", name, tuple(t.shape))
    return t.contiguous()


def _heads(heads: int, kv_heads: int) -> None:
    _need(kv_heads >= 1 and heads >= kv_heads and heads % kv_heads == 0 and heads // kv_heads <= MAX_GROUP,
          "%d query heads over %d key heads", heads, kv_heads)


def _strides(t: torch.Tensor):
    """Element strides of all axes but the last; an axis of one step gets its dense stride."""
    got, dense = [], t.shape[-1]
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        got.append(s if n > 1 else dense)
        dense *= max(n, 1)
    return got[::-1]


def _fits(t: torch.Tensor, spread: int = 1 << 30) -> bool:
    """Whether the attention kernels can read t in place: 16-byte runs, whole rows, a tile within 32-bit offsets."""
    if t.stride(-1) != 1 or t.data_ptr() % 16:
        return False
    st, es = _strides(t), t.element_size()
    return (all(s >= 0 and s * es % 16 == 0 for s in st) and t.shape[-1] <= st[-2] <= MAX_TOKEN_STRIDE
            and st[-1] * t.shape[-2] * es < spread)


def _dense(t: torch.Tensor) -> torch.Tensor:
    if _fits(t):
        return t
    t = t.contiguous()
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


def _run(name: str, t: torch.Tensor, *args) -> None:
    """The C entry on the device and current stream of t."""
    if t.device.index == torch.cuda.current_device():
        check(getattr(lib(), name)(*args, stream_of(t)), name)
    else:
        with torch.cuda.device(t.device):
            check(getattr(lib(), name)(*args, stream_of(t)), name)


# ----------------------------------------------------------------------------- rotary positions
def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_len: int = 4096, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inverse frequencies [dim / 2] in fp64, scale) for ``rotary``: base^(-2i/dim), i < dim / 2.

    ``scaling`` for histories ``factor`` times longer than the ``original_len`` positions a model was trained on:
    ``"linear"`` divides every frequency by ``factor``; ``"base"`` raises the base to base * factor^(dim / (dim - 2)),
    so that the slowest pair is stretched by ``factor`` and the fastest is kept; ``"parts"`` keeps pairs that make at
    least ``fast`` turns over ``original_len``, divides those that make at most ``slow``, goes linearly (in turns)
    between, and returns the scale 0.1 ln(factor) + 1.  The scale is 1 otherwise.
    """
    _need(dim >= 2 and dim % 2 == 0, "%d features cannot be turned in pairs", dim)
    _need(base > 0 and math.isfinite(base) and factor >= 1 and math.isfinite(factor), "base %g, factor %g", base,
          factor)
    if scaling == "base":
        _need(dim > 2, "the base cannot be raised for %d features", dim)
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        _need(fast > slow and original_len >= 1, "turns %g to %g over %d positions", slow, fast, original_len)
        turns = original_len * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError("scaling %r (None, 'linear', 'base' or 'parts')" % (scaling,))
    return freq.to(device) if device is not None else freq, scale


def _frequencies(inv_freq: torch.Tensor, dim: int) -> torch.Tensor:
    if inv_freq.dtype not in (torch.float64, torch.float32):
        raise TypeError("inv_freq has to be float64 or float32, got %s" % inv_freq.dtype)
    _need(inv_freq.dim() == 1 and 1 <= inv_freq.shape[0] and 2 * inv_freq.shape[0] <= dim <= MAX_ROTARY_DIM,
          "%s frequencies for heads of %d features (up to %d)", tuple(inv_freq.shape), dim, MAX_ROTARY_DIM)
    return inv_freq.to(torch.float64).contiguous()


def _turn(q, k, positions, inv_freq, interleaved, scale, inverse):
    n, _, d = q.shape
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
    if n == 0:
        return qo, ko
    q = q if q.stride(-1) == 1 else q.contiguous()
    k = k if k is None or k.stride(-1) == 1 else k.contiguous()
    hk = k.shape[1] if k is not None else 0
    _run("tagan_rotary", q, dtype_code(q), n, q.shape[1], hk, d, 2 * inv_freq.shape[0], ptr(q), *_strides(q), ptr(k),
         *(_strides(k) if hk else (0, 0)), ptr(positions), _POS_TYPES[positions.dtype], ptr(inv_freq), scale,
         interleaved, inverse, ptr(qo), *_strides(qo), ptr(ko), *(_strides(ko) if hk else (0, 0)))
    return qo, ko


class RotaryFn(torch.autograd.Function):
    """(q, k) turned by their positions; the gradient is turned back."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved: bool, scale: float):
        ctx.save_for_backward(positions, inv_freq)
        ctx.cfg = (interleaved, scale)
        ctx.set_materialize_grads(False)
        return _turn(q, k, positions, inv_freq, interleaved, scale, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 6
        if dq is None:
            dk, _ = _turn(dk, None, positions, inv_freq, *ctx.cfg, 1)
        else:
            dq, dk = _turn(dq, dk, positions, inv_freq, *ctx.cfg, 1)
        return dq, dk, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
           interleaved: bool = False, scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [N, heads, d] and k [N, kv_heads, d] (or None) turned by ``positions`` [N] (int32, int64, float32 or float64:
    indices or event times) times ``inv_freq`` [r / 2]: the first r features of each head in pairs (i, i + r/2), or
    (2i, 2i + 1) with ``interleaved``, times ``scale``; the features behind them are copied.  Angles are formed in
    fp64.  Gradients flow to q and k."""
    _storage(q, k)
    _need(q.dim() == 3 and (k is None or (k.dim() == 3 and k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2])),
          "q %s and k %s", tuple(q.shape), None if k is None else tuple(k.shape))
    _need(q.shape[1] >= 1 and (k is None or k.shape[1] >= 1), "no heads")
    if positions.dtype not in _POS_TYPES:
        raise TypeError("positions of %s" % positions.dtype)
    _need(positions.shape == (q.shape[0],), "%s positions for %d tokens", tuple(positions.shape), q.shape[0])
    _need(math.isfinite(scale), "scale %g", scale)
    inv_freq = _frequencies(inv_freq, q.shape[2])
    _on_device(q, k, positions, inv_freq)
    return RotaryFn.apply(q, k, positions.contiguous(), inv_freq, bool(interleaved), float(scale))


def _cache(t: torch.Tensor, name: str) -> None:
    _need(t.dim() == 4, "%s %s: [batch, capacity, heads, features] is wanted", name, tuple(t.shape))
    _need(not t.requires_grad, "%s is written and read in place: it cannot require a gradient", name)
    _need(t.stride(-1) == 1, "%s needs unit feature stride", name)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  lens: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
                  scale: float = 1.0) -> torch.Tensor:
    """New tokens q [B, L, heads, d], k and v [B, L, kv_heads, d] at positions ``lens[b] + i``: writes turned k and v
    to rows ``lens[b] + i`` of the caches [B, capacity, kv_heads, d] in place and returns the turned q, in one launch.

    ``lens`` [B] int32 counts the rows already there and is not advanced; rows that would lie outside the capacity are
    not written.  No autograd."""
    _storage(q, k, v, k_cache, v_cache)
    _cache(k_cache, "k_cache")
    _cache(v_cache, "v_cache")
    _need(q.dim() == 4 and k.dim() == 4 and k.shape == v.shape and q.shape[:2] == k.shape[:2]
          and q.shape[3] == k.shape[3], "q %s, k %s and v %s", tuple(q.shape), tuple(k.shape), tuple(v.shape))
    B, L, heads, d = q.shape
    hk = k.shape[2]
    _heads(heads, hk)
    _need(k_cache.shape == v_cache.shape and k_cache.shape[0] == B and k_cache.shape[2:] == k.shape[2:],
          "caches %s and %s for k %s", tuple(k_cache.shape), tuple(v_cache.shape), tuple(k.shape))
    for c in (k_cache, v_cache):
        _need(all(s > 0 for n, s in zip(c.shape, c.stride()) if n > 1), "a cache with shared rows cannot be written")
    lens = _index(lens, "lens", B)
    _need(math.isfinite(scale), "scale %g", scale)
    inv_freq = _frequencies(inv_freq, d)
    _on_device(q, k, v, k_cache, v_cache, lens, inv_freq)
    q, k, v = (t.detach() if t.stride(-1) == 1 else t.detach().contiguous() for t in (q, k, v))
    out = torch.empty((B, L, heads, d), dtype=q.dtype, device=q.device)
    if B and L:
        _run("tagan_rotary_append", q, dtype_code(q), B, L, heads, hk, d, 2 * inv_freq.shape[0], ptr(q), *_strides(q),
             ptr(k), *_strides(k), ptr(v), *_strides(v), ptr(lens), ptr(inv_freq), float(scale), int(interleaved),
             ptr(out), *_strides(out), ptr(k_cache), *_strides(k_cache), ptr(v_cache), *_strides(v_cache),
             k_cache.shape[1])
    return out


# ----------------------------------------------------------------------------- packed attention
class PackedAttnFn(torch.autograd.Function):
    """softmax(scale q kᵀ) v inside each packed sequence; saves the output and the rows' log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, offsets, offsets_k, causal: bool, scale: float):
        q, k, v = _dense(q), _dense(k), _dense(v)
        n, heads, d = q.shape
        nk, hk, _ = k.shape
        out = torch.empty((n, heads, d), dtype=q.dtype, device=q.device)
        needs = any(ctx.needs_input_grad[:3])
        lse = torch.empty((n, heads), dtype=torch.float32, device=q.device) if needs else None
        if n:
            _run("tagan_packed_attn_fwd", q, dtype_code(q), offsets.shape[0] - 1, n, nk, heads, hk, d, ptr(q),
                 *_strides(q), ptr(k), *_strides(k), ptr(v), *_strides(v), ptr(offsets), ptr(offsets_k), int(causal),
                 scale, ptr(out), *_strides(out), ptr(lse))
        if needs:
            ctx.save_for_backward(q, k, v, out, lse, offsets, offsets_k)
            ctx.cfg = (causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, offsets, offsets_k = ctx.saved_tensors
        causal, scale = ctx.cfg
        dout = _dense(dout)
        n, heads, d = q.shape
        nk, hk, _ = k.shape
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if n or nk:
            size = lib().tagan_packed_attn_bwd_workspace(n, heads)
            ws = torch.empty(max(int(size), 1), dtype=torch.uint8, device=q.device)
            _run("tagan_packed_attn_bwd", q, dtype_code(q), offsets.shape[0] - 1, n, nk, heads, hk, d, ptr(q),
                 *_strides(q), ptr(k), *_strides(k), ptr(v), *_strides(v), ptr(offsets), ptr(offsets_k), int(causal),
                 scale, ptr(out), *_strides(out)[:2], ptr(lse), ptr(dout), *_strides(dout), ptr(dq), *_strides(dq),
                 ptr(dk), *_strides(dk), ptr(dv), *_strides(dv), ptr(ws), size)
        return dq, dk, dv, None, None, None, None


def _dims(d: int, scale: Optional[float]) -> float:
    _need(8 <= d <= MAX_HEAD_DIM and d % 8 == 0, "heads of %d features (a multiple of 8 up to %d)", d, MAX_HEAD_DIM)
    scale = d ** -0.5 if scale is None else float(scale)
    _need(math.isfinite(scale) and scale > 0, "scale %g has to be positive and finite", scale)
    return scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
              offsets_k: Optional[torch.Tensor] = None, causal: bool = True,
              scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of packed histories: q [N, heads, d], k and v [M, kv_heads, d] -> [N, heads, d].

    ``offsets`` [B + 1] int32 on the device, ascending: history b has queries ``offsets[b]`` to ``offsets[b + 1]`` and
    keys by ``offsets_k`` (None: the same).  Query head h reads key head ``h // (heads / kv_heads)``.  ``causal`` lets
    query i of Lq see keys j <= i + Lk - Lq: the last query sees the last key.  ``scale`` defaults to d^-0.5.

    Queries that see no key (an empty history, or Lq > Lk with ``causal``) and tokens outside every history (before
    the first offset, behind the last) give zeros and get zero gradients; offsets beyond the token count are taken as
    the token count.  What a query does not see, infinities and NaN included, does not reach its output.  Gradients
    flow to q, k and v (sums over the group for k and v), in a fixed order: the same inputs give the same bits.
    """
    _storage(q, k, v)
    _need(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and q.shape[2] == k.shape[2],
          "q %s, k %s and v %s", tuple(q.shape), tuple(k.shape), tuple(v.shape))
    _heads(q.shape[1], k.shape[1])
    scale = _dims(q.shape[2], scale)
    _need(max(q.shape[0] * (q.shape[1] // k.shape[1]), k.shape[0]) < (1 << 31) - 1024, "%d and %d tokens", q.shape[0],
          k.shape[0])
    offsets = _index(offsets, "offsets")
    _need(offsets.shape[0] >= 1, "offsets are empty")
    if offsets_k is None:
        _need(q.shape[0] == k.shape[0], "%d queries and %d keys need offsets_k", q.shape[0], k.shape[0])
        offsets_k = offsets
    else:
        offsets_k = _index(offsets_k, "offsets_k", offsets.shape[0])
    _on_device(q, k, v, offsets, offsets_k)
    return PackedAttnFn.apply(q, k, v, offsets, offsets_k, bool(causal), scale)


def cached_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                     scale: Optional[float] = None) -> torch.Tensor:
    """New tokens against the cache: q [B, L, heads, d], caches [B, capacity, kv_heads, d] -> [B, L, heads, d].

    ``lens`` [B] int32 counts the cached rows of each history, the L new ones included: query i sees rows
    j < lens[b] - L + 1 + i, and zeros come back where that is none.  Rows from ``lens[b]`` on are not used, whatever
    they hold.  The caches are read in place (unit feature stride, other strides on 16 bytes).  No autograd."""
    _storage(q, k_cache, v_cache)
    _cache(k_cache, "k_cache")
    _cache(v_cache, "v_cache")
    _need(q.dim() == 4 and k_cache.shape == v_cache.shape and q.shape[0] == k_cache.shape[0]
          and q.shape[3] == k_cache.shape[3], "q %s and caches %s, %s", tuple(q.shape), tuple(k_cache.shape),
          tuple(v_cache.shape))
    B, L, heads, d = q.shape
    cap, hk = k_cache.shape[1:3]
    _heads(heads, hk)
    scale = _dims(d, scale)
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        _need(c.numel() == 0 or _fits(c, 1 << 62), "%s: strides %s cannot be read in place", name, c.stride())
    lens = _index(lens, "lens", B)
    _on_device(q, k_cache, v_cache, lens)
    q = _dense(q.detach())
    out = torch.empty((B, L, heads, d), dtype=q.dtype, device=q.device)
    if B and L:
        size = int(lib().tagan_cached_attn_workspace(B, L, cap, heads, hk, d))
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _run("tagan_cached_attn", q, dtype_code(q), B, L, cap, heads, hk, d, ptr(q), *_strides(q), ptr(k_cache),
             *_strides(k_cache), ptr(v_cache), *_strides(v_cache), ptr(lens), scale, ptr(out), *_strides(out), ptr(ws),
             size)
    return out
