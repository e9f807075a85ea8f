"""Attention over packed histories with rotary positions (csrc/packed_attn.hip, csrc/rotary.hip).

Beside the rectangular temporal attention of ``kernels.TemporalAttnFn`` ([rows, T], equal heads, T <= 128 on the matrix
cores): histories of different lengths lie behind one another in one token axis, several query heads may share a key
head, and positions enter as turns of the query and key features.

* ``rotary_frequencies`` / ``rotary``        turn q and k by their positions (differentiable)
* ``attention``                              softmax attention inside each packed history (differentiable)
* ``rotary_append`` / ``cached_attention``   serving: write new tokens behind each cached history, attend to it

fp32 or bf16 storage, fp32 statistics and sums.  In bf16 each probability, and each gradient of a score, is rounded to bf16
as an operand of its second product: errors are about 1.4 times those of one rounding of the result.  Over few keys such
roundings do not average out: in batches of up to 64 keys to an average history, those of up to 128 keys keep what the
rounding took away as a second operand and have the error of one rounding.

Everything runs on the current HIP stream of the tensors' device, allocates from PyTorch's caching allocator only, never
waits for the device and can be captured in a HIP graph; offsets and lengths stay on the device.  Wrong arguments raise
TypeError / ValueError, and what only the C entries know of RuntimeError, before anything is launched.

A captured backward: capture forward and backward together (``graph_step.GraphedStep``) and let no eager graph of the
same leaves live across the capture: such a graph keeps the leaves' gradient accumulation on the eager stream, which a
capture must not touch.
"""
import math
from typing import Optional, Tuple

import torch

from ._lib import check, dtype_code, lib, require_hip

MAX_HEAD_DIM = 128        # attention: multiples of 8 up to this
MAX_ROTARY_DIM = 256
MAX_GROUP = 512           # query heads to a key head
MAX_TOKEN_STRIDE = 1 << 21
_POS_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


# ----------------------------------------------------------------------------- arguments
# A serving step's time is the host's: the checks below build no message and no list unless something is wrong.
def _refuse(text: str, *args):
    raise ValueError(text % args)


def _shapes(*tensors) -> str:
    return ", ".join("None" if t is None else str(tuple(t.shape)) for t in tensors)


def _on_device(first: torch.Tensor, *rest) -> None:
    index = first.get_device()
    if index < 0:
        require_hip(first)
    for t in rest:
        if t is not None and t.get_device() != index:
            require_hip(t)
            _refuse("tensors on %s and %s", first.device, t.device)


def _storage(first: torch.Tensor, *rest) -> None:
    dtype = first.dtype
    if dtype is not torch.float32 and dtype is not torch.bfloat16:
        raise TypeError("float32 or bfloat16 is wanted, got %s" % dtype)
    for t in rest:
        if t is not None and t.dtype is not dtype:
            raise TypeError("tensors of %s and %s" % (dtype, t.dtype))


def _index(t: torch.Tensor, name: str, size: Optional[int] = None) -> torch.Tensor:
    if t.dtype is not torch.int32:
        raise TypeError("%s has to be int32, got %s" % (name, t.dtype))
    if t.dim() != 1 or (size is not None and t.shape[0] != size):
        _refuse("%s has shape %s", name, _shapes(t))
    return t.contiguous()


def _heads(heads: int, kv_heads: int) -> None:
    if kv_heads < 1 or heads < kv_heads or heads % kv_heads or heads // kv_heads > MAX_GROUP:
        _refuse("%d query heads over %d key heads", heads, kv_heads)


def _fits(t: torch.Tensor) -> bool:
    """Whether the attention kernels can read t in place: 16-byte runs, whole rows, a tile within 32-bit offsets (an axis
    of one step is never stepped over)."""
    if t.stride(-1) != 1 or t.data_ptr() % 16:
        return False
    es, d, heads, tokens = t.element_size(), t.shape[-1], t.shape[-2], t.shape[-3]
    return (all(n <= 1 or (s >= 0 and s * es % 16 == 0) for n, s in zip(t.shape[:-1], t.stride()))
            and (tokens <= 1 or d <= t.stride(-3) <= MAX_TOKEN_STRIDE)
            and (heads <= 1 or t.stride(-2) * heads * es < 1 << 30))


def _dense(t: torch.Tensor) -> torch.Tensor:
    if t.is_contiguous() and t.data_ptr() % 16 == 0 and t.shape[-1] * t.shape[-2] <= MAX_TOKEN_STRIDE:
        return t
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


def _run(name: str, t: torch.Tensor, *args) -> None:
    """The C entry on the device and current stream of t."""
    index = t.device.index
    if index == torch.cuda.current_device():
        rc = getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


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
    if dim < 2 or dim % 2:
        _refuse("%d features cannot be turned in pairs", dim)
    if not (base > 0 and math.isfinite(base) and factor >= 1 and math.isfinite(factor)):
        _refuse("base %g, factor %g", base, factor)
    if scaling == "base":
        if dim == 2:
            _refuse("the base cannot be raised for 2 features")
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if not (fast > slow and original_len >= 1):
            _refuse("turns %g to %g over %d positions", slow, fast, original_len)
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
    if inv_freq.dim() != 1 or not 2 <= 2 * inv_freq.shape[0] <= dim <= MAX_ROTARY_DIM:
        _refuse("%s frequencies for heads of %d features (up to %d)", _shapes(inv_freq), dim, MAX_ROTARY_DIM)
    return inv_freq.to(torch.float64).contiguous()


def _turn(q, k, positions, inv_freq, interleaved, scale, inverse):
    n, heads, d = q.shape
    q = q if q.stride(-1) == 1 else q.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko, hk = None, 0
    if k is not None:
        k = k if k.stride(-1) == 1 else k.contiguous()
        ko, hk = torch.empty_like(k, memory_format=torch.contiguous_format), k.shape[1]
    if n:
        kin = (k.data_ptr(), *k.stride()[:2]) if hk else (None, 0, 0)
        kout = (ko.data_ptr(), hk * d, d) if hk else (None, 0, 0)
        _run("tagan_rotary", q, dtype_code(q), n, heads, hk, d, 2 * inv_freq.shape[0], q.data_ptr(), *q.stride()[:2],
             *kin, positions.data_ptr(), _POS_TYPES[positions.dtype], inv_freq.data_ptr(), scale, interleaved, inverse,
             qo.data_ptr(), heads * d, d, *kout)
    return qo, ko


class RotaryFn(torch.autograd.Function):
    """(q, k) turned by their positions, or back; the gradient is the other turn, of any order."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved: bool, scale: float, inverse: int):
        ctx.save_for_backward(positions, inv_freq)
        ctx.cfg = (interleaved, scale, 1 - inverse)
        ctx.set_materialize_grads(False)
        return _turn(q, k, positions, inv_freq, interleaved, scale, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 7
        turn = RotaryFn.apply if torch.is_grad_enabled() else _turn
        if dq is None:
            dk, _ = turn(dk, None, positions, inv_freq, *ctx.cfg)
        else:
            dq, dk = turn(dq, dk, positions, inv_freq, *ctx.cfg)
        return dq, dk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
           interleaved: bool = False, scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [N, heads, d] and k [N, kv_heads, d] (or None) turned by ``positions`` [N] (int32, int64, float32 or float64:
    indices or event times) times ``inv_freq`` [r / 2]: the first r features of each head in pairs (i, i + r/2), or
    (2i, 2i + 1) with ``interleaved``, times ``scale``; the features behind them are copied.  Angles are formed in
    fp64.  Gradients flow to q and k (not to positions)."""
    _storage(q, k)
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        _refuse("q and k: %s", _shapes(q, k))
    if q.shape[1] < 1 or (k is not None and k.shape[1] < 1):
        _refuse("no heads: %s", _shapes(q, k))
    if positions.dtype not in _POS_TYPES:
        raise TypeError("positions of %s" % positions.dtype)
    if positions.dim() != 1 or positions.shape[0] != q.shape[0]:
        _refuse("%s positions for %d tokens", _shapes(positions), q.shape[0])
    if not math.isfinite(scale):
        _refuse("scale %g", scale)
    inv_freq = _frequencies(inv_freq, q.shape[2])
    _on_device(q, k, positions, inv_freq)
    return RotaryFn.apply(q, k, positions.contiguous(), inv_freq, bool(interleaved), float(scale), 0)


def _cache(t: torch.Tensor, name: str) -> None:
    if t.dim() != 4:
        _refuse("%s %s: [batch, capacity, heads, features] is wanted", name, _shapes(t))
    if t.requires_grad:
        _refuse("%s is written and read in place: it cannot require a gradient", name)
    if t.stride(-1) != 1:
        _refuse("%s needs unit feature stride", name)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  lens: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
                  scale: float = 1.0) -> torch.Tensor:
    """New tokens q [B, L, heads, d], k and v [B, L, kv_heads, d] at positions ``lens[b] + i``: writes turned k and v
    to rows ``lens[b] + i`` of the caches [B, capacity, kv_heads, d] in place and returns the turned q, in one launch.

    ``lens`` [B] int32 counts the rows already there and is not advanced; rows that would lie outside the capacity are
    not written.  No autograd; a backward that kept rows of the caches raises after it, as after any write in place."""
    _storage(q, k, v, k_cache, v_cache)
    _cache(k_cache, "k_cache")
    _cache(v_cache, "v_cache")
    if (q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2]
            or q.shape[3] != k.shape[3]):
        _refuse("q, k and v: %s", _shapes(q, k, v))
    B, L, heads, d = q.shape
    hk = k.shape[2]
    _heads(heads, hk)
    if k_cache.shape != v_cache.shape or k_cache.shape[0] != B or k_cache.shape[2:] != k.shape[2:]:
        _refuse("caches and k: %s", _shapes(k_cache, v_cache, k))
    for c in (k_cache, v_cache):
        if 0 in c.stride() and any(n > 1 and s <= 0 for n, s in zip(c.shape, c.stride())):
            _refuse("a cache with shared rows cannot be written")
    if k_cache.data_ptr() == v_cache.data_ptr() and k_cache.numel():
        _refuse("one tensor cannot be both caches: k and v would be written to the same rows")
    lens = _index(lens, "lens", B)
    if not math.isfinite(scale):
        _refuse("scale %g", scale)
    inv_freq = _frequencies(inv_freq, d)
    _on_device(q, k, v, k_cache, v_cache, lens, inv_freq)
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q.detach(), k.detach(), v.detach()))
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B and L:
        _run("tagan_rotary_append", q, dtype_code(q), B, L, heads, hk, d, 2 * inv_freq.shape[0], q.data_ptr(),
             *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], lens.data_ptr(),
             inv_freq.data_ptr(), scale, 1 if interleaved else 0, out.data_ptr(), L * heads * d, heads * d, d,
             k_cache.data_ptr(), *k_cache.stride()[:3], v_cache.data_ptr(), *v_cache.stride()[:3], k_cache.shape[1])
        torch.autograd.graph.increment_version((k_cache, v_cache))   # a backward that kept them has to notice
    return out


# ----------------------------------------------------------------------------- packed attention
class PackedAttnFn(torch.autograd.Function):
    """softmax(scale q kᵀ) v inside each packed sequence; saves the output (bf16: with its rounding, 2 bytes more to an
    element) and the rows' log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, offsets, offsets_k, causal: bool, scale: float):
        q, k, v = _dense(q), _dense(k), _dense(v)
        n, heads, d = q.shape
        nk, hk, _ = k.shape
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        needs = any(ctx.needs_input_grad[:3])
        lse = torch.empty((n, heads), dtype=torch.float32, device=q.device) if needs else None
        rest = torch.empty_like(out) if needs and q.dtype is torch.bfloat16 else None
        if n:
            size = lib().tagan_packed_attn_fwd_workspace(offsets.shape[0] - 1, n, nk, heads, hk, d)
            ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
            _run("tagan_packed_attn_fwd", q, dtype_code(q), offsets.shape[0] - 1, n, nk, heads, hk, d, q.data_ptr(),
                 *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], offsets.data_ptr(),
                 offsets_k.data_ptr(), causal, scale, out.data_ptr(), heads * d, d,
                 lse.data_ptr() if needs else None, None if rest is None else rest.data_ptr(),
                 ws.data_ptr() if size else None, size)
        if needs:
            ctx.save_for_backward(q, k, v, out, lse, rest, offsets, offsets_k)
            ctx.cfg = (causal, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():      # create_graph: the gradients would pass as constants
            raise RuntimeError("packed.attention has no second derivative")
        q, k, v, out, lse, rest, offsets, offsets_k = ctx.saved_tensors
        causal, scale = ctx.cfg
        dout = _dense(dout)
        n, heads, d = q.shape
        nk, hk, _ = k.shape
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        if n or nk:
            size = lib().tagan_packed_attn_bwd_workspace(n, heads)
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device=q.device)
            _run("tagan_packed_attn_bwd", q, dtype_code(q), offsets.shape[0] - 1, n, nk, heads, hk, d, q.data_ptr(),
                 *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], offsets.data_ptr(),
                 offsets_k.data_ptr(), causal, scale, out.data_ptr(), heads * d, d, lse.data_ptr(),
                 None if rest is None else rest.data_ptr(), dout.data_ptr(), *dout.stride()[:2], dq.data_ptr(), heads * d, d, dk.data_ptr(), hk * d, d, dv.data_ptr(), hk * d, d,
                 ws.data_ptr(), size)
        return dq, dk, dv, None, None, None, None


def _dims(d: int, scale: Optional[float]) -> float:
    if d < 8 or d > MAX_HEAD_DIM or d % 8:
        _refuse("heads of %d features (a multiple of 8 up to %d)", d, MAX_HEAD_DIM)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 127:
        _refuse("scale %g has to lie in 2^-126 to 2^127", scale)
    return scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
              offsets_k: Optional[torch.Tensor] = None, causal: bool = True,
              scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of packed histories: q [N, heads, d], k and v [M, kv_heads, d] -> [N, heads, d].

    ``offsets`` [B + 1] int32 on the device, ascending: history b has queries ``offsets[b]`` to ``offsets[b + 1]`` and
    keys by ``offsets_k`` (None: the same).  Query head h reads key head ``h // (heads / kv_heads)``.  ``causal`` lets
    query i of Lq see keys j <= i + Lk - Lq: the last query sees the last key.  ``scale`` defaults to d^-0.5;
    scale log2(e) q·k has to stay within fp32's range.

    Queries that see no key (an empty history, or Lq > Lk with ``causal``) and tokens outside every history (before
    the first offset, behind the last) give zeros and get zero gradients; offsets beyond the token count are taken as
    the token count.  What a query does not see, infinities and NaN included, does not reach its output; an infinity or
    NaN in a value that it sees makes that feature of its output infinite or NaN, however small the weight.  Gradients
    flow to q, k and v (sums over the group for k and v), in a fixed order: the same inputs give the same bits.
    An infinity or NaN in q, k, v or the output's gradient may reach any gradient of its history, and of no other.  There
    is no second derivative (``create_graph`` raises).
    """
    _storage(q, k, v)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        _refuse("q, k and v: %s", _shapes(q, k, v))
    n, heads, d = q.shape
    _heads(heads, k.shape[1])
    scale = _dims(d, scale)
    if max(n * (heads // k.shape[1]), k.shape[0]) >= (1 << 31) - 1024:
        _refuse("%d and %d tokens", n, k.shape[0])
    offsets = _index(offsets, "offsets")
    if offsets.shape[0] < 1:
        _refuse("offsets are empty")
    if offsets_k is None:
        if n != k.shape[0]:
            _refuse("%d queries and %d keys need offsets_k", n, k.shape[0])
        offsets_k = offsets
    else:
        offsets_k = _index(offsets_k, "offsets_k", offsets.shape[0])
    _on_device(q, k, v, offsets, offsets_k)
    return PackedAttnFn.apply(q, k, v, offsets, offsets_k, bool(causal), scale)


def cached_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                     scale: Optional[float] = None) -> torch.Tensor:
    """New tokens against the cache: q [B, L, heads, d], caches [B, capacity, kv_heads, d] -> [B, L, heads, d].

    ``lens`` [B] int32 counts the tokens of each history, the L new ones included: query i sees the rows
    j < lens[b] - L + 1 + i of the cache, and zeros come back where that is none.  A length past the capacity leaves
    that window where it is (the rows that ``rotary_append`` had no room for are missing from it).  Rows from ``lens[b]``
    on are not used, whatever they hold.  The caches are read in place: unit feature stride, other strides and the start on 16 bytes, token strides
    up to 2^21 elements, fewer than 2^31 - 1024 rows (RuntimeError otherwise).  No autograd."""
    _storage(q, k_cache, v_cache)
    _cache(k_cache, "k_cache")
    _cache(v_cache, "v_cache")
    if q.dim() != 4 or k_cache.shape != v_cache.shape or q.shape[0] != k_cache.shape[0] or q.shape[3] != k_cache.shape[3]:
        _refuse("q and caches: %s", _shapes(q, k_cache, v_cache))
    B, L, heads, d = q.shape
    cap, hk = k_cache.shape[1:3]
    _heads(heads, hk)
    scale = _dims(d, scale)
    lens = _index(lens, "lens", B)
    _on_device(q, k_cache, v_cache, lens)
    q = _dense(q.detach())
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B and L:
        size = lib().tagan_cached_attn_workspace(B, L, cap, heads, hk, d)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _run("tagan_cached_attn", q, dtype_code(q), B, L, cap, heads, hk, d, q.data_ptr(), *q.stride()[:3],
             k_cache.data_ptr(), *k_cache.stride()[:3], v_cache.data_ptr(), *v_cache.stride()[:3], lens.data_ptr(), scale,
             out.data_ptr(), L * heads * d, heads * d, d, ws.data_ptr() if size else None, size)
    return out
