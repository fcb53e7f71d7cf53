"""Softmax attention of training batches and prompts, and attention from a key/value cache held in 8 bits.

CUDA bf16 tensors with heads of up to 128 (a multiple of 8) run the kernels of ``csrc/attention``; other tensors (fp16, fp32, other heads) run the statements
in :mod:`triune_b200.ops.reference`, which hold the [B, H, T, S] scores and weights in fp32 several times over and repeat shared heads:
2048 tokens, 16 heads: 268 MB a sequence each. ``attention_supported`` tells. This is the role of the library call in the reference's ``use_sdpa`` branch
(``triune/model/attention.py:606-653``) and dense attention (``triune/universal.py:200-266``); the 8-bit cache has no counterpart there."""

from __future__ import annotations

from typing import Any, Mapping, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from .. import _ext
from . import _tick, inference_call
from . import reference as ref
from .hybrid import status_word

KV8_BLOCK, KV8_RING = ref.KV8_BLOCK, ref.KV8_RING
KV8_TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
Position = Union[int, torch.Tensor]


def _shapes(q, k, v) -> Tuple[int, int, int, int]:
    """-> B, T, S, D"""
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 4 or len(ks) != 4 or vs != ks:
        raise ValueError(f"attention takes queries [B, T, H, D] and keys and values [B, S, G, D], got {tuple(qs)}, {tuple(ks)}, {tuple(vs)}")
    (B, T, H, D), (Bk, S, G, Dk) = qs, ks
    if B != Bk or D != Dk:
        raise ValueError(f"queries {tuple(qs)} and keys {tuple(ks)} differ in batch or head size")
    if G == 0 or H % G:
        raise ValueError(f"query heads ({H}) must be a multiple of the key/value heads ({G})")
    if not q.dtype == k.dtype == v.dtype or not q.device == k.device == v.device:
        raise ValueError("queries, keys and values must have one type and device")
    return B, T, S, D


def _scale(scale: Optional[float], D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:  # an fp32 number, also times log2(e)
        raise ValueError(f"the scale of the scores must be positive (1e-30 to 1e30), got {scale}")
    return scale


def _whole_numbers(x: torch.Tensor, name: str, batch: int, device, one: bool = False) -> torch.Tensor:
    """``x`` as contiguous int64, one number per sequence (``one``: or one for all)."""
    if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool or x.device != device:
        raise ValueError(f"{name} must be whole numbers on {device}")
    if not (x.numel() == batch or one and x.numel() == 1):
        raise ValueError(f"{name} must have {'one entry or ' if one else ''}an entry per sequence ({batch}), got shape {tuple(x.shape)}")
    return x.reshape(-1).long().contiguous()


def _kernels(x: torch.Tensor) -> bool:
    return _ext.use_kernels(x) and x.dtype == torch.bfloat16 and x.shape[-1] % 8 == 0 and 8 <= x.shape[-1] <= 128


def attention_supported(q: torch.Tensor) -> bool:
    """Whether :func:`attention` runs these queries on the framework's kernels."""
    return q.dim() == 4 and _kernels(q)


class _AttentionFn(torch.autograd.Function):
    """What is traced: a trace records the function. Calls that are not go through the extension's own node of the graph, which
    does the same without Python in the backward pass."""

    @staticmethod
    def forward(ctx, q, k, v, scale, causal, window, lengths, starts, start):
        out, lse, rest = _ext.ext().attention_fwd(q, k, v, scale, causal, window, lengths, starts, start, True, status_word(q.device))
        _tick()
        ctx.save_for_backward(q, k, v, out, rest, lse, lengths, starts)
        ctx.how = (scale, causal, window, start)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, rest, lse, lengths, starts = ctx.saved_tensors
        scale, causal, window, start = ctx.how
        grads = _ext.ext().attention_bwd(q, k, v, out, rest, grad.to(q.dtype), lse, scale, causal, window, lengths, starts, start, status_word(q.device))
        _tick(2)
        return (*grads, None, None, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, window: Optional[int] = None,
              key_lengths: Optional[torch.Tensor] = None, query_start: Optional[Position] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of queries ``q`` [B, T, H, D] over ``k``, ``v`` [B, S, G, D] -> [B, T, H, D]; H is a multiple of G, and
    query head h reads key/value head ``h // (H / G)``. Differentiable (once) in q, k and v; gradients of shared heads are summed.

    Query i of a sequence stands at position ``query_start + i`` (a number, or whole numbers on the device, one or one per sequence;
    by default S - T, so that the last query stands at the last key). It sees key j where j < ``key_lengths`` of the sequence
    (whole numbers [B] on the device, by default S), and, with ``causal``, j <= its position, and, with ``window``, j > its position -
    window. A query that sees no key gives zeros and passes no gradient on. Scores are multiplied by ``scale`` (by default
    D ** -0.5), which must be positive.

    What keys and values past ``key_lengths`` hold does not matter, whatever it is. A value that is an infinity or NaN reaches the
    outputs of the queries that see it and of no others; gradients are not kept apart in this way. On CUDA, weights and their gradients are rounded to bf16 for
    the matrix products, sums and statistics are fp32, and results do not depend on the order in which blocks run. Forward and backward
    can be captured into a CUDA graph; as with any operator, PyTorch ends the capture of a backward pass with an error where a graph of the
    same leaves that was not captured is still alive. Where a bounded wait of a kernel expires, what waited for it is NaN
    (:func:`triune_b200.ops.hybrid.check_status` tells)."""
    B, T, S, D = _shapes(q, k, v)
    scale = _scale(scale, D)
    if window is not None and (int(window) != window or window < 1):
        raise ValueError(f"a window is a number of keys (at least 1), got {window}")
    if window is not None and not causal:
        raise ValueError("a window needs a causal mask")
    lengths = None if key_lengths is None else _whole_numbers(key_lengths, "key_lengths", B, q.device)
    starts, start = None, S - T
    if torch.is_tensor(query_start):
        starts = _whole_numbers(query_start, "query_start", B, q.device, one=True)
        starts = starts.expand(B).contiguous() if starts.numel() != B else starts
    elif query_start is not None:
        start = int(query_start)
    if _kernels(q):
        how = (scale, bool(causal), min(int(window or 0), 1 << 61), lengths, starts, start)
        if inference_call(q, k, v):
            out, _, _ = _ext.ext().attention_fwd(q, k, v, *how, False, status_word(q.device))
            _tick()
            return out
        if torch.jit.is_tracing() or forward_ad._current_level >= 0:  # tangents: refused
            return _AttentionFn.apply(q, k, v, *how)
        _tick(3)  # with its backward pass, which is launched without Python
        return _ext.ext().attention(q, k, v, *how, status_word(q.device))
    return ref.attention(q, k, v, bool(causal), window, lengths, start if starts is None else starts, scale)


# ---------------------------------------------------------------------------------------------------- the cache in 8 bits
def kv8_cache(batch: int, kv_heads: int, capacity: int, head_dim: int, kind: str = "int8", device=None) -> dict:
    """Empty tensors of an 8-bit key/value cache for ``capacity`` tokens per sequence (rounded up to whole blocks of 64):

    ``k8``, ``v8``  codes [B, G, capacity, pitch], int8 or float8_e4m3fn (pitch: 64 or 128, the head size rounded up)
    ``ks``, ``vs``  fp32 [B, G, capacity / 64], one scale per block of 64 tokens and head: largest magnitude / 127 (or / 448)
    ``kt``, ``vt``  bf16 [B, G, 128, pitch], the last 128 tokens as they came: position x is in row x % 128

    A block's codes and scale are written when its last token arrives; until then its tokens are read as they came."""
    if kind not in KV8_TYPES:
        raise ValueError(f"a cache in 8 bits is 'int8' or 'e4m3', got {kind!r}")
    if not 8 <= head_dim <= 128 or head_dim % 8:
        raise ValueError(f"head sizes are multiples of 8 up to 128, got {head_dim}")
    if batch < 0 or kv_heads < 1 or capacity < 0:
        raise ValueError(f"batch {batch}, heads {kv_heads}, capacity {capacity}")
    pitch, room = 64 if head_dim <= 64 else 128, -(-capacity // KV8_BLOCK) * KV8_BLOCK
    new = lambda *shape, dtype: torch.zeros(batch, kv_heads, *shape, dtype=dtype, device=device)  # noqa: E731
    cache = {}
    for n in ("k", "v"):
        cache[n + "8"] = torch.zeros(batch, kv_heads, room, pitch, dtype=torch.uint8, device=device).view(KV8_TYPES[kind])
        cache[n + "s"] = new(room // KV8_BLOCK, dtype=torch.float32)
        cache[n + "t"] = new(KV8_RING, pitch, dtype=torch.bfloat16)
    return cache


def _parts(cache: Mapping[str, torch.Tensor]) -> Tuple[torch.Tensor, ...]:
    return cache["k8"], cache["v8"], cache["ks"], cache["vs"], cache["kt"], cache["vt"]


def _kv8_kernels(cache: Mapping[str, torch.Tensor]) -> bool:
    return _ext.use_kernels(cache["k8"])


def _at(pos: Position, name: str, cache, tokens: int = 0) -> Tuple[int, Optional[torch.Tensor]]:
    """-> (number, None) or (0, int64 tensor). Numbers are checked against the capacity here, positions on the device by the kernels."""
    codes = cache["k8"]
    if torch.is_tensor(pos):
        return 0, _whole_numbers(pos, name, codes.shape[0], codes.device, one=True)
    pos = int(pos)
    if pos + tokens > codes.shape[2]:
        raise ValueError(f"{name} {pos}{f' and {tokens} tokens' if tokens else ''}: past the cache's capacity of {codes.shape[2]}")
    return pos, None


def _new_rows(cache, k, v) -> None:
    codes = cache["k8"]
    cs, ks, vs, device = codes.shape, k.shape, v.shape, codes.device
    if len(ks) != 4 or vs != ks or ks[0] != cs[0] or ks[2] != cs[1] or ks[3] > cs[3] or ks[3] % 8:
        raise ValueError(f"keys and values [B, T, G, D] that fit a cache of codes {tuple(cs)}, got {tuple(ks)} and {tuple(vs)}")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.device != device or v.device != device:
        raise ValueError("keys and values of an 8-bit cache are bfloat16 on the cache's device")


def _no_gradients(*tensors) -> None:
    if not inference_call(*tensors):
        raise RuntimeError("the 8-bit cache serves: no gradients, tangents or traces pass through it (torch.no_grad)")


def kv8_append(cache: Mapping[str, torch.Tensor], k: torch.Tensor, v: torch.Tensor, pos: Position) -> None:
    """Writes ``k``, ``v`` [B, T, G, D] (bf16) into ``cache`` (:func:`kv8_cache`) at positions ``pos`` .. ``pos + T - 1``. ``pos`` is a number, or whole numbers on the device,
    one or one per sequence; the cache must hold all earlier positions. A sequence whose position is negative is idle: nothing
    of it is written. Tokens past the capacity raise where ``pos`` is a number and are not stored where it is on the device.

    What the cache holds does not depend on how the tokens were portioned. Up to 64 tokens can be taken back: go on from an earlier
    position. A block with an infinity or NaN in it reads as NaN throughout once it is full."""
    _no_gradients(k, v)
    _new_rows(cache, k, v)
    host, dev = _at(pos, "position", cache, k.shape[1])
    if _kv8_kernels(cache):
        _ext.ext().kv8_append(*_parts(cache), k, v, host, dev)
        _tick()
    else:
        ref.kv8_append(cache, k, v, host if dev is None else dev)


def kv8_expand(cache: Mapping[str, torch.Tensor], length: Position, head_dim: int, rows: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of the first ``length`` positions in bf16, [B, rows, G, D] each (``rows``: by default the length where it
    is a number, else the capacity); zeros from the sequence's length on.

    The block in which a length lies is read from the last 128 tokens that came: a length is a multiple of 64, or at most 64 less than what was appended.
    For others the rows from their last multiple of 64 on are those of later tokens; the cache does not know what was appended, so this is not checked."""
    host, dev = _at(length, "length", cache)
    room, pitch = cache["k8"].shape[2:]
    rows = (max(0, host) if dev is None else room) if rows is None else int(rows)
    if not 0 <= rows <= room or not 8 <= head_dim <= pitch or head_dim % 8:
        raise ValueError(f"{rows} rows of {head_dim}: the cache has {room} of {pitch}")
    if _kv8_kernels(cache):
        k, v = _ext.ext().kv8_expand(*_parts(cache), rows, head_dim, host, dev)
        _tick()
        return k.transpose(1, 2), v.transpose(1, 2)
    return ref.kv8_expand(cache, host if dev is None else dev, head_dim, rows)


def kv8_attention(q: torch.Tensor, cache: Mapping[str, torch.Tensor], pos: Position, k: Optional[torch.Tensor] = None,
                  v: Optional[torch.Tensor] = None, scale: Optional[float] = None, most: Optional[int] = None,
                  as_given: bool = False) -> torch.Tensor:
    """Attention of ``q`` [B, T, H, D] at positions ``pos`` .. ``pos + T - 1`` over the cached keys up to each query's own ->
    [B, T, H, D]. With ``k`` and ``v`` [B, T, G, D], the queries' tokens are appended first (:func:`kv8_append`, also on
    ``pos``); without, the cache must hold them already, and at most 64 behind them (or ``pos + T`` is a multiple of 64; :func:`kv8_expand`). Keys and values are those that the cache holds once these tokens are in it: a block that the call
    fills is read as codes by all its queries, also by those before the block's last token. Their outputs depend, by what codes round
    off, on the rest of the block, and so on later tokens and on how tokens are portioned. A call is strictly causal where no token but its
    first ends a block (position % 64 == 63), as single tokens are; and with ``as_given``, by which queries see the call's own ``k`` and ``v`` as
    they are given, and earlier blocks that were full before as codes. ``most`` is a bound on the tokens that any sequence holds after this call, by
    default the capacity (or ``pos + T`` where ``pos`` is a number), for which the work is laid out; tokens past it are not promised to be seen.

    Idle sequences (negative positions) give zeros; a query past the capacity (positions on the device only) gives NaN."""
    codes = cache["k8"]
    cs, qs = codes.shape, q.shape
    if len(qs) != 4 or qs[0] != cs[0] or qs[2] % cs[1] or qs[3] > cs[3] or qs[3] % 8 or qs[3] < 8:
        raise ValueError(f"queries [B, T, H, D] that fit a cache of codes {tuple(cs)}, got {tuple(qs)}")
    if q.dtype != torch.bfloat16 or q.device != codes.device:
        raise ValueError("queries of an 8-bit cache are bfloat16 on the cache's device")
    if (k is None) != (v is None):
        raise ValueError("new keys come with new values")
    if as_given and k is None:
        raise ValueError("as_given is about new keys and values, and there are none")
    _no_gradients(q, k, v)
    scale, T = _scale(scale, qs[3]), qs[1]
    if k is not None:
        _new_rows(cache, k, v)
        ks = k.shape
        if ks[1] != T or ks[3] != qs[3]:
            raise ValueError(f"new keys {tuple(ks)} for queries {tuple(qs)}")
    host, dev = _at(pos, "position", cache, T)
    room = cs[2] if dev is not None else max(0, host + T)
    most = room if most is None else min(int(most), room)
    if not _kv8_kernels(cache):
        at = host if dev is None else dev
        if as_given:
            out = ref.kv8_attention(q, cache, at, scale, k, v)
            ref.kv8_append(cache, k, v, at)
            return out
        if k is not None:
            ref.kv8_append(cache, k, v, at)
        return ref.kv8_attention(q, cache, at, scale)
    out = _ext.ext().kv8_attention(*_parts(cache), q, k, v, host, dev, scale, most, as_given, status_word(q.device))
    _tick(2 + (k is not None))
    return out


def kv8_kind(cache: Mapping[str, Any]) -> str:
    """``"int8"`` or ``"e4m3"``."""
    return next(n for n, t in KV8_TYPES.items() if cache["k8"].dtype == t)
