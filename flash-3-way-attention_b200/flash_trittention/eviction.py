"""A three-way cache that stays short: the attention weight that each cached token has got, and eviction of the lightest.

A new token's triple dot product costs the square of its context, so a context that is halved costs a quarter.  After a layer's step::

    o, lse = tdp_decode(q, cache, table, context, softmax_scale, return_lse=True)
    tdp_weigh(weights, q, lse, cache, table, context, softmax_scale)               # weights: [B, N, length] fp32, zeros at first
    o, m = dps_decode(q, cache, table, context, softmax_scale)                     # the dot-product-sum form (after dps_append)
    dps_weigh(weights, q, k2, m, cache, table, context, softmax_scale, k_diff)

and once a sequence has become too long::

    context, kept = cache_evict(weights, cache, table, context, keep, first=4, recent=256)

Each head keeps tokens of its own.  They become tokens ``0 .. keep - 1`` of the cache: windows count distances among those that are left, and where rows
were rotated by their positions before they were written, the positions of later tokens go on from the ones that they had, not from the rows' new numbers.  A prompt is weighed by its
last tokens: a call for ``n`` of them, with the ``context`` before them.

The reference has no counterpart: it computes whole sequences.
"""
import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native
from .cache import TrittentionCache, _UNLIMITED, _cache, _check_new, _describe, _need_lse

__all__ = ["tdp_weigh", "dps_weigh", "cache_evict"]


def _weights(cache, table, weights, out, decay=1.0):
    """The library's description of weights ``[B, N, length]`` and where the new ones go."""
    out = weights if out is None else out
    lead = (table.shape[0], cache.codes.shape[2])
    for name, t in (("weights", weights), ("the new weights", out)):
        if t.dim() != 3 or t.shape[:2] != lead or t.dtype != torch.float32 or t.device != cache.codes.device or t.shape[2] < 1:
            raise ValueError(f"{name} must be float32 [{lead[0]}, {lead[1]}, tokens] on {cache.codes.device}, got {t.dtype} {list(t.shape)} on {t.device}")
        if t.shape[2] > 1 and t.stride(2) != 1:
            raise ValueError(f"{name} must have their tokens next to one another, got strides {t.stride()}")
        if t.requires_grad:
            raise ValueError(f"{name} are sums that calls add to: no gradient flows through them")
    room = 1
    for size, step in sorted(((n, st) for n, st in zip(out.shape, out.stride()) if n > 1), key=lambda x: x[1]):
        if step < room:
            raise ValueError(f"the new weights have places that are several tokens' (strides {out.stride()} of shape {list(out.shape)})")
        room = step * size
    if out.data_ptr() == weights.data_ptr() and out.stride() != weights.stride():
        raise ValueError("the new weights start where the old ones do, but are laid out in another way")
    if not (math.isfinite(decay) and decay >= 0):
        raise ValueError(f"decay must be a finite number >= 0, got {decay}")
    stride = lambda t: [st if size > 1 else 0 for st, size in zip(t.stride()[:2], t.shape)]  # noqa: E731
    return _native.Weights(weights.data_ptr(), out.data_ptr(), *stride(weights), *stride(out), weights.shape[2], out.shape[2], decay)


def _sums(name, t, q):
    if t.shape != q.shape[:3] or t.dtype != torch.float32 or t.device != q.device:
        raise ValueError(f"{name} must be float32 {list(q.shape[:3])} on {q.device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.detach().contiguous()


def _same_places(table, other):
    """Whether two tables of as many sequences are one as far as both reach."""
    return table.data_ptr() == other.data_ptr() and all(s == t for n, m, s, t in zip(table.shape, other.shape, table.stride(), other.stride()) if min(n, m) > 1)


def tdp_weigh(weights: Tensor, q: Tensor, lse: Tensor, cache: TrittentionCache, table: Tensor, context: Tensor, softmax_scale: float = 1 / 8,
              k1_window: Optional[int] = None, k2_window: Optional[int] = None, kk_left: Optional[int] = None, kk_right: Optional[int] = None,
              counts: Optional[Tensor] = None, decay: float = 1.0, out: Optional[Tensor] = None) -> None:
    """Adds the attention weight that cached tokens get from new ones in the triple dot product, as ``j`` and as ``k``, to ``weights``.

    ``weights[b, n, x]`` (float32, ``[B, N, length]``) of token ``x`` of sequence ``b`` becomes ``decay * weights[b, n, x]`` plus, for each new token ``i``,
    ``sum_k P_i[x, k] + sum_j P_i[j, x]`` with ``P_i[j, k] = exp(S_i[j, k] - lse_i)``: 2 in all.  ``lse`` is what ``tdp_decode(..., return_lse=True)`` returned
    for the same arguments; a token whose ``lse`` is ``-inf`` adds nothing.  Of the new tokens' own weights what was there before does not count.  Weights of tokens past ``context[b] + counts[b]`` and of free
    slots stay; a token that ``weights`` has no place for is reported by the next call or ``check_status()``.

    ``out``: the new weights go there, and ``weights`` stays (drafts that may be rejected, say); of its memory it is ``weights`` itself or shares none with it.  Drafts are weighed once they are accepted, as a chain.
    Elements of ``q * K2`` have 22 significant bits (above 2^-30 of the largest possible), everything else is fp32; a call repeats itself bit for bit."""
    softmax_scale, decay = float(softmax_scale), float(decay)
    if torch.compiler.is_compiling():
        from . import ops

        _cache(cache)
        return ops.tdp_weigh(weights if out is None else out, None if out is None else weights, q, lse, cache.codes, cache.exponents, table, context, softmax_scale,
                             k1_window, k2_window, kk_left, kk_right, counts, decay)
    done = _native.host_weigh(*_cache(cache), table, context, counts, None, weights, out, decay, softmax_scale, q, lse, k1_window, k2_window, kk_left, kk_right)
    if done is not None:
        _native.host_result(done, "tritt_tdp_weigh")
        return
    q, = _check_new(cache, table, (q,))
    c, keep = _describe(cache, table, context, q.shape[2], counts, None)
    w, lse = _weights(cache, table, weights, out, decay), _sums("lse", lse, q)
    windows = [_UNLIMITED if v is None else min(int(v), _UNLIMITED) for v in (k1_window, k2_window, kk_left, kk_right)]
    if min(windows) < 0:
        raise ValueError(f"window arguments must be >= 0, got {(k1_window, k2_window, kk_left, kk_right)}")
    _native.tdp_weigh(c, w, q, lse, softmax_scale, *windows)


def dps_weigh(weights: Tensor, q: Tensor, k2: Tensor, m: Tensor, cache: TrittentionCache, table: Tensor, context: Tensor, softmax_scale: float = 1 / 8,
              k_diff: int = 1024, counts: Optional[Tensor] = None, decay: float = 1.0, out: Optional[Tensor] = None) -> None:
    """The same in the dot-product sum, with its two soft-maxes: new token ``i`` adds ``exp(softmax_scale * q_i.K2[x] + lse[x] - m_i)`` for its query, and for its inner attention
    ``exp(softmax_scale * k2_i.K1[x] - lse[i])`` to the tokens ``x`` that ``dps_append`` attended to (1 in all for each).  ``k2`` are the rows that ``dps_append`` was given, ``m`` is what
    ``dps_decode`` returned."""
    softmax_scale, decay = float(softmax_scale), float(decay)
    _need_lse(_cache(cache))
    if torch.compiler.is_compiling():
        from . import ops

        return ops.dps_weigh(weights if out is None else out, None if out is None else weights, q, k2, m, *cache, table, context, softmax_scale, k_diff, counts, decay)
    done = _native.host_weigh(*cache, table, context, counts, None, weights, out, decay, softmax_scale, q, m, k2, k_diff)
    if done is not None:
        _native.host_result(done, "tritt_dps_weigh")
        return
    q, k2 = _check_new(cache, table, (q, k2))
    c, keep = _describe(cache, table, context, q.shape[2], counts, None)
    w, m = _weights(cache, table, weights, out, decay), _sums("m", m, q)
    if k_diff < 0:
        raise ValueError(f"k_diff must be >= 0, got {k_diff}")
    _native.dps_weigh(c, w, q, k2, m, softmax_scale, min(int(k_diff), _UNLIMITED))


def cache_evict(weights: Tensor, cache: TrittentionCache, table: Tensor, context: Tensor, keep: int, first: int = 0, recent: int = 0,
                table_out: Optional[Tensor] = None, weights_out: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Keeps ``keep`` tokens of each sequence and head: its ``first`` first ones, its ``recent`` last ones, and of the others those with the largest ``weights`` (of equal ones the
    lower numbers; NaN counts as the largest).  Returns ``(context, kept)``: the tokens that are left, ``[B]`` int32, and their old numbers in order, ``[B, N, keep]`` int32, ``-1``
    behind the last.  A sequence that has no more than ``keep`` tokens keeps them all, a free slot of the batch stays one.

    The kept rows, exponents and log-sum-exps become tokens ``0, 1, 2, ...``, and so do their weights; the pages behind them are free (what they hold is left as it is).  A page that several sequences
    share must not be written: with ``table_out`` (int32 ``[B, pages]``, of pages that the call does not read, or ``table`` itself: in place) the rows go there and the old ones stay, and with ``weights_out`` (float32 ``[B, N, tokens]``, of memory that ``weights`` has no part of)
    the weights."""
    keep, first, recent = int(keep), int(first), int(recent)
    if keep < 1 or first < 0 or recent < 0 or first + recent > keep:
        raise ValueError(f"keep must be at least 1 and first + recent, each at least 0, at most keep: got {keep}, {first} and {recent}")
    if keep > _UNLIMITED:
        raise ValueError(f"keep must be at most {_UNLIMITED}, got {keep}")
    if torch.compiler.is_compiling():
        from . import ops

        return ops.cache_evict(*_cache(cache), weights if weights_out is None else weights_out, None if weights_out is None else weights, table, context, keep, first, recent,
                               table_out)
    out = _native.host_evict(*_cache(cache), table, context, None, None, weights, weights_out, keep, first, recent, table_out)
    if out is not None:
        return _native.host_result(out, "tritt_cache_evict")
    c, alive = _describe(cache, table, context, 1, None, None)
    dev, page = cache.codes.device, cache.codes.shape[3]
    w = _weights(cache, table, weights, weights_out)
    if w.after_length < keep:
        raise ValueError(f"weights have room for {w.after_length} tokens, {keep} are kept")
    if table_out is not None:
        if table_out.shape[:1] != table.shape[:1] or table_out.dim() != 2 or table_out.dtype != torch.int32 or table_out.device != dev or table_out.shape[1] * page < keep:
            raise ValueError(f"table_out must be int32 [{table.shape[0]}, pages for {keep} tokens] on {dev}, got {table_out.dtype} {list(table_out.shape)} on {table_out.device}")
        # (decided before either is laid out for the library, which knows a call in place by the pointer)
        table_out = None if _same_places(table, table_out) else table_out if table_out.stride(1) == 1 else table_out.contiguous()
    context_out = torch.empty(c.B, dtype=torch.int32, device=dev)
    kept = torch.empty(c.B, c.N, keep, dtype=torch.int32, device=dev)
    _native.cache_evict(c, w, table_out, keep, first, recent, context_out, kept)
    return context_out, kept
