"""Serving three-way attention: a paged cache of quantised rows, and attention of one or a few new tokens over it.

A layer's step with the triple dot product writes the new tokens' rows and attends::

    cache_write(cache, table, context, k1, k2, v1, v2)
    o = tdp_decode(q, cache, table, context, softmax_scale, k1_window, k2_window, kk_left, kk_right)

and with the dot-product sum, whose score separates into two chained soft-maxes, attends once for the row that it writes::

    dps_append(cache, table, context, k1, k2, v1, v2, softmax_scale, k_diff)
    o, m = dps_decode(q, cache, table, context, softmax_scale)

Each call is about ``n`` new tokens of ``B`` sequences (tensors ``[B, N, n, D]``): one, a chunk of a prompt, or the drafted tokens of
speculative decoding.  ``context`` (``[B]`` int32) holds how many tokens of each sequence come before them; new token ``i`` is number
``context[b] + i``, for ``i < counts[b]`` where the batch is padded (``counts``, ``[B]`` int32), and lives in row ``number % page_size`` of page
``table[b, number // page_size]`` (``table``: ``[B, pages of a sequence]`` int32).  A sequence with ``context[b] < 0`` is a free slot of the batch:
nothing of it is read or written.

``ancestors`` (``[B, n]`` int64, see ``tree_ancestors``) makes the new tokens a tree: token ``i`` attends to the context, to the earlier new
tokens ``m`` whose bit is set in ``ancestors[b, i]``, and to itself; windows count distances along these.  Without it the new tokens are a chain.  The drafts that are accepted are written again, as a chain.

A place that the table or the cache does not have, and a kernel that gave up, are reported by the next call or ``check_status()``.  The
calls enqueue work on the current stream, and can be captured; which tokens there are is read on the device.

The reference has no counterpart: it computes whole sequences.
"""
from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _native
from ._derivatives import Undifferentiable, forward_mode
from .norm_rotary import HEAD_DIMS

__all__ = ["TrittentionCache", "new_cache", "cache_write", "cache_read", "tree_ancestors", "tdp_decode", "dps_append", "dps_decode"]

MAX_ANCESTORS = 64
_UNLIMITED = 1 << 30


class TrittentionCache(NamedTuple):
    """``codes`` ``[pages, 4, N, page_size, D]`` (float16, float8_e4m3fn or int8), ``exponents`` ``[pages, 4, N, page_size]`` (uint8) and, of
    the dot-product sum, ``lse`` ``[pages, N, page_size]`` (float32).  The parts are K1, K2, SiLU(V1), and V2 or W.

    An element is ``code * 2 ** (exponent - 127)``, one exponent for a row: the least with which the row's largest element fits (448 for
    8-bit floats, 127 for int8, below 2^15 for float16: of 16-bit tensors that keeps all bits of all but the smallest elements).  An
    element that is infinite or NaN makes its row read as NaN (exponent 255), and what attends to it NaN."""

    codes: Tensor
    exponents: Tensor
    lse: Optional[Tensor] = None


def new_cache(pages: int, page_size: int, heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda",
              dps: bool = False) -> TrittentionCache:
    """An empty cache of ``pages`` pages of ``page_size`` tokens (a power of two from 16 on); ``dps``: for the dot-product-sum form."""
    if dtype not in _native.CODES:
        raise ValueError(f"a cache is held in float16, float8_e4m3fn or int8, not {dtype}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of 2 from 16 on, got {page_size}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    shape = (pages, 4, heads, page_size)
    return TrittentionCache(torch.zeros(*shape, head_dim, dtype=dtype, device=device), torch.zeros(shape, dtype=torch.uint8, device=device),
                            torch.zeros(pages, heads, page_size, dtype=torch.float32, device=device) if dps else None)


def tree_ancestors(parents: Sequence[int], device=None) -> Tensor:
    """``[n]`` int64 words for drafted tokens whose parents are ``parents`` (``-1``: the last token of the context; a parent comes before its
    children): bit ``m`` of word ``i`` is set if token ``m`` is token ``i`` or an ancestor of it."""
    if not 0 < len(parents) <= MAX_ANCESTORS:
        raise ValueError(f"expected 1 to {MAX_ANCESTORS} tokens, got {len(parents)}")
    words = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"the parent of token {i} must be -1 or an earlier token, got {p}")
        words.append((words[p] if p >= 0 else 0) | 1 << i)
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device=device)


def _int_vector(name, t, shape, dtype, device):
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} of shape {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.contiguous()


def _describe(cache, table, context, n, counts, ancestors):
    """The library's description of a call, and the tensors that it points to."""
    codes, exponents, lse = cache
    if codes.dim() != 5 or codes.shape[1] != 4 or codes.dtype not in _native.CODES:
        raise ValueError(f"codes must be [pages, 4, heads, page_size, head_dim] of float16, float8_e4m3fn or int8, got {codes.dtype} "
                         f"{list(codes.shape)}")
    if not codes.is_cuda:
        raise RuntimeError("the cache must be on a CUDA device (there is no CPU path)")
    pages, _, N, page_size, D = codes.shape
    dev = codes.device
    for name, t, shape, dtype in (("exponents", exponents, (pages, 4, N, page_size), torch.uint8), ("lse", lse, (pages, N, page_size), torch.float32)):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != dev):
            raise ValueError(f"{name} must be {dtype} of shape {list(shape)} on {dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    for name, t in (("codes", codes), ("exponents", exponents), ("lse", lse)):
        if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f"the cache's {name} must be contiguous and start on a 16-byte boundary")
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {D}")
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != dev or 0 in table.shape:
        raise ValueError(f"table must be int32 [sequences, pages] on {dev}, got {table.dtype} {list(table.shape)} on {table.device}")
    B = table.shape[0]
    if table.stride(1) != 1:
        table = table.contiguous()
    context = _int_vector("context", context, (B,), torch.int32, dev)
    if counts is not None:
        counts = _int_vector("counts", counts, (B,), torch.int32, dev)
    if n < 1:
        raise ValueError(f"expected at least one new token, got {n}")
    if ancestors is not None:
        if n > MAX_ANCESTORS:
            raise ValueError(f"at most {MAX_ANCESTORS} new tokens can have ancestors, got {n}")
        ancestors = _int_vector("ancestors", ancestors, (B, n), torch.int64, dev)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    c = _native.Cache(codes=codes.data_ptr(), exponents=exponents.data_ptr(), lse=ptr(lse), pages=pages, page_size=page_size, N=N, D=D,
                      code=_native.CODES[codes.dtype], table=table.data_ptr(), table_stride=table.stride(0) if B > 1 else 0,
                      table_pages=table.shape[1], context=context.data_ptr(), counts=ptr(counts), ancestors=ptr(ancestors), B=B, n=n)
    return c, (table, context, counts, ancestors)


def _check_new(cache, table, tensors):
    """New tokens' tensors against the cache, and laid out for the kernels."""
    x = tensors[0]
    if x.dim() != 4:
        raise ValueError(f"expected [batch, heads, tokens, head_dim] tensors, got shape {tuple(x.shape)}")
    want = (table.shape[0], cache.codes.shape[2], x.shape[2], cache.codes.shape[4])
    for t in tensors:
        if t.shape != want or t.dtype != x.dtype or t.device != cache.codes.device:
            raise ValueError(f"expected tensors of shape {list(want)}, all {x.dtype}, on {cache.codes.device}; got {list(t.shape)}, {t.dtype}, "
                             f"{t.device}")
    _native.dtype_code(x.dtype)
    return [_native.strided(t.detach()) for t in tensors]


def _cache(cache):
    if not isinstance(cache, TrittentionCache):
        raise ValueError(f"expected a TrittentionCache, got {type(cache).__name__}")
    return cache


def _flags(input_precision):
    if input_precision not in (None, "ieee"):
        raise ValueError(f"input_precision must be None or 'ieee', got {input_precision!r}")
    return _native.FLAG_FORCE_SIMT if input_precision == "ieee" else 0


def _wants_derivative(q):
    return (torch.is_grad_enabled() and q.requires_grad) or forward_mode()


def _need_lse(cache):
    if cache.lse is None:
        raise ValueError("the cache has no log-sum-exps: it is not one of the dot-product-sum form (new_cache(..., dps=True))")


def cache_write(cache: TrittentionCache, table: Tensor, context: Tensor, k1: Tensor, k2: Tensor, v1: Tensor, v2: Tensor,
                counts: Optional[Tensor] = None) -> None:
    """Quantises the new tokens' rows of K1, K2, SiLU(V1) and V2 into their places (``v1`` is the raw tensor); nothing else changes."""
    if torch.compiler.is_compiling():
        from . import ops

        _cache(cache)
        return ops.cache_write(cache.codes, cache.exponents, table, context, counts, k1, k2, v1, v2)
    done = _native.host_cache_write(*_cache(cache), table, context, counts, None, k1, k2, v1, v2)
    if done is not None:
        _native.host_result(done, "tritt_cache_write")
        return
    new = _check_new(cache, table, (k1, k2, v1, v2))
    c, keep = _describe(cache, table, context, new[0].shape[2], counts, None)
    _native.cache_write(c, new, _native.dtype_code(new[0].dtype), new[0].device)


def cache_read(cache: TrittentionCache, table: Tensor, context: Tensor, n: int, dtype: torch.dtype = torch.bfloat16,
               counts: Optional[Tensor] = None) -> Tuple[Tensor, ...]:
    """``n`` tokens of each sequence from token ``context[b]`` on, read back: the four parts ``[B, N, n, D]`` in ``dtype`` and, of a
    dot-product-sum cache, the log-sum-exps ``[B, N, n]``.  Zeros for tokens past ``counts[b]``."""
    if torch.compiler.is_compiling():
        from . import ops

        return tuple(ops.cache_read(*_cache(cache), table, context, n, dtype, counts))
    out = _native.host_cache_read(*_cache(cache), table, context, counts, None, n, _native.dtype_code(dtype))
    if out is not None:
        return _native.host_result(out, "tritt_cache_read")
    c, keep = _describe(cache, table, context, int(n), counts, None)
    code, dev = _native.dtype_code(dtype), cache.codes.device
    parts = tuple(torch.empty(c.B, c.N, c.n, c.D, dtype=dtype, device=dev) for _ in range(4))
    lse = None if cache.lse is None else torch.empty(c.B, c.N, c.n, dtype=torch.float32, device=dev)
    _native.cache_read(c, parts, lse, code, dev)
    return parts if lse is None else (*parts, lse)


def tdp_decode(q: Tensor, cache: TrittentionCache, table: Tensor, context: Tensor, softmax_scale: float = 1 / 8,
               k1_window: Optional[int] = None, k2_window: Optional[int] = None, kk_left: Optional[int] = None,
               kk_right: Optional[int] = None, counts: Optional[Tensor] = None, ancestors: Optional[Tensor] = None,
               return_lse: bool = False, input_precision: Optional[str] = None):
    """Triple-dot-product attention of new tokens whose rows are in the cache (``cache_write`` comes first): ``o`` ``[B, N, n, D]`` in ``q``'s
    type, or ``(o, lse)`` with the fp32 log-sum-exp ``[B, N, n]``.

    The mask is that of ``flash_trittention`` with ``causal``, over positions; a window of ``None`` has no limit.  A row past ``counts[b]`` or of a
    free slot is 0, its log-sum-exp ``-inf``.  16-bit queries with head dimension 64 or 128 run on the tensor cores: operands of at least 11
    significant bits, fp32 sums and soft-max.  fp32 queries, other head dimensions and ``input_precision="ieee"`` run in fp32 on the CUDA
    cores.  No gradient flows through the cache, and there is none for ``q``: a backward pass through the result raises.
    """
    flags, softmax_scale = _flags(input_precision), float(softmax_scale)
    if torch.compiler.is_compiling():
        from . import ops

        _cache(cache)
        o, lse = ops.tdp_decode(q, cache.codes, cache.exponents, table, context, softmax_scale, k1_window, k2_window, kk_left, kk_right, counts,
                                ancestors, input_precision)
        return (o, lse) if return_lse else o
    if _wants_derivative(q):
        return Undifferentiable.apply("tdp_decode", lambda: tdp_decode(q, cache, table, context, softmax_scale, k1_window, k2_window, kk_left, kk_right,
                                                                       counts, ancestors, return_lse, input_precision), q)
    out = _native.host_decode(_native.OP_TDP_DECODE, *_cache(cache), table, context, counts, ancestors, flags, softmax_scale, q, k1_window,
                              k2_window, kk_left, kk_right, bool(return_lse))
    if out is not None:
        o, lse = _native.host_result(out, "tritt_tdp_decode")
        return (o, lse) if return_lse else o
    q, = _check_new(cache, table, (q,))
    c, keep = _describe(cache, table, context, q.shape[2], counts, ancestors)
    windows = [_UNLIMITED if w is None else min(int(w), _UNLIMITED) for w in (k1_window, k2_window, kk_left, kk_right)]
    if min(windows) < 0:
        raise ValueError(f"window arguments must be >= 0, got {(k1_window, k2_window, kk_left, kk_right)}")
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    _native.tdp_decode(c, q, o, lse, softmax_scale, *windows, flags=flags)
    return (o, lse) if return_lse else o


def dps_append(cache: TrittentionCache, table: Tensor, context: Tensor, k1: Tensor, k2: Tensor, v1: Tensor, v2: Tensor,
               softmax_scale: float = 1 / 8, k_diff: int = 1024, counts: Optional[Tensor] = None, ancestors: Optional[Tensor] = None,
               input_precision: Optional[str] = None) -> None:
    """Writes new tokens of the dot-product-sum form: K1, K2, SiLU(V1), and for each token ``t``, attending from its ``k2`` to the tokens ``s``
    with ``position(t) - position(s) <= k_diff``, the row ``W = softmax(softmax_scale * k1[s].k2[t]) SiLU(v1[s]) * v2[t]`` and the
    log-sum-exp.  These do not depend on a query and are computed once.  Kernels as for ``tdp_decode``."""
    flags, softmax_scale = _flags(input_precision), float(softmax_scale)
    if torch.compiler.is_compiling():
        from . import ops

        _need_lse(_cache(cache))
        return ops.dps_append(*cache, table, context, k1, k2, v1, v2, softmax_scale, k_diff, counts, ancestors, input_precision)
    done = _native.host_decode(_native.OP_DPS_APPEND, *_cache(cache), table, context, counts, ancestors, flags, softmax_scale, k1, k2, v1, v2,
                               k_diff)
    if done is not None:
        _native.host_result(done, "tritt_dps_append")
        return
    _need_lse(cache)
    new = _check_new(cache, table, (k1, k2, v1, v2))
    c, keep = _describe(cache, table, context, new[0].shape[2], counts, ancestors)
    if k_diff < 0:
        raise ValueError(f"k_diff must be >= 0, got {k_diff}")
    _native.dps_append(c, new, softmax_scale, min(int(k_diff), _UNLIMITED), flags=flags)


def dps_decode(q: Tensor, cache: TrittentionCache, table: Tensor, context: Tensor, softmax_scale: float = 1 / 8,
               counts: Optional[Tensor] = None, ancestors: Optional[Tensor] = None,
               input_precision: Optional[str] = None) -> Tuple[Tensor, Tensor]:
    """Dot-product-sum attention of new tokens that ``dps_append`` has written: ``(o [B, N, n, D], m [B, N, n] fp32 log-sum-exp)``, as the module
    ``TrittentionTriton`` returns them.  Rows past ``counts[b]`` or of a free slot are 0 and ``-inf``.  Kernels and derivatives (none) as for
    ``tdp_decode``."""
    flags, softmax_scale = _flags(input_precision), float(softmax_scale)
    if torch.compiler.is_compiling():
        from . import ops

        _need_lse(_cache(cache))
        return ops.dps_decode(q, *cache, table, context, softmax_scale, counts, ancestors, input_precision)
    if _wants_derivative(q):
        return Undifferentiable.apply("dps_decode", lambda: dps_decode(q, cache, table, context, softmax_scale, counts, ancestors, input_precision), q)
    out = _native.host_decode(_native.OP_DPS_DECODE, *_cache(cache), table, context, counts, ancestors, flags, softmax_scale, q)
    if out is not None:
        return _native.host_result(out, "tritt_dps_decode")
    _need_lse(cache)
    q, = _check_new(cache, table, (q,))
    c, keep = _describe(cache, table, context, q.shape[2], counts, ancestors)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    m = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    _native.dps_decode(c, q, o, m, softmax_scale, flags=flags)
    return o, m
