"""Norms of queries and keys for each head with the position rotation in the same pass, in front of either attention.

The reference has no counterpart: its attention takes tensors that are normed and rotated elsewhere.
"""
import ctypes as C
import functools
import math
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _native
from ._derivatives import Undifferentiable, forward_mode

__all__ = ["qk_norm_rotary", "rotary_tables", "rotary_axes"]

HEAD_DIMS = (16, 32, 64, 128, 256)
MAX_AXES = 4


def rotary_tables(length: int, rot_dim: int, base: float = 10000.0, device=None, axes: Optional[Sequence[int]] = None) -> Tuple[Tensor, Tensor]:
    """``(cos, sin)``, each ``[length, rot_dim / 2]`` fp32, of the angles ``position * base ** (-2 i / rot_dim)``, which are formed in
    64 bits: in 32 the angle of position 100 000 would be off by 0.004.

    With ``axes`` (see ``rotary_axes``) each axis has all speeds of its own, as the rows and columns of a picture do: the ``r``-th of its ``m`` pairs
    turns by ``position * base ** (-r / m)``.  Without it the pairs of all axes share one range of speeds."""
    if length < 1 or rot_dim < 16 or rot_dim % 16:
        raise ValueError(f"expected a length of at least 1 and a rot_dim that is a multiple of 16, got {length} and {rot_dim}")
    power = torch.arange(0, rot_dim, 2, device=device, dtype=torch.float64) / rot_dim
    if axes is not None:
        axes = _axes_of(axes, rot_dim // 2)
        power = torch.tensor([axes[:i].count(a) / axes.count(a) for i, a in enumerate(axes)], device=device, dtype=torch.float64)
    step = base ** -power
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * step
    return angle.cos().float(), angle.sin().float()


def rotary_axes(sections: Sequence[int], mixed: bool = False) -> Tuple[int, ...]:
    """The axis of each rotated pair where axis ``a`` has ``sections[a]`` of them: one axis after the other, or with ``mixed`` in turn for as long
    as each has pairs left (``(4, 2, 2)``: ``0 1 2 0 1 2 0 0``)."""
    left = [int(n) for n in sections]
    if not 0 < len(left) <= MAX_AXES or min(left) < 0 or sum(left) == 0:
        raise ValueError(f"expected the numbers of pairs of 1 to {MAX_AXES} axes, got {tuple(sections)}")
    if not mixed:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    return tuple(a for turn in range(max(left)) for a, n in enumerate(left) if turn < n)


def _axes_of(axes, pairs):
    axes = tuple(int(a) for a in axes)
    if len(axes) != pairs or min(axes) < 0 or max(axes) >= MAX_AXES:
        raise ValueError(f"axes must name the axis, 0 to {MAX_AXES - 1}, of each of the {pairs} rotated pairs, got {axes}")
    return axes


@functools.lru_cache(maxsize=64)
def _pack_axes(axes: Tuple[int, ...], pairs: int) -> bytes:
    """What the library takes: the number of axes, then two bits for each pair."""
    axes, of = _axes_of(axes, pairs), bytearray(32)
    for i, a in enumerate(axes):
        of[i // 4] |= a << 2 * (i % 4)
    return bytes([max(axes) + 1]) + bytes(of)


def _packed(axes, cos):
    if axes is None:
        return None
    if cos is None:
        raise ValueError("axes without cos and sin")
    try:
        return _pack_axes(tuple(axes), cos.shape[-1])
    except TypeError:   # (while a graph with symbols for sizes is traced: they are no keys of what is kept)
        return _pack_axes(tuple(int(a) for a in axes), int(cos.shape[-1]))


def _check(xs, ws, cos, sin, positions, axes=None):
    q = xs[0]
    if q.dim() != 4:
        raise ValueError(f"expected [batch, heads, seq_len, head_dim] tensors, got shape {tuple(q.shape)}")
    B, N, T, D = q.shape
    for name, t in zip(("k1", "k2"), xs[1:]):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} ({tuple(t.shape)}, {t.dtype}, {t.device}) does not match q ({tuple(q.shape)}, {q.dtype}, {q.device})")
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {D}")
    if q.numel() == 0:
        raise ValueError(f"empty tensors: {tuple(q.shape)}")
    _native.dtype_code(q.dtype)
    given = [w for w in ws if w is not None]
    for w in given:
        if w.shape not in ((D,), (N, D)) or w.shape != given[0].shape:
            raise ValueError(f"weights must all be [{D}] or all [{N}, {D}], got {[tuple(w.shape) for w in given]}")
        if w.dtype not in (q.dtype, torch.float32) or w.dtype != given[0].dtype or w.device != q.device:
            raise ValueError(f"weights must all be {q.dtype} or all float32, on {q.device}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is None:
        if positions is not None:
            raise ValueError("positions without cos and sin")
        return
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"cos and sin must be float32 tables [positions, rot_dim / 2], got {tuple(cos.shape)} {cos.dtype}, "
                         f"{tuple(sin.shape)} {sin.dtype}")
    rot = 2 * cos.shape[1]
    if rot % 16 or not 0 < rot <= D or cos.shape[0] < 1:
        raise ValueError(f"rot_dim must be a multiple of 16 up to head_dim {D}, got {rot}")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError(f"cos and sin must be on {q.device}")
    if axes is not None:
        count = axes[0]
        if positions is None or positions.dim() not in (2, 3) or not count <= positions.shape[0] <= MAX_AXES or positions.shape[1:] not in (
                (T,), (B, T)) or positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise ValueError(f"with axes positions must be int32 or int64 of shape [axes, {T}] or [axes, {B}, {T}], {count} to {MAX_AXES} axes, on "
                             f"{q.device}")
    elif positions is None:
        if T > cos.shape[0]:
            raise ValueError(f"the tables have {cos.shape[0]} positions, the sequence {T}")
    elif positions.shape not in ((T,), (B, T)) or positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError(f"positions must be int32 or int64 of shape [{T}] or [{B}, {T}] on {q.device}")


def _arguments(xs, ws, cos, sin, positions, eps, interleaved, axes=None):
    """The library's argument structure but for its outputs, and the tensors that it points to."""
    B, N, T, D = xs[0].shape
    a = _native.NormRotary(B=B, N=N, T=T, D=D, dtype=_native.dtype_code(xs[0].dtype), eps=eps)
    keep = [_native.strided(x) for x in xs]
    for i, x in enumerate(keep):
        a.x[i] = _native.rows(x)
    weights = [None if w is None else _native.aligned(w) for w in ws]
    for i, w in enumerate(weights):
        if w is not None:
            a.w[i] = w.data_ptr()
            a.weight_heads, a.weight_dtype = int(w.dim() == 2), _native.dtype_code(w.dtype)
    if cos is not None:
        cos, sin = _native.aligned(cos), _native.aligned(sin)
        a.cos, a.sin, a.table, a.rot, a.interleaved = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1], int(interleaved)
        if positions is not None:
            a.positions, a.positions64 = positions.data_ptr(), int(positions.dtype == torch.int64)
            a.position_stride_t = positions.stride(-1)
            a.position_stride_b = positions.stride(-2) if positions.dim() - (axes is not None) == 2 else 0
    return a, keep + weights + [cos, sin, positions]


def _rest(axes):
    """Packed axes as further arguments of a call: none where there are none."""
    return () if axes is None else (axes,)


def _axes_argument(axes, positions):
    """The library's structure for packed axes, as a further argument."""
    if axes is None:
        return {}
    return {"axes": _native.Axes(position_stride=positions.stride(0), count=axes[0], of=(C.c_ubyte * 32)(*axes[1:]))}


def norm_rotary_forward(xs, ws, cos, sin, positions, eps, interleaved, axes=None):
    """``axes``: packed (``_packed``)."""
    out = _native.host_norm_rotary(*xs, *ws, cos, sin, positions, eps, interleaved, *_rest(axes))
    if out is not None:
        return _native.host_result(out, "tritt_qk_norm_rotary_fwd")
    _check(xs, ws, cos, sin, positions, axes)
    if not xs[0].is_cuda:
        raise RuntimeError("qk_norm_rotary runs on CUDA tensors only (there is no CPU path)")
    a, keep = _arguments(xs, ws, cos, sin, positions, eps, interleaved, axes)
    ys = tuple(torch.empty(xs[0].shape, dtype=xs[0].dtype, device=xs[0].device) for _ in range(3))
    for i, y in enumerate(ys):
        a.y[i] = _native.rows(y)
    _native.norm_rotary(a, xs[0].device, **_axes_argument(axes, positions))
    return ys


def norm_rotary_backward(xs, ws, cos, sin, positions, eps, interleaved, dys, weights_too, axes=None):
    """``(dq, dk1, dk2, dw, dw, dw)``; the inputs' gradients are laid out as the inputs, the weights' are ``None`` if not wanted."""
    out = _native.host_norm_rotary_backward(*xs, *ws, cos, sin, positions, eps, interleaved, *dys, *weights_too, *_rest(axes))
    if out is not None:
        return _native.host_result(out, "tritt_qk_norm_rotary_bwd")
    a, keep = _arguments(xs, ws, cos, sin, positions, eps, interleaved, axes)
    dys = [_native.strided(torch.zeros_like(x) if dy is None else dy) for x, dy in zip(xs, dys)]
    dxs = [torch.empty_like(x) for x in xs]
    dws = [torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None and want else None for w, want in zip(ws, weights_too)]
    out = []
    for i in range(3):
        a.y[i] = _native.rows(dys[i])
        out.append(_native.strided(dxs[i]))   # (a layout that the kernel does not write gets a contiguous stand-in, and is copied)
        a.dx[i] = _native.rows(out[i])
        a.dw[i] = None if dws[i] is None else dws[i].data_ptr()
    _native.norm_rotary(a, xs[0].device, backward=True, **_axes_argument(axes, positions))
    return (*(dx if o is dx else dx.copy_(o) for dx, o in zip(dxs, out)), *dws)


class QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions, eps, interleaved, axes):
        ys = norm_rotary_forward((q, k1, k2), (w_q, w_k1, w_k2), cos, sin, positions, eps, interleaved, *axes)
        ctx.save_for_backward(q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions)
        ctx.rest, ctx.axes = (eps, interleaved), axes
        ctx.set_materialize_grads(False)
        return ys

    @staticmethod
    def backward(ctx, *dys):
        q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions = ctx.saved_tensors
        if all(dy is None for dy in dys):
            return (None,) * 12

        def compute():
            return norm_rotary_backward((q, k1, k2), (w_q, w_k1, w_k2), cos, sin, positions, *ctx.rest, dys, ctx.needs_input_grad[3:6],
                                        *ctx.axes)

        # (with create_graph)
        grads = Undifferentiable.apply("the gradient of qk_norm_rotary", compute, q, k1, k2, w_q, w_k1, w_k2, *dys) if torch.is_grad_enabled() else compute()
        return (*grads, None, None, None, None, None, None)


def qk_norm_rotary(q: Tensor, k1: Tensor, k2: Tensor, q_weight: Optional[Tensor] = None, k1_weight: Optional[Tensor] = None,
                   k2_weight: Optional[Tensor] = None, cos: Optional[Tensor] = None, sin: Optional[Tensor] = None,
                   positions: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                   axes: Optional[Sequence[int]] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``q, k1, k2`` normed for each head and rotated by their positions, in one pass; differentiable once, backwards (a second derivative and
    forward mode raise).

    Each row ``x`` of a tensor ``[B, N, T, D]`` becomes ``u = x / sqrt(mean(x^2) + eps) * weight``, and of its first ``2 * cos.shape[1]``
    elements each pair ``(a, b)`` becomes ``(a c - b s, b c + a s)`` with the values of its position in ``cos`` and ``sin`` (see
    ``rotary_tables``): the pairs ``(i, i + rot_dim / 2)``, or with ``interleaved`` ``(2 i, 2 i + 1)``.

    * The three tensors may be views with any strides whose rows are contiguous and 16-byte aligned (the parts of one fused
      projection, say); others are copied first.  The results are contiguous, as the attention takes them; arithmetic is fp32, rounded once.
    * A weight is ``[D]`` or, for each head, ``[N, D]``, in the tensors' type or float32, or ``None`` for ones.
    * ``positions`` (``[T]`` or ``[B, T]``, int32 or int64) default to ``0 .. T - 1``.  One that the tables do not have takes their nearest row,
      and the failure is reported by the next call or ``check_status()``.
    * Positions may have several axes (the time, row and column of a video's tokens): ``axes`` names the one of each rotated pair (see
      ``rotary_axes``), 1 to 4 in all, and ``positions`` are ``[axes, T]`` or ``[axes, B, T]``.
    * ``head_dim`` is 16, 32, 64, 128 or 256, ``rot_dim`` a multiple of 16; without ``cos`` and ``sin`` nothing is rotated.

    In the dot-product-sum form, whose score is a sum of products of two vectors, rotated scores depend on distances alone; the triple
    product has no such rotation, positions still tell its rows apart.
    """
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be a finite number >= 0, got {eps}")
    if torch.compiler.is_compiling():
        from .ops import norm_rotary

        return norm_rotary(q, k1, k2, q_weight, k1_weight, k2_weight, cos, sin, positions, eps, bool(interleaved),
                           None if axes is None else [int(a) for a in axes])
    axes = _packed(axes, cos)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k1, k2, q_weight, k1_weight, k2_weight))) or forward_mode():
        return QkNormRotary.apply(q, k1, k2, q_weight, k1_weight, k2_weight, cos, sin, positions, eps, bool(interleaved), _rest(axes))
    return norm_rotary_forward((q, k1, k2), (q_weight, k1_weight, k2_weight), cos, sin, positions, eps, bool(interleaved), *_rest(axes))
