"""Norms of queries and keys for each head with the position rotation in the same pass, in front of either attention.

The reference has no counterpart: its attention takes tensors that are normed and rotated elsewhere.
"""
import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native
from ._derivatives import Undifferentiable, forward_mode

__all__ = ["qk_norm_rotary", "rotary_tables"]

HEAD_DIMS = (16, 32, 64, 128, 256)


def rotary_tables(length: int, rot_dim: int, base: float = 10000.0, device=None) -> Tuple[Tensor, Tensor]:
    """``(cos, sin)``, each ``[length, rot_dim / 2]`` fp32, of the angles ``position * base ** (-2 i / rot_dim)``, which are formed in
    64 bits: in 32 the angle of position 100 000 would be off by 0.004."""
    if length < 1 or rot_dim < 16 or rot_dim % 16:
        raise ValueError(f"expected a length of at least 1 and a rot_dim that is a multiple of 16, got {length} and {rot_dim}")
    step = base ** (-torch.arange(0, rot_dim, 2, device=device, dtype=torch.float64) / rot_dim)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * step
    return angle.cos().float(), angle.sin().float()


def _check(xs, ws, cos, sin, positions):
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
    if positions is None:
        if T > cos.shape[0]:
            raise ValueError(f"the tables have {cos.shape[0]} positions, the sequence {T}")
    elif positions.shape not in ((T,), (B, T)) or positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError(f"positions must be int32 or int64 of shape [{T}] or [{B}, {T}] on {q.device}")


def _arguments(xs, ws, cos, sin, positions, eps, interleaved):
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
            a.position_stride_b = positions.stride(0) if positions.dim() == 2 else 0
    return a, keep + weights + [cos, sin, positions]


def norm_rotary_forward(xs, ws, cos, sin, positions, eps, interleaved):
    out = _native.host_norm_rotary(*xs, *ws, cos, sin, positions, eps, interleaved)
    if out is not None:
        return _native.host_result(out, "tritt_qk_norm_rotary_fwd")
    _check(xs, ws, cos, sin, positions)
    if not xs[0].is_cuda:
        raise RuntimeError("qk_norm_rotary runs on CUDA tensors only (there is no CPU path)")
    a, keep = _arguments(xs, ws, cos, sin, positions, eps, interleaved)
    ys = tuple(torch.empty(xs[0].shape, dtype=xs[0].dtype, device=xs[0].device) for _ in range(3))
    for i, y in enumerate(ys):
        a.y[i] = _native.rows(y)
    _native.norm_rotary(a, xs[0].device)
    return ys


def norm_rotary_backward(xs, ws, cos, sin, positions, eps, interleaved, dys, weights_too):
    """``(dq, dk1, dk2, dw, dw, dw)``; the inputs' gradients are laid out as the inputs, the weights' are ``None`` if not wanted."""
    out = _native.host_norm_rotary_backward(*xs, *ws, cos, sin, positions, eps, interleaved, *dys, *weights_too)
    if out is not None:
        return _native.host_result(out, "tritt_qk_norm_rotary_bwd")
    a, keep = _arguments(xs, ws, cos, sin, positions, eps, interleaved)
    dys = [_native.strided(torch.zeros_like(x) if dy is None else dy) for x, dy in zip(xs, dys)]
    dxs = [torch.empty_like(x) for x in xs]
    dws = [torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None and want else None for w, want in zip(ws, weights_too)]
    out = []
    for i in range(3):
        a.y[i] = _native.rows(dys[i])
        out.append(_native.strided(dxs[i]))   # (a layout that the kernel does not write gets a contiguous stand-in, and is copied)
        a.dx[i] = _native.rows(out[i])
        a.dw[i] = None if dws[i] is None else dws[i].data_ptr()
    _native.norm_rotary(a, xs[0].device, backward=True)
    return (*(dx if o is dx else dx.copy_(o) for dx, o in zip(dxs, out)), *dws)


class QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions, eps, interleaved):
        ys = norm_rotary_forward((q, k1, k2), (w_q, w_k1, w_k2), cos, sin, positions, eps, interleaved)
        ctx.save_for_backward(q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions)
        ctx.rest = (eps, interleaved)
        ctx.set_materialize_grads(False)
        return ys

    @staticmethod
    def backward(ctx, *dys):
        q, k1, k2, w_q, w_k1, w_k2, cos, sin, positions = ctx.saved_tensors
        if all(dy is None for dy in dys):
            return (None,) * 11

        def compute():
            return norm_rotary_backward((q, k1, k2), (w_q, w_k1, w_k2), cos, sin, positions, *ctx.rest, dys, ctx.needs_input_grad[3:6])

        # (with create_graph)
        grads = Undifferentiable.apply("the gradient of qk_norm_rotary", compute, q, k1, k2, w_q, w_k1, w_k2, *dys) if torch.is_grad_enabled() else compute()
        return (*grads, None, None, None, None, None)


def qk_norm_rotary(q: Tensor, k1: Tensor, k2: Tensor, q_weight: Optional[Tensor] = None, k1_weight: Optional[Tensor] = None,
                   k2_weight: Optional[Tensor] = None, cos: Optional[Tensor] = None, sin: Optional[Tensor] = None,
                   positions: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> Tuple[Tensor, Tensor, Tensor]:
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
    * ``head_dim`` is 16, 32, 64, 128 or 256, ``rot_dim`` a multiple of 16; without ``cos`` and ``sin`` nothing is rotated.

    In the dot-product-sum form, whose score is a sum of products of two vectors, rotated scores depend on distances alone; the triple
    product has no such rotation, positions still tell its rows apart.
    """
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be a finite number >= 0, got {eps}")
    if torch.compiler.is_compiling():
        from .ops import norm_rotary

        return norm_rotary(q, k1, k2, q_weight, k1_weight, k2_weight, cos, sin, positions, eps, bool(interleaved))
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k1, k2, q_weight, k1_weight, k2_weight))) or forward_mode():
        return QkNormRotary.apply(q, k1, k2, q_weight, k1_weight, k2_weight, cos, sin, positions, eps, bool(interleaved))
    return norm_rotary_forward((q, k1, k2), (q_weight, k1_weight, k2_weight), cos, sin, positions, eps, bool(interleaved))
