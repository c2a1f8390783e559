"""64-bit restatement of the operators around the attention: norms with rotation, the quantised cache, attention of new tokens over it.

Plain loops over sequences, heads and new tokens, from the definitions in ``include/tritt.h``.  Each attention also returns what the error of a
kernel of limited precision is bounded by: the sum of the absolute values that a result is the difference of.
"""
import math

import torch

CODES = {"fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}


def norm_rotary(x, w, cos, sin, positions, eps=1e-6, interleaved=False):
    """fp64 result for one tensor [B, N, T, D] (differentiable)."""
    B, N, T, D = x.shape
    u = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        u = u * (w[None, :, None, :] if w.dim() == 2 else w)
    if cos is None:
        return u
    at = torch.arange(T).expand(B, T) if positions is None else positions.long().expand(B, T)
    at = at.clamp(0, cos.shape[0] - 1)
    c, s, half = cos.double()[at][:, None], sin.double()[at][:, None], cos.shape[1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = u[..., first], u[..., second]
    out = u.clone()
    out[..., first] = a * c - b * s
    out[..., second] = b * c + a * s
    return out


def silu(x):
    return x / (1 + torch.exp(-x))


def quantise(x, code):
    """(codes, exponent bytes, values) of fp64 rows [..., D]."""
    x = torch.where(x.abs() < 2.0 ** -126, torch.zeros_like(x), x)
    top = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    mantissa, e = torch.frexp(torch.where(finite, top, torch.zeros_like(top)))   # mantissa in [0.5, 1)
    e = e.long()
    if code == "fp16":
        e = e - 15
    else:
        m, shift = math.frexp(TOP[code])
        e = e - shift + (mantissa > m).long()
    e = torch.where(top == 0, torch.full_like(e, -126), e).clamp(min=-126)
    y = torch.where(finite.unsqueeze(-1), x, torch.zeros_like(x)) * torch.exp2(-e.double()).unsqueeze(-1)
    codes = (y.round() if code == "int8" else y).to(CODES[code])
    byte = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return codes, byte, values(codes, byte)


def values(codes, byte):
    v = codes.double() * torch.exp2(byte.double() - 127).unsqueeze(-1)
    return torch.where((byte == 255).unsqueeze(-1), torch.full_like(v, math.nan), v)


def visible(i, ancestors):
    """Numbers of the new tokens that new token i attends to, in order."""
    if ancestors is None:
        return list(range(i + 1))
    word = int(ancestors[i])
    return [m for m in range(i) if word >> m & 1] + [i]


def _tokens(ctx, i, ancestors):
    """(row numbers, positions) of the tokens that new token i attends to without a window, and its own position."""
    new = visible(i, ancestors)
    rows = list(range(ctx)) + [ctx + m for m in new]
    return torch.tensor(rows), torch.arange(len(rows)), len(rows) - 1


def tdp_row(q, k1, k2, v1, v2, ctx, i, alpha, windows=(None, None, None, None), ancestors=None):
    """One new token and head: q [D], cached values [tokens, D] in 64 bits (v1 gated).  -> (o, lse, sum of p |v1 v2|, largest sum of
    |alpha q k1 k2| over the attended pairs)."""
    k1w, k2w, kkl, kkr = (1 << 40 if w is None else w for w in windows)
    rows, pos, at = _tokens(ctx, i, ancestors)
    s = alpha * torch.einsum("d,jd,kd->jk", q, k1[rows], k2[rows])
    size = abs(alpha) * torch.einsum("d,jd,kd->jk", q.abs(), k1[rows].abs(), k2[rows].abs())
    pj, pk = pos[:, None], pos[None]
    seen = (at - pj <= k1w) & (at - pk <= k2w) & (pk - pj <= kkl) & (pj - pk <= kkr)
    if not bool(seen.any()):
        return _nothing(q)
    s = s.masked_fill(~seen, -math.inf)
    lse = s.flatten().logsumexp(0)
    p = (s - lse).exp()
    v1, v2 = v1[rows], v2[rows]
    o, mass = (v1 * (p @ v2)).sum(0), (v1.abs() * (p @ v2.abs())).sum(0)
    return o, lse, mass, size[seen].max()


def tdp_small(q, k1, k2, v1, v2, ctx, i, alpha, windows, ancestors, below):
    """Sum of |v1 v2| over the attended pairs of ``tdp_row`` whose p is less than ``below`` times the largest, times the largest p."""
    k1w, k2w, kkl, kkr = (1 << 40 if w is None else w for w in windows)
    rows, pos, at = _tokens(ctx, i, ancestors)
    s = alpha * torch.einsum("d,jd,kd->jk", q, k1[rows], k2[rows])
    pj, pk = pos[:, None], pos[None]
    s = s.masked_fill(~((at - pj <= k1w) & (at - pk <= k2w) & (pk - pj <= kkl) & (pj - pk <= kkr)), -math.inf)
    top = s.max()
    small = ((s < top + math.log(below)) & (s > -math.inf)).double()
    return (top - s.flatten().logsumexp(0)).exp() * (v1[rows].abs() * (small @ v2[rows].abs())).sum(0)


def dps_row(q, key, value, bias, ctx, i, alpha, window=None, ancestors=None):
    """The same for a soft-max over single tokens, with a bias for each or none."""
    rows, pos, at = _tokens(ctx, i, ancestors)
    s = alpha * (key[rows] @ q)
    size = abs(alpha) * (key[rows].abs() @ q.abs())
    if bias is not None:
        s, size = s + bias[rows], size + bias[rows].abs()
    seen = at - pos <= (1 << 40 if window is None else window)
    return _finish(s, size, seen, value[rows])


def _nothing(x):
    zero = torch.zeros_like(x)
    return zero, torch.tensor(-math.inf, dtype=torch.float64), zero, torch.tensor(0.0, dtype=torch.float64)


def _finish(s, size, seen, w):
    if not bool(seen.any()):
        return _nothing(w[0])
    s, w = s[seen], w[seen]
    lse = s.logsumexp(0)
    p = (s - lse).exp()
    return p @ w, lse, p @ w.abs(), size[seen].max()


class Sequences:
    """A batch's cached tokens in 64 bits, as a list of [4, N, tokens, D] values and lse [N, tokens], and the same in pages."""

    def __init__(self, parts, code, page_size, pages, table, lse=None):
        # parts: list over sequences of [4, N, tokens, D] (V1 gated already)
        self.table, self.page_size = table, page_size
        N, D = parts[0].shape[1], parts[0].shape[3]
        self.codes = torch.zeros(pages, 4, N, page_size, D, dtype=CODES[code])
        self.exponents = torch.zeros(pages, 4, N, page_size, dtype=torch.uint8)
        self.lse = None if lse is None else torch.zeros(pages, N, page_size)
        self.values = []
        for b, x in enumerate(parts):
            codes, byte, value = quantise(x, code)
            self.values.append(value)
            for t in range(x.shape[2]):
                page, row = int(table[b, t // page_size]), t % page_size
                self.codes.view(torch.uint8 if code != "fp16" else torch.float16)[page, :, :, row] = codes[:, :, t].view(
                    torch.uint8 if code != "fp16" else torch.float16)
                self.exponents[page, :, :, row] = byte[:, :, t]
                if lse is not None:
                    self.lse[page, :, row] = lse[b][:, t].float()
        self.bias = None if lse is None else [x.float().double() for x in lse]
