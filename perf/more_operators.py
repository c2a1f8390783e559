"""What keeps a three-way attention's cache short, and positions with several axes: what is timed, on which inputs, and what it computes.

* ``axes``: norms of q, k1, k2 for each head with the rotation by positions that have several axes, as tokens of images and video have
  (``qk_norm_rotary(..., axes=)``), forward, or forward and backward;
* ``tdp``: the attention weight that each cached token gets from new ones as j and as k of the triple dot product, added to what it got
  before (``tdp_weigh``);
* ``dps``: the same of the dot-product sum, from the new tokens' queries and from their inner attention (``dps_weigh``);
* ``evict``: of each sequence and head the tokens with the largest weights are kept, their rows moved together (``cache_evict``), and where
  a cached element has 8 bits read back (``cache_read``).

A case is a dict of plain values.  Common to the cached ones: ``B`` sequences of ``N`` heads, ``n`` new tokens each, the longest has
``context`` cached tokens and the others fewer (``_contexts``); ``code`` is what a cached element is held in; ``page`` is the page size in
tokens.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CODES = {"fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TABLE = 32768   # positions in the rotation's tables


def _package():
    where = os.path.join(os.getcwd(), "flash-3-way-attention_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    import flash_trittention

    return flash_trittention


# ---------------------------------------------------------------- cases

def _axes(B, N, T, D, dtype, train, sections, mixed=False, interleaved=False, per_head=False):
    """``sections``: pairs of each axis, as text; ``mixed``: the axes take turns among the pairs."""
    return dict(op="axes", B=B, N=N, T=T, D=D, dtype=dtype, train=train, sections=sections, mixed=mixed, interleaved=interleaved,
                per_head=per_head)


def _tdp(B, N, n, D, dtype, code, context, page, decay=1.0, k1w=-1, k2w=-1, kkl=-1, kkr=-1):
    return dict(op="tdp", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page, decay=decay, k1w=k1w, k2w=k2w, kkl=kkl,
                kkr=kkr)


def _dps(B, N, n, D, dtype, code, context, page, k_diff, decay=1.0):
    return dict(op="dps", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page, k_diff=k_diff, decay=decay)


def _evict(B, N, D, code, context, page, keep, first, recent, sum_form):
    return dict(op="evict", B=B, N=N, D=D, code=code, context=context, page=page, keep=keep, first=first, recent=recent, sum_form=sum_form)


def listed():
    return [
        # one token of each of 16 sequences of a video: a serving step's smallest call
        dict(_axes(16, 16, 1, 128, "bf16", False, "16,24,24"), name="axes_token_16x16x128_bf16"),
        # a training step at the headline benchmark's heads and length, four sequences (the largest of its kind)
        dict(_axes(4, 16, 2048, 128, "bf16", True, "16,24,24", mixed=True), name="axes_train_4x16x2048x128_bf16"),
        # images (height and width), a ragged length, weights of each head, neighbours rotated, half of the elements left alone
        dict(_axes(3, 5, 333, 64, "fp16", True, "8,8", False, True, True), name="axes_train_3x5x333x64_fp16"),
        # one token over short contexts
        dict(_tdp(4, 8, 1, 64, "fp16", "e4m3", 700, 64), name="tdp_token_4x8x700x64_e4m3"),
        # one token over the longest contexts, older weights fading
        dict(_tdp(2, 16, 1, 64, "bf16", "int8", 4095, 16, 0.99), name="tdp_token_2x16x4095x64_int8"),
        # the last 8 tokens of a prompt at the headline benchmark's length and head dimension
        dict(_tdp(1, 16, 8, 128, "bf16", "fp16", 2040, 64), name="tdp_last8_16x2040x128_fp16"),
        # local attention under the banded benchmark's windows
        dict(_tdp(8, 16, 16, 64, "fp16", "int8", 4095, 16, 1.0, 128, 128, 32, 32), name="tdp_16_8x16x4095x64_int8_band"),
        # one token of each of 32 long sequences: bound by the cache's bytes
        dict(_dps(32, 16, 1, 64, "bf16", "e4m3", 8191, 64, 1024), name="dps_token_32x16x8191x64_e4m3"),
        # the last 24 tokens of a prompt
        dict(_dps(4, 16, 24, 128, "fp16", "fp16", 3001, 32, 4096, 0.9), name="dps_last24_4x16x3001x128_fp16"),
        # short contexts back to 512 tokens
        dict(_evict(4, 8, 64, "e4m3", 700, 64, 512, 4, 64, False), name="evict_4x8x700x64_e4m3"),
        # half of long contexts, with the dot-product sum's log-sum-exps
        dict(_evict(8, 16, 64, "fp16", 8191, 64, 4096, 4, 256, True), name="evict_8x16x8191x64_fp16"),
        # one very long context
        dict(_evict(1, 16, 128, "fp16", 65001, 256, 16384, 16, 1000, False), name="evict_16x65001x128_fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["axes", "tdp", "dps", "evict"])
    D, N = rng.choice([64, 128]), rng.choice([4, 5, 8, 16])
    dtype, code, page = rng.choice(["bf16", "fp16"]), rng.choice(["fp16", "e4m3", "int8"]), rng.choice([16, 32, 64, 128, 256])
    B = _log_int(rng, 1, 32)
    if op == "axes":
        D = rng.choice([32, 64, 128, 256])
        T = min(_log_int(rng, 1, max(1, 4 * 16 * 2048 * 128 // (B * N * D) // 2)), 8191)
        pairs = rng.choice([D // 4, D // 2])
        count = rng.choice([2, 3, 4])
        cut = sorted(rng.sample(range(1, pairs), count - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cut, cut + [pairs]))
        return _axes(B, N, T, D, rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.6, sections, rng.random() < 0.4, rng.random() < 0.4,
                     rng.random() < 0.5)
    decay = rng.choice([1.0, 0.97, 0.0])
    if op == "evict":
        context = _log_int(rng, 40, max(50, min(65000, 16 * 65001 * 128 // (B * N * D))))
        keep = rng.randrange(context // 8 + 1, context)
        first = rng.randrange(0, min(17, keep // 4 + 1))
        return _evict(B, N, D, code, context, page, keep, first, rng.randrange(0, keep - first), rng.random() < 0.5)
    n = rng.choice([1, 1, 2, 5, 8, 16, 33])
    if op == "tdp":
        windows = (-1, -1, -1, -1)
        if rng.random() < 0.4:
            windows = tuple(rng.choice([-1, rng.randrange(0, 300)]) for _ in range(4))
        # (the plain form holds one score for each pair)
        most = math.isqrt(16 * 8 * 2048 * 2048 // 2 // (B * N * n))
        context = _log_int(rng, 1, max(2, min(4000, most))) - 1
        return _tdp(B, N, n, D, dtype, code, context, page, decay, *windows)
    context = _log_int(rng, 1, max(2, min(9000, 32 * 16 * 8191 * 64 // (2 * B * N * D)))) - 1
    n = min(n, max(1, 8 * 16 * 8191 * 24 // (B * N * (context + 1))))
    return _dps(B, N, n, D, dtype, code, context, page, rng.choice([100, 1024, 4096, 10000]), decay)


def _contexts(case):
    """Cached tokens of each sequence before the new ones: the longest, and others down to about half of it."""
    c = case["context"]
    return [max(0, c - (b * 997) % (c // 2 + 1)) for b in range(case["B"])]


def _axis_of_pairs(case):
    """The axis of each rotated pair: one after the other, or taking turns for as long as each has pairs left."""
    left = [int(x) for x in case["sections"].split(",")]
    if not case["mixed"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


# ---------------------------------------------------------------- inputs

def _scale(D):
    return 1.0 / math.sqrt(D)


def _split(x, top, f16):
    """(codes as floats that are not yet rounded, exponents) of rows: the least e with max |x| 2^-e <= top, or < 2^15 for fp16 codes."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = e - 15 if f16 else e - math.frexp(top)[1] + (m > math.frexp(top)[0]).to(e.dtype)
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(-126, 127)
    return torch.ldexp(x, -e.unsqueeze(-1)), e


def _encode(x, code):
    """Codes and biased exponents (one byte a row) of fp32 rows."""
    y, e = _split(x, 448.0 if code == "e4m3" else 127.0, code == "fp16")
    y = y.round() if code == "int8" else y
    return y.to(_CODES[code]), (e + 127).to(torch.uint8)


def _decode(codes, exponents):
    return torch.ldexp(codes.float(), exponents.int().unsqueeze(-1) - 127)


def _positions(case, g, dev):
    """``[axes, B, T]``: tokens of pictures of 24 rows of 32, one after the other, from a place of each sequence's own on."""
    start = torch.randint(0, 1000, (case["B"], 1), generator=g, device=dev)
    at = start * 768 + torch.arange(case["T"], device=dev)
    every = [at // 768 + 11 * start, at % 768 // 32, at % 32, at % 7]
    count = len(case["sections"].split(","))
    return torch.stack(every[:count] if count > 2 else every[1:3]).int()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    B, N, D = case["B"], case["N"], case["D"]
    if case["op"] == "axes":
        T, dtype = case["T"], _TYPES[case["dtype"]]
        # the five tensors come out of one projection, [B, T, 5, N, D]; heads differ in size as a trained model's do
        x = (randn(B, T, 5, N, D) * torch.exp(0.5 * randn(N, 1))).to(dtype)
        q, k1, k2 = (x[:, :, i].transpose(1, 2) for i in range(3))
        w = [(1 + 0.2 * randn(*((N, D) if case["per_head"] else (D,)))).to(dtype) for _ in range(3)]
        axis = _axis_of_pairs(case)
        turn = torch.arange(_TABLE, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(len(axis), device=dev, dtype=torch.float64) / len(axis))
        s = dict(case=case, q=q, k1=k1, k2=k2, w=w, cos=turn.cos().float(), sin=turn.sin().float(), positions=_positions(case, g, dev),
                 axes=tuple(axis), axis_index=torch.tensor(axis, device=dev))
        if case["train"]:
            for name in ("q", "k1", "k2"):
                s[name] = s[name].detach().requires_grad_(True)
            s["w"] = [t.requires_grad_(True) for t in w]
            s["dy"] = [randn(B, N, T, D).to(dtype) for _ in range(3)]
        return s
    code, page, contexts = case["code"], case["page"], _contexts(case)
    n = case.get("n", 0)
    most = -(-(max(contexts) + n) // page)
    pages = B * most + 3
    free = torch.randperm(pages, generator=g, device=dev)
    # the parts K1, K2, SiLU(V1) and V2, or for the dot-product-sum W, whose rows are means of the others' and smaller
    x = randn(4, pages, N, page, D)
    x[2] = x[2] * torch.sigmoid(x[2])
    x[3] *= torch.exp(0.5 * randn(pages, N, page, 1))
    codes, exponents = _encode(x, code)
    codes, exponents = codes.transpose(0, 1).contiguous(), exponents.transpose(0, 1).contiguous()
    del x
    s = dict(case=case, codes=codes, exponents=exponents, lse=None, table=free[: B * most].view(B, most).int(),
             context=torch.tensor(contexts, device=dev, dtype=torch.int32))
    length = most * page
    # weights that tokens have gathered from about as many new ones as come now: a few have most, many nearly nothing, some exactly none
    gathered = torch.exp(2.0 * randn(B, N, length)) * (torch.rand(B, N, length, generator=g, device=dev) > 0.05)
    s["weights"] = gathered = gathered * (0.25 * max(1, n) / max(contexts + [1]))
    if case["op"] == "evict":
        if case["sum_form"]:
            s["lse"] = 5.0 + randn(pages, N, page)
        # (the kept rows go to pages of their own, as where others still read the old ones)
        few = -(-case["keep"] // page)
        new = torch.arange(pages, pages + B * few, device=dev, dtype=torch.int32).view(B, few)
        s["table_out"] = new
        for name in ("codes", "exponents", "lse"):
            if s[name] is not None:
                s[name] = torch.cat((s[name].view(torch.uint8) if s[name].element_size() == 1 else s[name], torch.zeros(
                    B * few, *s[name].shape[1:], device=dev, dtype=torch.uint8 if s[name].element_size() == 1 else s[name].dtype))).view(
                        s[name].dtype)
        s["weights_out"] = torch.zeros(B, N, few * page, device=dev)
        s["start"] = torch.zeros(B, device=dev, dtype=torch.int32)
        return s
    s["out"] = torch.zeros_like(gathered)
    s["q"] = randn(B, N, n, D).to(_TYPES[case["dtype"]])
    if case["op"] == "tdp":
        s["total"] = _tdp_scores(s)[0].flatten(3).logsumexp(-1)
        return s
    s["lse"] = 5.0 + randn(pages, N, page)
    s["k2"] = randn(B, N, n, D).to(_TYPES[case["dtype"]])
    inner = _dps_inner(s)
    at, row, _ = _places(s, s["context"], n)
    s["lse"][at, :, row] = inner.logsumexp(-1).transpose(1, 2)
    s["total"] = _dps_outer(s).logsumexp(-1)
    return s


# ---------------------------------------------------------------- the operators

def _windows(case):
    return [None if case[w] < 0 else case[w] for w in ("k1w", "k2w", "kkl", "kkr")]


def run(s):
    case = s["case"]
    if not own:
        return globals()["_plain_" + case["op"]](s)
    ft = _package()
    if case["op"] == "axes":
        y = ft.qk_norm_rotary(s["q"], s["k1"], s["k2"], *s["w"], s["cos"], s["sin"], s["positions"], interleaved=case["interleaved"],
                              axes=s["axes"])
        if not case["train"]:
            return list(y)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, [s["q"], s["k1"], s["k2"], *s["w"]], s["dy"]))
    cache = ft.TrittentionCache(s["codes"], s["exponents"], s["lse"])
    where = (cache, s["table"], s["context"])
    if case["op"] == "tdp":
        ft.tdp_weigh(s["weights"], s["q"], s["total"], *where, _scale(case["D"]), *_windows(case), decay=case["decay"], out=s["out"])
        return s["out"]
    if case["op"] == "dps":
        ft.dps_weigh(s["weights"], s["q"], s["k2"], s["total"], *where, _scale(case["D"]), case["k_diff"], decay=case["decay"], out=s["out"])
        return s["out"]
    context, kept = ft.cache_evict(s["weights"], *where, case["keep"], case["first"], case["recent"], table_out=s["table_out"],
                                   weights_out=s["weights_out"])
    if case["code"] == "fp16":
        return [context, kept, s["weights_out"], s["codes"], s["exponents"]] + ([s["lse"]] if case["sum_form"] else [])
    return [context, kept, s["weights_out"], *ft.cache_read(cache, s["table_out"], s["start"], case["keep"], torch.bfloat16)]


# ---------------------------------------------------------------- plain forms

def _plain_axes_one(x, w, s):
    case = s["case"]
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.float().unsqueeze(1) if w.dim() == 2 else w.float())
    half = len(s["axes"])
    at = s["positions"][s["axis_index"]].permute(1, 2, 0).long()                # [B, T, pairs]
    pair = torch.arange(half, device=x.device)
    c, n = s["cos"][at, pair].unsqueeze(1), s["sin"][at, pair].unsqueeze(1)
    if case["interleaved"]:
        a, b = y[..., : 2 * half: 2], y[..., 1: 2 * half: 2]
        turned = torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half: 2 * half]
        turned = torch.cat((a * c - b * n, b * c + a * n), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _plain_axes(s):
    x = [s["q"], s["k1"], s["k2"]]
    y = [_plain_axes_one(t, w, s).to(t.dtype) for t, w in zip(x, s["w"])]
    if not s["case"]["train"]:
        return y
    return [t.detach() for t in y] + list(torch.autograd.grad(y, x + s["w"], s["dy"]))


def _places(s, first, count, table="table"):
    """Page and row of the tokens first[b] .. first[b] + count - 1, [B, count], and the tokens' numbers (past a table's end: its last token)."""
    page, table = s["codes"].shape[3], s[table]
    at = first.long()[:, None] + torch.arange(count, device=first.device)
    kept = at.clamp(max=table.shape[1] * page - 1)
    return table.long().gather(1, kept // page), kept % page, at


def _rows(s, part, first, count, table="table"):
    """fp32 rows of one part, [B, N, count, D]."""
    p, r, _ = _places(s, first, count, table)
    codes = s["codes"][p, part, :, r] if s["codes"].dtype != torch.float8_e4m3fn else s["codes"].view(torch.uint8)[p, part, :, r].view(
        torch.float8_e4m3fn)
    return _decode(codes, s["exponents"][p, part, :, r]).transpose(1, 2)


def _tdp_scores(s):
    """Scores [B, N, n, K, J] (-inf where not attended), and the numbers of the first tokens j and k of each sequence."""
    case = s["case"]
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    contexts, n = _contexts(case), case["n"]
    parts = []
    for part, window in ((0, k1w), (1, k2w)):   # rows that no window reaches are not gathered
        first = [max(0, c - window) for c in contexts]
        parts.append((torch.tensor(first, device=s["q"].device), max(c + n - f for c, f in zip(contexts, first))))
    (fj, nj), (fk, nk) = parts
    pos_q = s["context"].long()[:, None] + torch.arange(n, device=fj.device)
    pos_j, pos_k = fj[:, None] + torch.arange(nj, device=fj.device), fk[:, None] + torch.arange(nk, device=fk.device)
    back_j, back_k = pos_q[:, :, None] - pos_j[:, None], pos_q[:, :, None] - pos_k[:, None]
    seen_j, seen_k = (back_j >= 0) & (back_j <= k1w), (back_k >= 0) & (back_k <= k2w)
    apart = pos_k[:, :, None] - pos_j[:, None]                   # [B, K, J]
    seen = seen_k[:, :, :, None] & seen_j[:, :, None] & ((apart <= kkl) & (-apart <= kkr))[:, None]
    a = s["q"].float().unsqueeze(3) * _rows(s, 1, fk, nk).unsqueeze(2) * _scale(case["D"])       # [B, N, n, K, D]
    p = a.flatten(2, 3) @ _rows(s, 0, fj, nj).transpose(2, 3)
    return p.view(*a.shape[:4], nj).masked_fill_(~seen.unsqueeze(1), -math.inf), fj, fk


def _begin(s):
    """Weights of before: of the cached tokens, faded; none of the new ones; of places behind them what is there."""
    case, old = s["case"], s["weights"]
    at = torch.arange(old.shape[2], device=old.device)
    ctx = s["context"].long()[:, None, None]
    w = torch.where(at < ctx, old * case["decay"], torch.zeros_like(old))
    return w, at, ctx


def _end(s, w, at, ctx):
    s["out"].copy_(torch.where(at < ctx + s["case"]["n"], w, s["out"]))
    return s["out"]


def _plain_tdp(s):
    p, fj, fk = _tdp_scores(s)
    p = p.sub_(s["total"][..., None, None]).exp_()
    w, at, ctx = _begin(s)
    for first, sums in ((fj, p.sum((2, 3))), (fk, p.sum((2, 4)))):
        here = at - first[:, None]                                # [B, L]: a place's number among the sums
        inside = (here >= 0) & (here < sums.shape[2])
        w = w + torch.where(inside[:, None], sums.gather(2, here.clamp(0, sums.shape[2] - 1)[:, None].expand(w.shape)), 0.0)
    return _end(s, w, at, ctx)


def _everything(s):
    first = torch.zeros(s["case"]["B"], device=s["context"].device, dtype=torch.int64)
    count = max(_contexts(s["case"])) + s["case"]["n"]
    back = (s["context"].long()[:, None] + torch.arange(s["case"]["n"], device=first.device))[:, :, None] - torch.arange(count, device=first.device)
    return first, count, back                                    # how far each token lies behind each new one, [B, n, count]


def _dps_inner(s):
    first, count, back = _everything(s)
    p = (s["k2"].float() * _scale(s["case"]["D"])) @ _rows(s, 0, first, count).transpose(2, 3)
    return p.masked_fill_(~((back >= 0) & (back <= s["case"]["k_diff"])).unsqueeze(1), -math.inf)


def _dps_outer(s):
    first, count, back = _everything(s)
    at, row, _ = _places(s, first, count)
    p = (s["q"].float() * _scale(s["case"]["D"])) @ _rows(s, 1, first, count).transpose(2, 3)
    return (p + s["lse"][at, :, row].permute(0, 2, 1).unsqueeze(2)).masked_fill_((back < 0).unsqueeze(1), -math.inf)


def _plain_dps(s):
    at, row, _ = _places(s, s["context"], s["case"]["n"])
    own_lse = s["lse"][at, :, row].transpose(1, 2).unsqueeze(3)
    new = _dps_outer(s).sub_(s["total"].unsqueeze(3)).exp_().sum(2) + _dps_inner(s).sub_(own_lse).exp_().sum(2)
    w, at, ctx = _begin(s)
    w = w + torch.nn.functional.pad(new, (0, w.shape[2] - new.shape[2]))
    return _end(s, w, at, ctx)


def _plain_evict(s):
    case = s["case"]
    keep, page = case["keep"], case["page"]
    w, length = s["weights"], s["weights"].shape[2]
    at = torch.arange(length, device=w.device)
    ctx = s["context"].long()[:, None, None]
    key = torch.where((at < case["first"]) | (at >= ctx - case["recent"]), math.inf, w)
    key = torch.where(at < ctx, key, -math.inf)
    kept = key.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values   # (ties: the lowest numbers first)
    # a sequence that has no more than `keep` tokens keeps them all, where they are
    count = ctx.clamp(max=keep)
    place = torch.arange(keep, device=w.device)
    kept = torch.where(ctx <= keep, place, kept)
    there = (place < count).expand(kept.shape)
    s["weights_out"][..., :keep] = torch.where(there, w.gather(2, kept), s["weights_out"][..., :keep])
    # rows [B, N, keep] of every part, from their pages to the new ones
    page_of, heads = s["table"].long()[:, None].expand(-1, case["N"], -1), torch.arange(case["N"], device=w.device)[None, :, None].expand(kept.shape)
    source = page_of.gather(2, (kept // page).clamp(max=page_of.shape[2] - 1))
    target = s["table_out"].long()[:, None].expand(-1, case["N"], -1).gather(2, (place // page).expand(kept.shape))
    t, h, r = target[there], heads[there], (place % page).expand(kept.shape)[there]
    f, o = source[there], (kept % page)[there]
    codes = s["codes"] if s["codes"].element_size() == 2 else s["codes"].view(torch.uint8)
    for part in range(4):
        codes[t, part, h, r] = codes[f, part, h, o]
        s["exponents"][t, part, h, r] = s["exponents"][f, part, h, o]
    if case["sum_form"]:
        s["lse"][t, h, r] = s["lse"][f, h, o]
    out = [count.flatten().int(), torch.where(there, kept, -1).int(), s["weights_out"]]
    if case["code"] == "fp16":
        return out + [s["codes"], s["exponents"]] + ([s["lse"]] if case["sum_form"] else [])
    out += [_rows(s, part, s["start"], keep, "table_out").bfloat16() for part in range(4)]
    if case["sum_form"]:
        p, row, _ = _places(s, s["start"], keep, "table_out")
        out.append(s["lse"][p, :, row].transpose(1, 2))
    return out


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _exact_axes(case, s):
    outs, grads_x, grads_w = [], [], []
    R = 2 * len(s["axes"])
    T = case["T"]
    turn = torch.empty(case["B"], 1, T, R // 2, dtype=torch.complex128, device=s["q"].device)   # rotation as a product of complex numbers
    for i, a in enumerate(s["axes"]):
        at = s["positions"][a].long()
        turn[:, 0, :, i] = torch.complex(s["cos"][:, i].double()[at], s["sin"][:, i].double()[at])

    def rotate(y, turn):
        head = y[..., :R]
        pairs = head.unflatten(-1, (R // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, y[..., R:]), -1)

    for i, name in enumerate(("q", "k1", "k2")):
        x, w = s[name].detach().double(), s["w"][i].detach().double()
        w_ = w[None, :, None] if case["per_head"] else w
        r = (x.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6) ** -0.5
        outs.append(rotate(x * r * w_, turn))
        if case["train"]:
            du = rotate(s["dy"][i].double(), turn.conj())
            h = x * r
            grads_w.append((du * h).sum((0, 2) if case["per_head"] else (0, 1, 2)))
            du = du * w_
            grads_x.append(r * (du - h * (du * h).sum(-1, keepdim=True) / case["D"]))
    return outs + grads_x + grads_w


def _exact_sequence(s, b, part, count):
    """Rows 0 .. count - 1 of sequence b, [N, count, D] in 64 bits."""
    page = s["codes"].shape[3]
    ids = s["table"][b, : -(-count // page)].long()
    codes = s["codes"].view(torch.uint8)[ids, part].view(s["codes"].dtype)
    value = codes.double() * torch.exp2(s["exponents"][ids, part].double() - 127).unsqueeze(-1)
    return value.transpose(0, 1).flatten(1, 2)[:, :count]


def _exact_tdp(case, s):
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    out = s["out"].double()
    dev, n = out.device, case["n"]
    for b, c in enumerate(_contexts(case)):
        k1, k2 = _exact_sequence(s, b, 0, c + n), _exact_sequence(s, b, 1, c + n)
        gain = torch.zeros(case["N"], c + n, dtype=torch.float64, device=dev)
        for i in range(n):
            lj, lk, end = max(0, c + i - k1w), max(0, c + i - k2w), c + i + 1
            pj, pk = torch.arange(lj, end, device=dev), torch.arange(lk, end, device=dev)
            apart = pk[None] - pj[:, None]
            for h in range(case["N"]):
                score = (k1[h, lj:end] * s["q"][b, h, i].double() * _scale(case["D"])) @ k2[h, lk:end].T
                prob = torch.exp(score - s["total"][b, h, i].double()) * ((apart <= kkl) & (-apart <= kkr))
                gain[h, lj:end] += prob.sum(1)
                gain[h, lk:end] += prob.sum(0)
        out[b, :, : c + n] = gain
        out[b, :, :c] += case["decay"] * s["weights"][b, :, :c].double()
    return out


def _exact_dps(case, s):
    out = s["out"].double()
    n = case["n"]
    for b, c in enumerate(_contexts(case)):
        count = c + n
        ids = s["table"][b, : -(-count // case["page"])].long()
        lse = s["lse"][ids].transpose(0, 1).flatten(1)[:, :count].double()
        k1, k2 = _exact_sequence(s, b, 0, count), _exact_sequence(s, b, 1, count)
        gain = torch.zeros(case["N"], count, dtype=torch.float64, device=out.device)
        for i in range(n):
            end, lo = c + i + 1, max(0, c + i - case["k_diff"])
            score = torch.einsum("nd,ntd->nt", s["q"][b, :, i].double() * _scale(case["D"]), k2[:, :end]) + lse[:, :end]
            gain[:, :end] += torch.exp(score - s["total"][b, :, i, None].double())
            score = torch.einsum("nd,ntd->nt", s["k2"][b, :, i].double() * _scale(case["D"]), k1[:, lo:end])
            gain[:, lo:end] += torch.exp(score - lse[:, c + i, None])
        out[b, :, :count] = gain
        out[b, :, :c] += case["decay"] * s["weights"][b, :, :c].double()
    return out


def _exact_evict(case, s):
    """Chosen one sequence and head at a time, on the host; the rows' values."""
    B, N, keep, page = case["B"], case["N"], case["keep"], case["page"]
    if B * N * max(_contexts(case)) > 4_000_000:
        return None
    weights, context = s["weights"].cpu().numpy(), _contexts(case)
    kept = np.full((B, N, keep), -1, dtype=np.int32)
    out_w = s["weights_out"].cpu().double().numpy()
    for b in range(B):
        c = context[b]
        for h in range(N):
            if c <= keep:
                at = np.arange(c)
            else:
                middle = np.arange(case["first"], c - case["recent"])
                order = np.lexsort((middle, -weights[b, h, middle].astype(np.float64)))
                chosen = middle[order[: keep - case["first"] - case["recent"]]]
                at = np.sort(np.concatenate((np.arange(case["first"]), chosen, np.arange(c - case["recent"], c))))
            kept[b, h, : len(at)] = at
            out_w[b, h, : len(at)] = weights[b, h, at]
    dev = s["codes"].device
    kept_t = torch.from_numpy(kept).to(dev)
    out = [torch.tensor([min(c, keep) for c in context], dtype=torch.int32, device=dev), kept_t, torch.from_numpy(out_w).to(dev)]
    codes, exponents, lse = s["codes"].view(torch.uint8).view(*s["codes"].shape[:4], -1).clone(), s["exponents"].clone(), s["lse"]
    lse = None if lse is None else lse.clone()
    heads = torch.arange(N, device=dev)
    values = [torch.zeros(B, N, keep, case["D"], dtype=torch.float64, device=dev) for _ in range(4)]
    sums = torch.zeros(B, N, keep, dtype=torch.float64, device=dev)
    for b in range(B):
        r = torch.arange(min(context[b], keep), device=dev)
        frm, to = kept_t[b, :, : len(r)].long(), s["table_out"][b].long()[r // page]
        src = s["table"][b].long()[frm // page]                  # [N, kept]
        for part in range(4):
            moved, power = codes[src, part, heads[:, None], frm % page], exponents[src, part, heads[:, None], frm % page]
            codes[to, part, :, r % page] = moved.transpose(0, 1)
            exponents[to, part, :, r % page] = power.transpose(0, 1)
            values[part][b, :, : len(r)] = moved.view(s["codes"].dtype).double() * torch.exp2(power.double() - 127).unsqueeze(-1)
        if lse is not None:
            lse[to, :, r % page] = s["lse"][src, heads[:, None], frm % page].transpose(0, 1)
            sums[b, :, : len(r)] = s["lse"][src, heads[:, None], frm % page].double()
    if case["code"] == "fp16":
        return out + [codes.view(torch.float16), exponents] + ([lse] if lse is not None else [])
    return out + values + ([sums] if lse is not None else [])


def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(case):
    """Attended pairs (j, k) of all new tokens, one head."""
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    total = 0
    for c in _contexts(case):
        for at in range(c, c + case["n"]):
            k = np.arange(max(0, at - k2w), at + 1)
            total += int(np.maximum(0, np.minimum(at, k + kkr) - np.maximum(max(0, at - k1w), k - kkl) + 1).sum())
    return total


def work(case):
    B, N, D = case["B"], case["N"], case["D"]
    if case["op"] == "axes":
        size = 4 if case["dtype"] == "fp32" else 2
        x, axis = 3 * B * N * case["T"] * D, _axis_of_pairs(case)
        tables = B * case["T"] * (8 * len(axis) + 4 * (max(axis) + 1))
        passes = 5 if case["train"] else 2   # x, y; and in the backward x, dy, dx
        return {"bytes": passes * x * size + tables, "flops": x * (20 if case["train"] else 8)}
    row = D * (2 if case["code"] == "fp16" else 1) + 1   # a cached row's codes and exponent
    contexts = _contexts(case)
    if case["op"] == "evict":
        kept = [min(c, case["keep"]) for c in contexts]
        moved = 2 * sum(kept) * (4 * row + 4 + (4 if case["sum_form"] else 0))   # rows and weights, in and out
        back = 0 if case["code"] == "fp16" else sum(kept) * 4 * row + B * case["keep"] * 4 * D * 2
        return {"bytes": N * (4 * sum(contexts) + moved + 4 * B * case["keep"] + back), "flops": N * sum(contexts)}
    n = case["n"]
    ends = B * N * n * (2 * D + 4)
    weights = sum(8 * c + 4 * n for c in contexts)               # of before and after
    if case["op"] == "tdp":
        k1w, k2w = (1 << 30 if w is None else w for w in _windows(case)[:2])
        rows = sum(min(c, k1w) + n + min(c, k2w) + n for c in contexts)
        return {"bytes": N * (rows * row + weights) + ends, "flops": (2 * D + 4) * N * _pairs(case)}
    rows = sum(c + n + min(c, case["k_diff"]) + n for c in contexts)
    reach = sum(c + i + 1 + min(c + i, case["k_diff"]) + 1 for c in contexts for i in range(n))
    return {"bytes": N * (rows * row + 4 * sum(contexts) + weights) + 2 * ends, "flops": (2 * D + 4) * N * reach}
