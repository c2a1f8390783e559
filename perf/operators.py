"""The operators around three-way attention as a model serves and trains with it: what is timed, on which inputs, and what they compute.

* ``norm``: norms of q, k1, k2 for each head with the position rotation in the same pass (``qk_norm_rotary``), forward, or forward and
  backward;
* ``cache``: rows of new tokens quantised into a paged cache and read back (``cache_write``, ``cache_read``);
* ``tdp``: triple-dot-product attention of one or a few new tokens, in a chain or a tree of drafts, over the cache (``tdp_decode``);
* ``append``: new tokens of the dot-product-sum form, whose inner attention over the cache leaves their rows W and log-sum-exps
  (``dps_append``), read back (``cache_read``);
* ``dps``: its outer attention of new tokens over the cache (``dps_decode``).

A case is a dict of plain values.  Common to the cached ones: ``B`` sequences of ``N`` heads, ``n`` new tokens each, the longest has
``context`` cached tokens and the others fewer (``_contexts``); ``code`` is what a cached element is held in; ``branch`` is 0 for a chain,
else token i's parent is token (i - 1) // branch; ``page`` is the page size in tokens.
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

def _norm(B, N, T, D, dtype, train, rot, interleaved=False, per_head=False, offset=0):
    return dict(op="norm", B=B, N=N, T=T, D=D, dtype=dtype, train=train, rot=rot, interleaved=interleaved, per_head=per_head, offset=offset)


def _cache(B, N, n, D, dtype, code, context, page):
    return dict(op="cache", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page)


def _tdp(B, N, n, D, dtype, code, context, page, branch=0, k1w=-1, k2w=-1, kkl=-1, kkr=-1):
    return dict(op="tdp", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page, branch=branch, k1w=k1w, k2w=k2w,
                kkl=kkl, kkr=kkr)


def _append(B, N, n, D, dtype, code, context, page, k_diff, branch=0):
    return dict(op="append", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page, branch=branch, k_diff=k_diff)


def _dps(B, N, n, D, dtype, code, context, page, branch=0):
    return dict(op="dps", B=B, N=N, n=n, D=D, dtype=dtype, code=code, context=context, page=page, branch=branch)


def listed():
    return [
        # one token of each of 16 sequences, far into their contexts: a serving step's smallest call
        dict(_norm(16, 16, 1, 128, "bf16", False, 128, offset=30000), name="norm_token_16x16x128_bf16"),
        # a training step at the headline benchmark's heads and length, four sequences (the largest)
        dict(_norm(4, 16, 2048, 128, "bf16", True, 128), name="norm_train_4x16x2048x128_bf16"),
        # a ragged length, weights of each head, neighbours rotated, half of the elements left alone
        dict(_norm(3, 5, 333, 64, "fp16", True, 32, True, True), name="norm_train_3x5x333x64_fp16"),
        # prompts of up to 2048 tokens written to a cache of 8-bit floats
        dict(_cache(8, 16, 2048, 64, "bf16", "e4m3", 0, 64), name="cache_prompt_8x16x2048x64_e4m3"),
        # a token of each of 64 sequences
        dict(_cache(64, 16, 1, 128, "fp16", "int8", 4000, 16), name="cache_token_64x16x128_int8"),
        # one token over short contexts
        dict(_tdp(4, 8, 1, 64, "fp16", "e4m3", 700, 64), name="tdp_token_4x8x700x64_e4m3"),
        # local attention under the banded benchmark's windows, a tree of 16 drafts for each sequence
        dict(_tdp(8, 16, 16, 64, "fp16", "int8", 4095, 16, 2, 128, 128, 32, 32), name="tdp_tree16_8x16x4095x64_int8_band"),
        # a chain of 8 tokens over the headline benchmark's length and head dimension: bound by its products
        dict(_tdp(1, 16, 8, 128, "bf16", "fp16", 2040, 64, 0), name="tdp_chain8_16x2040x128_fp16"),
        # one token written, with its inner attention over at most 1024 tokens
        dict(_append(32, 16, 1, 64, "bf16", "e4m3", 4000, 64, 1024), name="append_token_32x16x4000x64_e4m3"),
        # a tree of 24 drafts, long inner attention
        dict(_append(4, 16, 24, 128, "fp16", "fp16", 3001, 32, 4096, 3), name="append_tree24_4x16x3001x128_fp16"),
        # one token of each of 32 long sequences: bound by the cache's bytes
        dict(_dps(32, 16, 1, 64, "bf16", "e4m3", 8191, 64), name="dps_token_32x16x8191x64_e4m3"),
        # a tree of 24 drafts
        dict(_dps(4, 16, 24, 128, "fp16", "fp16", 3001, 32, 3), name="dps_tree24_4x16x3001x128_fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "cache", "tdp", "append", "dps"])
    D, N = rng.choice([64, 128]), rng.choice([4, 5, 8, 16])
    dtype, code, page = rng.choice(["bf16", "fp16"]), rng.choice(["fp16", "e4m3", "int8"]), rng.choice([16, 32, 64, 128, 256])
    B = _log_int(rng, 1, 32)
    if op == "norm":
        D = rng.choice([32, 64, 128, 256])
        T = _log_int(rng, 1, max(1, 4 * 16 * 2048 * 128 // (B * N * D) // 2))
        T = min(T, 8191)
        return _norm(B, N, T, D, rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.6, rng.choice([0, D // 2, D]), rng.random() < 0.4,
                     rng.random() < 0.5, rng.choice([0, rng.randrange(1, _TABLE - T)]))
    if op == "cache":
        n = _log_int(rng, 1, max(2, 8 * 16 * 2048 * 64 // (B * N * D)))
        return _cache(B, N, n, D, dtype, code, rng.randrange(0, 3000), page)
    n, branch = rng.choice([1, 1, 2, 5, 8, 16, 33]), rng.choice([0, 2, 3])
    if op == "tdp":
        windows = (-1, -1, -1, -1)
        if rng.random() < 0.5:
            windows = tuple(rng.choice([-1, rng.randrange(0, 300)]) for _ in range(4))
        # (the plain form holds one score for each pair)
        most = math.isqrt(16 * 8 * 2048 * 2048 // 2 // (B * N * n))
        context = _log_int(rng, 1, max(2, min(4000, most))) - 1
        return _tdp(B, N, n, D, dtype, code, context, page, branch, *windows)
    context = _log_int(rng, 1, max(2, min(9000, 32 * 16 * 8191 * 64 // (2 * B * N * D)))) - 1
    n = min(n, max(1, 8 * 16 * 8191 * 24 // (B * N * (context + 1))))
    if op == "append":
        return _append(B, N, n, D, dtype, code, context, page, rng.choice([100, 1024, 4096, 10000]), branch)
    return _dps(B, N, n, D, dtype, code, context, page, branch)


def _contexts(case):
    """Cached tokens of each sequence before the new ones: the longest, and others down to about half of it."""
    c, new = case["context"], case["op"] == "cache"
    return [max(0, c - (b * 997) % (c // 2 + 1)) if not new or c else 0 for b in range(case["B"])]


def _counts(case):
    """New tokens of each sequence: all of them, but for prompts, whose batch is padded to the longest."""
    n = case["n"]
    return [max(1, n - (b * 131) % (n // 2 + 1)) if case["op"] == "cache" else n for b in range(case["B"])]


def _parents(n, branch):
    return [i - 1 if branch == 0 else (i - 1) // branch if i else -1 for i in range(n)]


def _ancestors(n, branch):
    """Bit m of word i: token i attends to token m (its ancestors and itself)."""
    words = []
    for i, p in enumerate(_parents(n, branch)):
        words.append((words[p] if p >= 0 else 0) | 1 << i)
    return words


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


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    B, N, D, dtype = case["B"], case["N"], case["D"], _TYPES[case["dtype"]]
    if case["op"] == "norm":
        T = case["T"]
        # the five tensors come out of one projection, [B, T, 5, N, D]; heads differ in size as a trained model's do
        x = (randn(B, T, 5, N, D) * torch.exp(0.5 * randn(N, 1))).to(dtype)
        q, k1, k2 = (x[:, :, i].transpose(1, 2) for i in range(3))
        w = [(1 + 0.2 * randn(*((N, D) if case["per_head"] else (D,)))).to(dtype) for _ in range(3)]
        s = dict(case=case, q=q, k1=k1, k2=k2, w=w, cos=None, sin=None, positions=None)
        if case["rot"]:
            turn = torch.arange(_TABLE, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (
                -torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64) * 2 / case["rot"])
            s.update(cos=turn.cos().float(), sin=turn.sin().float())
            if case["offset"]:
                start = torch.arange(B, device=dev, dtype=torch.int64) * 31 % case["offset"]
                s.update(positions=case["offset"] - start[:, None] + torch.arange(T, device=dev))
        if case["train"]:
            for name in ("q", "k1", "k2"):
                s[name] = s[name].detach().requires_grad_(True)
            s["w"] = [t.requires_grad_(True) for t in w]
            s["dy"] = [randn(B, N, T, D).to(dtype) for _ in range(3)]
        return s
    n, code, page = case["n"], case["code"], case["page"]
    contexts = _contexts(case)
    most = -(-(max(contexts) + n) // page)
    pages = B * most + 3
    table = torch.randperm(pages, generator=g, device=dev)[: B * most].view(B, most).int()
    if case["op"] == "cache":
        codes = torch.zeros(pages, 4, N, page, D, device=dev, dtype=_CODES[code])
        exponents = torch.zeros(pages, 4, N, page, device=dev, dtype=torch.uint8)
    else:
        # the parts K1, K2, SiLU(V1) and V2, or for the dot-product-sum W, whose rows are means of the others' and smaller
        x = randn(4, pages, N, page, D)
        x[2] = x[2] * torch.sigmoid(x[2])
        if case["op"] in ("append", "dps"):
            x[3] *= 0.2 * torch.exp(0.5 * randn(pages, N, page, 1))
        codes, exponents = _encode(x, code)
        codes, exponents = codes.transpose(0, 1).contiguous(), exponents.transpose(0, 1).contiguous()
        del x
    s = dict(case=case, codes=codes, exponents=exponents, table=table, ancestors=None, counts=None, lse=None,
             context=torch.tensor(contexts, device=dev, dtype=torch.int32))
    if case["op"] in ("append", "dps"):
        s["lse"] = 5.0 + randn(pages, N, page)
    if case.get("branch"):
        words = torch.from_numpy(np.array(_ancestors(n, case["branch"]), dtype=np.uint64).view(np.int64))
        s["ancestors"] = words.to(dev).expand(B, n).contiguous()
    if case["op"] == "cache":
        s["counts"] = torch.tensor(_counts(case), device=dev, dtype=torch.int32)
    if case["op"] in ("tdp", "dps"):
        s["q"] = randn(B, N, n, D).to(dtype)
    else:
        x = randn(B, n, 4, N, D).to(dtype)
        s.update({name: x[:, :, i].transpose(1, 2) for i, name in enumerate(("k1", "k2", "v1", "v2"))})
    return s


# ---------------------------------------------------------------- the operators

def _windows(case):
    return [None if case[w] < 0 else case[w] for w in ("k1w", "k2w", "kkl", "kkr")]


def run(s):
    case = s["case"]
    if not own:
        return globals()["_plain_" + case["op"]](s)
    ft = _package()
    if case["op"] == "norm":
        y = ft.qk_norm_rotary(s["q"], s["k1"], s["k2"], *s["w"], s["cos"], s["sin"], s["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return list(y)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, [s["q"], s["k1"], s["k2"], *s["w"]], s["dy"]))
    cache = ft.TrittentionCache(s["codes"], s["exponents"], s["lse"])
    where = (cache, s["table"], s["context"])
    if case["op"] == "cache":
        ft.cache_write(*where, s["k1"], s["k2"], s["v1"], s["v2"], counts=s["counts"])
        return list(ft.cache_read(*where, case["n"], s["k1"].dtype, counts=s["counts"]))
    if case["op"] == "append":
        ft.dps_append(*where, s["k1"], s["k2"], s["v1"], s["v2"], _scale(case["D"]), case["k_diff"], ancestors=s["ancestors"])
        return list(ft.cache_read(*where, case["n"], s["k1"].dtype))
    if case["op"] == "dps":
        return list(ft.dps_decode(s["q"], *where, _scale(case["D"]), ancestors=s["ancestors"]))
    return ft.tdp_decode(s["q"], *where, _scale(case["D"]), *_windows(case), ancestors=s["ancestors"])


# ---------------------------------------------------------------- plain forms

def _plain_norm_one(x, w, s):
    case = s["case"]
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.float().unsqueeze(1) if w.dim() == 2 else w.float())
    if s["cos"] is None:
        return y
    at = s["positions"].unsqueeze(1) if s["positions"] is not None else torch.arange(x.shape[2], device=x.device)
    c, n, half = s["cos"][at], s["sin"][at], case["rot"] // 2
    if case["interleaved"]:
        a, b = y[..., : 2 * half: 2], y[..., 1: 2 * half: 2]
        turned = torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half: 2 * half]
        turned = torch.cat((a * c - b * n, b * c + a * n), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _plain_norm(s):
    x = [s["q"], s["k1"], s["k2"]]
    y = [_plain_norm_one(t, w, s).to(t.dtype) for t, w in zip(x, s["w"])]
    if not s["case"]["train"]:
        return y
    return [t.detach() for t in y] + list(torch.autograd.grad(y, x + s["w"], s["dy"]))


def _places(s, first, count):
    """Page and row of the tokens first[b] .. first[b] + count - 1, [B, count], and the tokens' numbers (past a table's end: its last token)."""
    page = s["codes"].shape[3]
    at = first.long()[:, None] + torch.arange(count, device=first.device)
    kept = at.clamp(max=s["table"].shape[1] * page - 1)
    return s["table"].long().gather(1, kept // page), kept % page, at


def _rows(s, part, first, count):
    """fp32 rows of one part, [B, N, count, D]."""
    p, r, _ = _places(s, first, count)
    codes = s["codes"][p, part, :, r] if s["codes"].dtype != torch.float8_e4m3fn else s["codes"].view(torch.uint8)[p, part, :, r].view(
        torch.float8_e4m3fn)
    return _decode(codes, s["exponents"][p, part, :, r]).transpose(1, 2)


def _store(s, part, rows):
    """Quantises fp32 rows [B, N, n, D] of the new tokens into one part."""
    p, r, _ = _places(s, s["context"], rows.shape[2])
    codes, exponents = _encode(rows.transpose(1, 2), s["case"]["code"])
    keep = slice(None)
    if s["counts"] is not None:
        keep = torch.arange(rows.shape[2], device=p.device) < s["counts"][:, None]
    bytes_ = torch.uint8 if codes.element_size() == 1 else codes.dtype
    s["codes"].view(bytes_)[p[keep], part, :, r[keep]] = codes.view(bytes_)[keep]
    s["exponents"][p[keep], part, :, r[keep]] = exponents[keep]


def _read_back(s):
    n, dtype = s["case"]["n"], s["k1"].dtype
    out = [_rows(s, part, s["context"], n) for part in range(4)]
    if s["counts"] is not None:
        keep = (torch.arange(n, device=s["context"].device) < s["counts"][:, None])[:, None, :, None]
        out = [torch.where(keep, t, 0.0) for t in out]
    out = [t.to(dtype) for t in out]
    if s["lse"] is not None:
        p, r, _ = _places(s, s["context"], n)
        out.append(s["lse"][p, :, r].transpose(1, 2))
    return out


def _silu(x):
    x = x.float()
    return x * torch.sigmoid(x)


def _plain_cache(s):
    for part, rows in enumerate((s["k1"].float(), s["k2"].float(), _silu(s["v1"]), s["v2"].float())):
        _store(s, part, rows)
    return _read_back(s)


def _seen(s, at):
    """(attended [B, n, J], position of the tokens numbered `at` [B, J], position of the new tokens [B, n])."""
    case, ctx = s["case"], s["context"].long()[:, None]
    n = case["n"]
    new = at - ctx                                               # number among the new tokens, or negative
    words = torch.from_numpy(np.array(_ancestors(n, case["branch"]), dtype=np.uint64).view(np.int64)).to(at.device)
    bits = (words[:, None] >> torch.arange(n, device=at.device)) & 1   # [n, n]
    depth = bits.sum(1) - 1
    inside = new.clamp(0, n - 1)
    seen = (new < 0)[:, None] | ((new < n)[:, None] & (bits.t()[inside].transpose(1, 2) > 0))
    return seen, torch.where(new < 0, at, ctx + depth[inside]), ctx + depth


def _plain_tdp(s):
    case = s["case"]
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    contexts, n = _contexts(case), case["n"]
    parts = []
    for part, window in ((0, k1w), (1, k2w)):   # rows that no window reaches are not gathered
        first = [max(0, c - window) for c in contexts]
        parts.append((torch.tensor(first, device=s["q"].device), max(c + n - f for c, f in zip(contexts, first))))
    (fj, nj), (fk, nk) = parts
    k1, v1, k2, v2 = _rows(s, 0, fj, nj), _rows(s, 2, fj, nj), _rows(s, 1, fk, nk), _rows(s, 3, fk, nk)
    (seen_j, pos_j, pos_q), (seen_k, pos_k, _) = _seen(s, fj[:, None] + torch.arange(nj, device=fj.device)), _seen(
        s, fk[:, None] + torch.arange(nk, device=fk.device))
    seen_j = seen_j & (pos_q[:, :, None] - pos_j[:, None] <= k1w)
    seen_k = seen_k & (pos_q[:, :, None] - pos_k[:, None] <= k2w)
    apart = pos_k[:, :, None] - pos_j[:, None]                   # [B, K, J]
    seen = seen_k[:, :, :, None] & seen_j[:, :, None] & ((apart <= kkl) & (-apart <= kkr))[:, None]
    a = s["q"].float().unsqueeze(3) * k2.unsqueeze(2) * _scale(case["D"])       # [B, N, n, K, D]
    p = a.flatten(2, 3) @ k1.transpose(2, 3)
    p = p.view(*a.shape[:4], nj).masked_fill_(~seen.unsqueeze(1), -math.inf)
    p = p.sub_(p.amax((3, 4), keepdim=True)).exp_()
    total = p.sum((3, 4))
    o = ((p.flatten(2, 3) @ v1).view_as(a) * v2.unsqueeze(2)).sum(3) / total.unsqueeze(-1)
    return o.to(s["q"].dtype)


def _all_seen(s):
    contexts = _contexts(s["case"])
    first = torch.zeros(len(contexts), device=s["context"].device, dtype=torch.int64)
    count = max(contexts) + s["case"]["n"]
    return first, count, _seen(s, torch.arange(count, device=first.device).expand(len(contexts), count))


def _plain_append(s):
    case = s["case"]
    for part, rows in ((0, s["k1"].float()), (1, s["k2"].float()), (2, _silu(s["v1"]))):
        _store(s, part, rows)
    first, count, (seen, pos, pos_q) = _all_seen(s)
    seen = seen & (pos_q[:, :, None] - pos[:, None] <= case["k_diff"])
    p = (s["k2"].float() * _scale(case["D"])) @ _rows(s, 0, first, count).transpose(2, 3)
    p = p.masked_fill_(~seen.unsqueeze(1), -math.inf)
    top = p.amax(3, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    _store(s, 3, p @ _rows(s, 2, first, count) / total * s["v2"].float())
    at, row, _ = _places(s, s["context"], case["n"])
    s["lse"][at, :, row] = (top + total.log()).squeeze(3).transpose(1, 2)
    return _read_back(s)


def _plain_dps(s):
    first, count, (seen, _, _) = _all_seen(s)
    at, row, _ = _places(s, first, count)
    p = (s["q"].float() * _scale(s["case"]["D"])) @ _rows(s, 1, first, count).transpose(2, 3)
    p = (p + s["lse"][at, :, row].permute(0, 2, 1).unsqueeze(2)).masked_fill_(~seen.unsqueeze(1), -math.inf)
    top = p.amax(3, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    return [(p @ _rows(s, 3, first, count) / total).to(s["q"].dtype), (top + total.log()).squeeze(3)]


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _exact_norm(case, s):
    outs, grads_x, grads_w = [], [], []
    R = case["rot"]
    turn = None
    if R:
        T = case["T"]
        at = s["positions"][:, None] if s["positions"] is not None else torch.arange(T, device=s["q"].device)[None, None]
        turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])   # rotation as a product of complex numbers

    def rotate(y, turn):
        if turn is None:
            return y
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
            du = rotate(s["dy"][i].double(), turn.conj() if turn is not None else None)
            h = x * r
            grads_w.append((du * h).sum((0, 2) if case["per_head"] else (0, 1, 2)))
            du = du * w_
            grads_x.append(r * (du - h * (du * h).sum(-1, keepdim=True) / case["D"]))
    return outs + grads_x + grads_w


def _exact_value(codes, exponents):
    return codes.double() * torch.exp2(exponents.double() - 127).unsqueeze(-1)


def _exact_quantised(x, code):
    """The value that the cache holds for fp64 rows."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()   # 2^e <= top < 2^(e + 1), whatever the logarithm's last bit
    if code == "fp16":
        e = e - 14
    else:
        most, low = (448.0, 8) if code == "e4m3" else (127.0, 6)
        e = e - low
        e = e + (top * torch.exp2(-e) > most).double()
    y = x * torch.exp2(-e)
    y = y.round() if code == "int8" else y.to(_CODES[code]).double()
    return y * torch.exp2(e)


def _exact_paths(case):
    """For each sequence: its tokens' rows in order, and for each new token the numbers of those that it attends to, by position."""
    parents, n = _parents(case["n"], case["branch"]), case["n"]
    for c in _contexts(case):
        lines = []
        for i in range(n):
            line, m = [], i
            while m >= 0:
                line.append(c + m)
                m = parents[m]
            lines.append(line[::-1])
        yield c, lines


def _exact_sequence(s, b, part, count):
    """Rows 0 .. count - 1 of sequence b, [N, count, D] in 64 bits."""
    page = s["codes"].shape[3]
    ids = s["table"][b, : -(-count // page)].long()
    codes = s["codes"].view(torch.uint8)[ids, part].view(s["codes"].dtype)
    return _exact_value(codes, s["exponents"][ids, part]).transpose(0, 1).flatten(1, 2)[:, :count]


def _exact_tdp(case, s):
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (c, lines) in enumerate(_exact_paths(case)):
        k1, k2, v1, v2 = (_exact_sequence(s, b, part, c + case["n"]) for part in range(4))
        for i, line in enumerate(lines):
            at = c + len(line) - 1                                 # the token's position
            token = lambda lo: torch.cat((torch.arange(lo, max(lo, c), device=out.device), torch.tensor(  # noqa: E731
                [t for d, t in enumerate(line) if c + d >= lo], device=out.device, dtype=torch.int64)))
            lj, lk = max(0, at - k1w), max(0, at - k2w)
            j, k = token(lj), token(lk)
            pj, pk = lj + torch.arange(len(j), device=out.device), lk + torch.arange(len(k), device=out.device)
            score = torch.einsum("nd,njd,nkd->njk", s["q"][b, :, i].double() * _scale(case["D"]), k1[:, j], k2[:, k])
            apart = pk[None] - pj[:, None]
            score = score.masked_fill((apart > kkl) | (-apart > kkr), -math.inf)
            prob = score.flatten(1).softmax(-1).view_as(score)
            out[b, :, i] = torch.einsum("njk,njd,nkd->nd", prob, v1[:, j], v2[:, k])
    return out


def _exact_append(case, s):
    back = [torch.zeros(s["k1"].shape, dtype=torch.float64, device=s["k1"].device) for _ in range(4)]
    lse = torch.zeros(s["k1"].shape[:3], dtype=torch.float64, device=s["k1"].device)
    v1 = s["v1"].double()
    for part, x in ((0, s["k1"].double()), (1, s["k2"].double()), (2, v1 / (1 + torch.exp(-v1)))):
        back[part] = _exact_quantised(x, case["code"])
    w = torch.zeros_like(back[0])
    for b, (c, lines) in enumerate(_exact_paths(case)):
        old = c + case["n"]
        keys, vals = _exact_sequence(s, b, 0, old), _exact_sequence(s, b, 2, old)
        keys[:, c:], vals[:, c:] = back[0][b], back[2][b]
        for i, line in enumerate(lines):
            at = c + len(line) - 1
            lo = max(0, at - case["k_diff"])
            j = torch.cat((torch.arange(lo, max(lo, c), device=w.device),
                           torch.tensor([t for d, t in enumerate(line) if c + d >= lo], device=w.device, dtype=torch.int64)))
            score = torch.einsum("nd,njd->nj", s["k2"][b, :, i].double() * _scale(case["D"]), keys[:, j])
            lse[b, :, i] = score.logsumexp(-1)
            w[b, :, i] = torch.einsum("nj,njd->nd", score.softmax(-1), vals[:, j]) * s["v2"][b, :, i].double()
    back[3] = _exact_quantised(w, case["code"])
    return back + [lse]


def _exact_dps(case, s):
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    m = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device=s["q"].device)
    for b, (c, lines) in enumerate(_exact_paths(case)):
        count = c + case["n"]
        keys, vals = _exact_sequence(s, b, 1, count), _exact_sequence(s, b, 3, count)
        ids = s["table"][b, : -(-count // case["page"])].long()
        bias = s["lse"][ids].transpose(0, 1).flatten(1)[:, :count].double()
        score = torch.einsum("nid,ntd->nit", s["q"][b].double() * _scale(case["D"]), keys) + bias[:, None]
        for i, line in enumerate(lines):
            hidden = torch.ones(count, dtype=torch.bool, device=o.device)
            hidden[:c], hidden[line] = False, False
            score[:, i].masked_fill_(hidden, -math.inf)
        m[b] = score.logsumexp(-1)
        o[b] = torch.einsum("nit,ntd->nid", score.softmax(-1), vals)
    return [o, m]


def _exact_cache(case, s):
    v1 = s["v1"].double()
    keep = torch.arange(case["n"], device=v1.device) < s["counts"][:, None]
    out = [_exact_quantised(x, case["code"]) for x in (s["k1"].double(), s["k2"].double(), v1 / (1 + torch.exp(-v1)), s["v2"].double())]
    return [t * keep[:, None, :, None] for t in out]


def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(case):
    """Attended pairs (j, k) of all new tokens, one head."""
    k1w, k2w, kkl, kkr = (1 << 30 if w is None else w for w in _windows(case))
    total = 0
    depths = [bin(w).count("1") - 1 for w in _ancestors(case["n"], case["branch"])]
    for c in _contexts(case):
        for d in depths:
            at = c + d
            k = np.arange(max(0, at - k2w), at + 1)
            total += int(np.maximum(0, np.minimum(at, k + kkr) - np.maximum(max(0, at - k1w), k - kkl) + 1).sum())
    return total


def work(case):
    B, N, D = case["B"], case["N"], case["D"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        x = 3 * B * N * case["T"] * D
        tables = 4 * case["rot"] * case["T"] * (B if case["offset"] else 1)
        passes = 5 if case["train"] else 2   # x, y; and in the backward x, dy, dx
        return {"bytes": passes * x * size + tables, "flops": x * (20 if case["train"] else 8)}
    n, row = case["n"], D * (2 if case["code"] == "fp16" else 1) + 1   # a cached row's codes and exponent
    contexts, depths = _contexts(case), [bin(w).count("1") for w in _ancestors(n, case.get("branch", 0))] if case["op"] != "cache" else []
    if case["op"] == "cache":
        tokens = sum(_counts(case)) * N
        # raw rows in, codes out, and read back: codes in, values out (zeros behind a sequence's last)
        return {"bytes": tokens * (4 * D * size + 8 * row) + 4 * B * N * n * D * size, "flops": tokens * 4 * D * 3}
    ends = 2 * B * N * n * D * size
    if case["op"] == "tdp":
        k1w, k2w = (1 << 30 if w is None else w for w in _windows(case)[:2])
        rows = sum(2 * (min(c, k1w) + n) + 2 * (min(c, k2w) + n) for c in contexts)
        return {"bytes": rows * N * row + ends, "flops": 4 * D * N * _pairs(case)}
    if case["op"] == "append":
        rows = sum(2 * min(c, case["k_diff"]) for c in contexts)
        pairs = sum(min(c + d, case["k_diff"] + 1) for c in contexts for d in depths)
        new = B * n * N * (2 * 4 * D * size + 8 * row + 12)   # raw rows in, codes out, and read back
        return {"bytes": rows * N * row + new, "flops": 4 * D * N * pairs}
    rows = sum(c + n for c in contexts)
    return {"bytes": rows * N * (2 * row + 4) + ends, "flops": 4 * D * N * sum(c + d for c in contexts for d in depths)}
