"""The paged cache and attention of new tokens over it, against the 64-bit definitions (``oracle/serving_oracle.py``).

Tolerances are counted from the arithmetic.  A result is sum p w / sum p; a kernel whose scores are off by at most d (absolutely) has every p
off by a factor within e^(+-d), the quotient by e^(+-2d): 2 d sum p |w|.  On top come its rounding of p (relative) and of the result:

* CUDA cores: scores are sums of D products in fp32, d <= (D + 8) 2^-24 of the sum of |products|, and the exponential of an argument of size s is
  off by 2^-22 + s 2^-23; sums of the p and p w add 2^-24 for each addition in a line.  All of it is covered by (D + 64) 2^-24 (1 + size).
* Tensor cores: operands of 11 significant bits: q times K2 is rounded once for the triple product, d <= 2^-11 of the sum of |products|; the
  dot-product sum has exact operands.  p is rounded to fp16: 2^-11 relative above its normal range, which with the scaling of the kernels
  ends 2^-24 below the largest p: for each of T^2 pairs at most 2^-24 times the largest |w| is lost.
"""
import math

import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from oracle import serving_oracle as orc

DEV = "cuda:0"
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _table(B, pages_each, pages, seed=0):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: B * pages_each].view(B, pages_each).int()


def _randn(*shape, seed, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


# ---------------------------------------------------------------- rows written and read back

def _rows(B, N, n, D, dtype, seed, strided):
    if strided:
        x = _randn(B, n, 4, N, D, seed=seed).to(dtype)
        return [x[:, :, i].transpose(1, 2) for i in range(4)]
    return [_randn(B, N, n, D, seed=seed + i).to(dtype) for i in range(4)]


WRITES = [  # B N n D dtype code page contexts counts strided
    (1, 1, 1, 64, "bf16", "e4m3", 16, [0], None, False),
    (3, 4, 21, 64, "fp16", "e4m3", 16, [0, 5, 40], [21, 1, 0], True),
    (2, 5, 9, 128, "bf16", "fp16", 16, [15, 16], None, True),
    (4, 3, 1, 128, "fp32", "int8", 64, [63, 64, 0, -1], None, False),
    (2, 2, 70, 32, "fp32", "fp16", 32, [3, 31], [70, 69], False),
    (1, 6, 33, 16, "fp16", "int8", 16, [2], None, True),
    (2, 3, 12, 256, "bf16", "int8", 128, [120, 0], [12, 99], True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,counts,strided", WRITES)
def test_written_rows(B, N, n, D, dtype, code, page, contexts, counts, strided):
    dt = TYPES[dtype]
    each = (max(contexts) + n + page - 1) // page
    pages = B * each + 2
    table = _table(B, each, pages)
    new = _rows(B, N, n, D, dt, 5, strided)
    cache = ft.new_cache(pages, page, N, D, orc.CODES[code], DEV)
    # what is there already stays
    cache.codes.view(torch.uint8).copy_(torch.randint(0, 100, cache.codes.view(torch.uint8).shape, generator=torch.Generator().manual_seed(1)))
    cache.exponents.fill_(77)
    before = [t.view(torch.uint8).cpu() for t in cache[:2]]
    ctx = torch.tensor(contexts, dtype=torch.int32)
    kw = dict(counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    ft.cache_write(cache, table.to(DEV), ctx.to(DEV), *(t.to(DEV) for t in new), **kw)
    back = ft.cache_read(cache, table.to(DEV), ctx.to(DEV), n, torch.float32, **kw)
    ft.check_status(DEV)
    after = [t.view(torch.uint8).cpu() for t in cache[:2]]
    exact = [new[0].double(), new[1].double(), orc.silu(new[2].double()), new[3].double()]
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for part, x in enumerate(exact):
        codes, byte, value = orc.quantise(x, code)
        step = {"fp16": 2.0 ** -10, "e4m3": 2.0 ** -3, "int8": 0.0}[code]   # (a SiLU within fp32's error of a border may be one code off)
        for b in range(B):
            used = 0 if contexts[b] < 0 else n if counts is None else min(n, counts[b])
            for i in range(n):
                got = back[part][b, :, i].double().cpu()
                if i >= used:
                    assert float(got.abs().max()) == 0
                    continue
                at = contexts[b] + i
                touched[table[b, at // page], at % page] = True
                if part != 2:
                    assert torch.equal(got, value[b, :, i])
                else:
                    # SiLU in fp32: its error (8 half steps of the exponential's argument and the quotient), then a rounding to the code's grid
                    grid = torch.exp2(byte[b, :, i].double() - 127).unsqueeze(-1) * ({"fp16": 2.0 ** -25, "e4m3": 2.0 ** -10, "int8": 0.5}[code])
                    bound = step / 2 * exact[2][b, :, i].abs() + grid + 2.0 ** -18 * exact[2][b, :, i].abs()
                    assert bool(((got - exact[2][b, :, i]).abs() <= bound).all())
    for a, b_, keep in zip(after, before, (touched, touched)):
        rest = ~keep
        assert torch.equal(a.transpose(1, 3)[rest] if a.dim() == 4 else a.permute(0, 3, 1, 2, 4)[rest],
                           b_.transpose(1, 3)[rest] if a.dim() == 4 else b_.permute(0, 3, 1, 2, 4)[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["fp16", "e4m3", "int8"])
def test_rows_at_the_codes_borders(code):
    """Largest elements just below, at and above a power of two times the codes' largest; zeros, subnormals, infinities, NaN."""
    x = torch.randn(1, 1, 16, 64, generator=torch.Generator().manual_seed(0))
    x = x / x.abs().amax(-1, keepdim=True)
    for i, top in enumerate([448.0, 448.0 * (1 + 2 ** -22), 448.0 * (1 - 2 ** -22), 127.0, 127.0 * (1 + 2 ** -22), 128.0, 2.0 ** 127, 2.0 ** -126,
                             2.0 ** -120, 1.0, 2.0 ** 15]):
        x[0, 0, i] *= top
        x[0, 0, i, 3] = top
    x[0, 0, 11] = 0
    x[0, 0, 12] *= 1e-42
    x[0, 0, 13, 9] = float("inf")
    x[0, 0, 14, 9] = float("nan")
    x[0, 0, 15, :] = -3.3e38
    cache = ft.new_cache(1, 16, 1, 64, orc.CODES[code], DEV)
    table, ctx = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ft.cache_write(cache, table, ctx, *(x.to(DEV),) * 4)
    back = ft.cache_read(cache, table, ctx, 16, torch.float32)
    _, byte, value = orc.quantise(x.double(), code)
    for part in (0, 1, 3):
        assert torch.equal(cache.exponents[0, part, 0].cpu(), byte[0, 0])
        # (a value below fp32's normal range may read as zero; -3.3e38 rounds to the 8-bit code -256 * 2^120 = -2^128, which fp32 does not have)
        got, want = back[part][0, 0].cpu().double(), value[0, 0].float().double()
        assert bool(((got == want) | (want.abs() < 2.0 ** -126) & (got == 0) | torch.isnan(got) & torch.isnan(want)).all())
    ft.check_status(DEV)


# ---------------------------------------------------------------- attention over the cache

class Batch:
    def __init__(self, B, N, n, D, dtype, code, page, contexts, dps=False, scale=1.0, seed=0, parents=None, strided=True):
        self.B, self.N, self.n, self.D, self.contexts, self.dt, self.code = B, N, n, D, contexts, TYPES[dtype], code
        each = max(1, (max(contexts) + n + page - 1) // page)
        pages = B * each + 1
        table = _table(B, each, pages, seed)
        parts = []
        for b in range(B):
            x = _randn(4, N, max(0, contexts[b]) + n, D, seed=seed + 10 * b, scale=scale).double()
            x[2] = orc.silu(x[2])
            parts.append(x)
        lse = [_randn(N, max(0, c) + n, seed=seed + 7 + b).double() + 2 for b, c in enumerate(contexts)] if dps else None
        self.seq = orc.Sequences(parts, code, page, pages, table, lse)
        self.cache = ft.TrittentionCache(self.seq.codes.to(DEV), self.seq.exponents.to(DEV), None if lse is None else self.seq.lse.to(DEV))
        self.table, self.context = table.to(DEV), torch.tensor(contexts, dtype=torch.int32, device=DEV)
        self.words = None if parents is None else ft.tree_ancestors(parents)
        self.ancestors = None if parents is None else self.words.to(DEV).expand(B, n).contiguous()
        q = _randn(B, n, 3, N, D, seed=seed + 99).to(self.dt)
        self.q = q[:, :, 1].transpose(1, 2) if strided else q[:, :, 1].transpose(1, 2).contiguous()

    def rows(self):
        for b in range(self.B):
            for h in range(self.N):
                for i in range(self.n):
                    yield b, h, i


def _score_error(D, size, fast, triple):
    """Largest error of a score, in natural-log units, from the sum of its products' absolute values."""
    return (D + 64) * 2.0 ** -24 * (1 + size) + (2.0 ** -11 * size if fast and triple else 0.0)


def _check_result(got, lse, ref, dt, D, pairs, fast, triple, where):
    o, want_lse, mass, size = ref
    d = _score_error(D, float(size), fast, triple)
    wmax = float(mass.max())
    bound = HALF_STEP[dt] * o.abs() + (math.expm1(2 * d) + (2.0 ** -10 if fast else 0)) * (mass + o.abs()) + (pairs * 2.0 ** -24 * 2.0 ** -10 * wmax if fast else 0) + 1e-30
    if dt == torch.float16:
        bound = bound + 2.0 ** -25
    # a result that the type does not have (fp16: from 65520 on, which rounds to infinity) is infinite
    got = got.double().cpu()
    over = torch.isinf(got) & (got.sign() == o.sign()) & (o.abs() + bound >= torch.finfo(dt).max * (1 + HALF_STEP[dt] / 2))
    err = torch.where(over, torch.zeros_like(o), (got - o).abs())
    assert bool((err <= bound).all()), f"{where}: off by {float(err.max()):.3e}, bound {float(bound[err.argmax()]):.3e}"
    if lse is not None:
        if want_lse == -math.inf:
            assert float(lse) == -math.inf, where
        else:
            assert abs(float(lse) - float(want_lse)) <= d + 2.0 ** -22 * (1 + abs(float(want_lse))), f"{where}: {float(lse)} {float(want_lse)}"


def _tree(n, branch):
    return [-1 if i == 0 else (i - 1) // branch for i in range(n)]


TDP = [  # B N n D dtype code page contexts windows parents precision
    (1, 1, 1, 64, "fp16", "e4m3", 16, [0], (None,) * 4, None),
    (3, 2, 1, 64, "bf16", "fp16", 16, [1, 40, -1], (None,) * 4, None),
    (2, 3, 5, 64, "fp16", "int8", 32, [37, 130], (None,) * 4, None),
    (2, 2, 7, 64, "bf16", "e4m3", 16, [150, 33], (None,) * 4, _tree(7, 2)),
    (2, 1, 9, 128, "fp16", "fp16", 64, [140, 0], (20, 50, 10, 3), _tree(9, 3)),
    (1, 2, 4, 128, "bf16", "int8", 16, [260], (128, 128, 32, 32), None),
    (1, 1, 3, 64, "fp16", "fp16", 16, [300], (None, 0, None, None), [-1, 0, 0]),
    (1, 1, 3, 64, "fp16", "e4m3", 16, [200], (0, None, None, 0), None),
    (1, 2, 2, 64, "bf16", "fp16", 256, [257], (None, None, 0, 0), None),
    (2, 1, 2, 128, "bf16", "e4m3", 128, [129, 127], (60, None, None, 40), None),
    (1, 1, 2, 32, "fp16", "e4m3", 16, [30], (None,) * 4, None),
    (2, 2, 3, 64, "fp32", "fp16", 16, [20, 31], (15, None, 8, None), [-1, -1, 1]),
    (1, 1, 1, 256, "bf16", "int8", 16, [25], (None,) * 4, None),
    (1, 1, 66, 64, "bf16", "fp16", 16, [10], (None,) * 4, None),
]


def _tdp_check(bt, out, lse, windows, alpha, fast, counts=None, heads=None):
    for b, h, i in bt.rows():
        ctx = bt.contexts[b]
        if heads is not None and h not in heads:
            continue
        here = ctx >= 0 and (counts is None or i < counts[b])
        x = bt.seq.values[b][:, h]
        ref = orc.tdp_row(bt.q[b, h, i].double(), x[0], x[1], x[2], x[3], ctx, i, alpha, windows, bt.words) if here else (
            torch.zeros(bt.D).double(), torch.tensor(-math.inf), torch.zeros(bt.D).double(), torch.tensor(0.0))
        _check_result(out[b, h, i], None if lse is None else lse[b, h, i], ref, bt.dt, bt.D, (ctx + bt.n) ** 2, fast, True, (b, h, i))


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,windows,parents", TDP)
def test_tdp_decode(B, N, n, D, dtype, code, page, contexts, windows, parents, precision):
    bt = Batch(B, N, n, D, dtype, code, page, contexts, parents=parents)
    alpha = 1 / math.sqrt(D)
    fast = precision is None and _native.decode_path(_native.OP_TDP_DECODE, D, _native.dtype_code(bt.dt)) == _native.PATH_TCGEN05
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, *windows, ancestors=bt.ancestors, return_lse=True,
                             input_precision=precision)
    ft.check_status(DEV)
    _tdp_check(bt, out, lse, windows, alpha, fast)
    assert torch.equal(out, ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, *windows, ancestors=bt.ancestors,
                                          input_precision=precision))


LONG = [  # B N n D dtype code page contexts windows parents: what does not fit in shared memory, and a table much longer than its sequences
    (1, 1, 1, 64, "fp16", "e4m3", 16, [1500], (None,) * 4, None),
    (1, 2, 2, 64, "bf16", "int8", 64, [2047], (None,) * 4, None),
    (3, 1, 1, 64, "fp16", "fp16", 32, [640, -1, 0], (None,) * 4, None),
    (2, 1, 9, 64, "bf16", "fp16", 32, [640, 5], (500, 600, 100, 50), _tree(9, 3)),
    (1, 1, 40, 64, "fp16", "e4m3", 64, [470], (30, None, 8, None), _tree(40, 2)),
    (1, 1, 130, 64, "bf16", "e4m3", 16, [400], (None,) * 4, None),
    (1, 1, 3, 64, "fp16", "fp16", 16, [1030], (None, 0, None, None), [-1, 0, 0]),
    (1, 1, 2, 64, "fp16", "e4m3", 16, [900], (0, None, None, 0), None),
    (1, 2, 2, 64, "bf16", "fp16", 256, [1000], (None, None, 0, 0), None),
    (1, 2, 7, 128, "fp16", "e4m3", 16, [515], (None, 40, None, None), _tree(7, 2)),
    (1, 1, 2, 128, "bf16", "fp16", 256, [1023], (None,) * 4, None),
    (4, 1, 1, 128, "fp16", "int8", 16, [300, -1, 0, 129], (None,) * 4, None),
    (2, 1, 5, 128, "bf16", "e4m3", 16, [700, 31], (300, 400, 64, 90), [-1, 0, 1, 0, 3]),
    (1, 1, 64, 128, "fp16", "fp16", 128, [250], (200, 1000, None, 100), _tree(64, 1)),
    (40, 3, 1, 64, "fp16", "e4m3", 16, [(37 * b) % 600 - 1 for b in range(40)], (None,) * 4, None),
]


def _widened(table, tokens, page):
    """The table with places for ``tokens`` tokens, the new ones of no page."""
    more = torch.full((table.shape[0], max(0, tokens // page - table.shape[1])), -1, dtype=torch.int32, device=table.device)
    return torch.cat([table, more], 1)


def _kernel_of_windows(bt, table, windows):
    c, keep = ft.cache._describe(bt.cache, table, bt.context, bt.n, None, bt.ancestors)
    w = [1 << 30 if x is None else x for x in windows[:2]]
    return _native.lib().tritt_decode_workspace(_native.OP_TDP_DECODE, _native.C.byref(c), _native.dtype_code(bt.dt), *w, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e-3])
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,windows,parents", LONG)
def test_tdp_decode_of_long_sequences(B, N, n, D, dtype, code, page, contexts, windows, parents, size):
    """The kernel that forms the products of all pairs' tiles.  Its p are at most 2^15 and rounded to fp16: 2^-11 relative, and of a pair below 2^-21
    of the largest 2^-32 of the largest.  With queries of 0.001 the log-sum-exp counts the attended pairs."""
    bt = Batch(B, N, n, D, dtype, code, page, contexts, parents=parents, seed=11)
    bt.q = bt.q * size
    alpha = 1 / math.sqrt(D)
    table = _widened(bt.table, 4096, page)
    assert not _kernel_of_windows(bt, table, windows)
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, *windows, ancestors=bt.ancestors, return_lse=True)
    ft.check_status(DEV)
    again = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, *windows, ancestors=bt.ancestors)
    assert torch.equal(out, again)
    for b, h, i in bt.rows():
        if (b * 7 + h * 5 + i * 3) % max(1, B * N * n // 24):   # (some two dozen rows of each case)
            continue
        where, ctx, x = (b, h, i), bt.contexts[b], bt.seq.values[b][:, h]
        if ctx < 0:
            assert float(out[b, h, i].abs().max()) == 0 and float(lse[b, h, i]) == -math.inf
            continue
        args = (bt.q[b, h, i].double(), x[0], x[1], x[2], x[3], ctx, i, alpha, windows, bt.words)
        o, want, mass, scores = orc.tdp_row(*args)
        d = _score_error(D, float(scores), True, True)
        bound = HALF_STEP[bt.dt] * o.abs() + (math.expm1(2 * d) + 2.0 ** -10) * (mass + o.abs()) + 2.0 ** -32 * orc.tdp_small(*args, 2.0 ** -20) + 2.0 ** -25
        err = (out[b, h, i].double().cpu() - o).abs()
        assert bool((err <= bound).all()), f"{where}: off by {float(err.max()):.3e}, bound {float(bound[err.argmax()]):.3e}"
        assert abs(float(lse[b, h, i]) - float(want)) <= d + 2.0 ** -22 * (1 + abs(float(want))), (where, float(lse[b, h, i]), float(want))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_sequences_under_a_long_table(D):
    """Pieces of a slab or none, with one tile and with two, behind one another: every run the same bits."""
    bt = Batch(40, 3, 1, D, "bf16", "int8", 16, [(37 * b) % 300 - 1 for b in range(40)], seed=19)
    table, q = _widened(bt.table, 4096, 16), bt.q.to(DEV)
    outs = [ft.tdp_decode(q, bt.cache, table, bt.context, 0.1, return_lse=True) for _ in range(60)]
    ft.check_status(DEV)
    assert all(torch.equal(o, outs[0][0]) and torch.equal(m, outs[0][1]) for o, m in outs)
    _tdp_check(bt, *outs[0], (None,) * 4, 0.1, True, heads=(1,))


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,windows,parents", TDP[:10])
def test_tdp_decode_under_a_long_table(B, N, n, D, dtype, code, page, contexts, windows, parents):
    """A table of more places than are in use takes another kernel where windows do not bound the tokens: the same definitions."""
    bt = Batch(B, N, n, D, dtype, code, page, contexts, parents=parents)
    alpha, table = 1 / math.sqrt(D), _widened(bt.table, 8192, page)
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, *windows, ancestors=bt.ancestors, return_lse=True)
    ft.check_status(DEV)
    _tdp_check(bt, out, lse, windows, alpha, True)


DPS_LONG = [  # B N n D dtype code page contexts k_diff parents
    (1, 1, 1, 64, "fp16", "e4m3", 16, [9000], 1 << 20, None),
    (40, 3, 1, 64, "bf16", "int8", 16, [(137 * b) % 2500 - 1 for b in range(40)], 1024, None),
    (2, 2, 24, 128, "fp16", "fp16", 64, [3001, 64], 5000, _tree(24, 2)),
    (2, 1, 33, 64, "bf16", "e4m3", 256, [2000, 700], 900, _tree(33, 3)),
    (1, 1, 100, 128, "bf16", "e4m3", 16, [1500], 1024, None),
    (1, 1, 300, 64, "fp16", "int8", 16, [800], 333, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e-3])
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,k_diff,parents", DPS_LONG)
def test_dps_decode_of_long_sequences(B, N, n, D, dtype, code, page, contexts, k_diff, parents, size):
    bt = Batch(B, N, n, D, dtype, code, page, contexts, dps=True, parents=parents, seed=13)
    bt.q = bt.q * size
    alpha, table = 1 / math.sqrt(D), _widened(bt.table, 16384, page)
    out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, ancestors=bt.ancestors)
    ft.check_status(DEV)
    _dps_check(bt, out, m, alpha, True)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,k_diff,parents", DPS_LONG)
def test_dps_append_counts_the_tokens_of_long_sequences(B, N, n, D, dtype, code, page, contexts, k_diff, parents):
    """Keys of zeros make every score zero: the log-sum-exp is the logarithm of how many tokens are attended to, W their values' mean times V2."""
    bt = Batch(B, N, n, D, dtype, code, page, contexts, dps=True, parents=parents, seed=17)
    x = torch.ones(B, N, n, D, device=DEV, dtype=bt.dt)
    ft.dps_append(bt.cache, _widened(bt.table, 16384, page), bt.context, x * 0, x * 0, x, x, 0.1, k_diff, ancestors=bt.ancestors)
    back = ft.cache_read(bt.cache, bt.table, bt.context, n, torch.float32)
    ft.check_status(DEV)
    gated = back[2].double().cpu()
    grid = {"fp16": 2.0 ** -11, "e4m3": 2.0 ** -4, "int8": 2.0 ** -7}[code]
    for b, h, i in bt.rows():
        ctx = contexts[b]
        if ctx < 0:
            continue
        val = bt.seq.values[b][2, h].clone()
        val[ctx:] = gated[b, h]
        zero = torch.zeros(ctx + n, D, dtype=torch.float64)
        y, lse, mass, _ = orc.dps_row(zero[0], zero, val, None, ctx, i, 0.1, k_diff, bt.words)
        assert abs(float(back[4][b, h, i]) - float(lse)) <= 2.0 ** -22 * (1 + float(lse)), (b, h, i)
        err = 2.0 ** -10 * mass                      # p = 1 is exact: what is left is the sums' and the code's rounding
        got, top = back[3][b, h, i].double().cpu(), float((y.abs() + err).max())
        rounding = (grid * y.abs() if code != "int8" else 0) + {"fp16": 2.0 ** -24, "e4m3": 2.0 ** -17, "int8": 2.0 ** -7}[code] * top
        assert bool(((got - y).abs() <= err * (1 + 2 * grid) + rounding + 1e-30).all()), (b, h, i)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_long_sequences_with_bad_rows_missing_places_and_padding(D):
    """NaN rows reach those that attend to them; a missing page is reported, its tokens left out; rows past a count and free slots are empty."""
    parents = [-1, 0, 0, 1]
    bt = Batch(3, 2, 4, D, "fp16", "e4m3", 16, [550, 550, -1], parents=parents, seed=5)
    table = _widened(bt.table, 4096, 16)
    counts = torch.tensor([4, 3, 4], dtype=torch.int32, device=DEV)
    ask = lambda t, *w: ft.tdp_decode(bt.q.to(DEV), bt.cache, t, bt.context, 0.1, *w, ancestors=bt.ancestors, counts=counts, return_lse=True)  # noqa: E731
    clean, clean_lse = ask(table, 500, 500)
    ft.check_status(DEV)
    empty = torch.zeros(3, 2, 4, dtype=torch.bool, device=DEV)
    empty[1, :, 3] = empty[2] = True
    assert not bool(clean[empty].any()) and bool((clean_lse[empty] == -math.inf).all()) and bool(torch.isfinite(clean_lse[~empty]).all())
    place = lambda t, part: (bt.table[0, t // 16].long(), part, 0, t % 16)  # noqa: E731
    for part in range(4):
        held = [(place(t, part), bt.cache.exponents[place(t, part)].clone()) for t in (551, 300, 30)]
        bt.cache.exponents[held[0][0]] = 255     # new token 1: tokens 1 and 3 attend to it
        bt.cache.exponents[held[2][0]] = 255     # behind every window of 500
        out, lse = ask(table, 500, 500)
        hit = torch.zeros_like(empty)
        hit[0, 0, 1] = hit[0, 0, 3] = True
        assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit]), part
        if part < 2:
            assert bool(torch.isnan(lse[hit]).all()), part
        bt.cache.exponents[held[1][0]] = 255     # in everyone's window
        hit[0, 0] = True
        out, lse = ask(table, 500, 500)
        assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit]), part
        for at, was in held:
            bt.cache.exponents[at] = was
    ft.check_status(DEV)
    assert torch.equal(ask(table, 500, 500)[0], clean)
    for page in (5000, -1, 1 << 30):
        bad = table.clone()
        bad[0, 10] = page                        # tokens 160 .. 175
        out, lse = ask(bad, 500, 500)
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        assert torch.equal(out[1:], clean[1:]) and bool(torch.isfinite(out).all())
        # the pairs that are left count: with queries of zeros the log-sum-exp is their number's logarithm
        _, lse = ft.tdp_decode(torch.zeros_like(bt.q).to(DEV), bt.cache, bad, bt.context, 0.1, counts=counts, return_lse=True)
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        for i in range(4):
            assert abs(float(lse[0, 0, i]) - 2 * math.log(550 + i + 1 - 16)) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kernels_at_the_border_between_them(D):
    """Windows on either side of what fits in shared memory give the same rows up to each kernel's own error, whichever kernel runs."""
    bt = Batch(1, 2, 3, D, "bf16", "fp16", 16, [600], seed=3)
    table, seen = _widened(bt.table, 4096, 16), set()
    for w in (40, 100, 128, 160, 200, 256, 300, 350, 400, 450, 500, 599):
        windows = (w, w, None, None)
        seen.add(_kernel_of_windows(bt, table, windows))
        out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, 0.1, *windows, return_lse=True)
        _tdp_check(bt, out, lse, windows, 0.1, True)
    assert seen == {False, True}
    ft.check_status(DEV)


@pytest.mark.gpu
def test_long_sequences_in_graphs_and_on_another_stream():
    bts = [Batch(2, 2, 3, 64, "bf16", "e4m3", 16, [790, 340], dps=True, seed=s) for s in (0, 50)]
    tables = [_widened(bt.table, 4096, 16) for bt in bts]

    def step(bt, table):
        ft.dps_append(bt.cache, table, bt.context, bt.q, bt.q, bt.q, bt.q, 0.125, 64)
        return [*ft.dps_decode(bt.q, bt.cache, table, bt.context, 0.125), ft.tdp_decode(bt.q, bt.cache, table, bt.context, 0.125)]

    for bt in bts:
        bt.q = bt.q.to(DEV)
    want = [[t.clone() for t in step(*x)] for x in zip(bts, tables)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in bts], [], []
    torch.cuda.synchronize()
    for bt, table, s in zip(bts, tables, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(bt, table))
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for bt in bts:
        bt.context.sub_(300)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for bt, table, b in zip(bts, tables, outs):
        assert all(torch.equal(x, y) for x, y in zip(step(bt, table), b))
    ft.check_status(DEV)


DPS = [  # B N n D dtype code page contexts k_diff parents
    (1, 1, 1, 64, "fp16", "e4m3", 16, [0], 1024, None),
    (3, 2, 1, 64, "bf16", "fp16", 16, [1, 40, -1], 1024, None),
    (4, 3, 1, 64, "bf16", "e4m3", 64, [63, 64, 65, 1000], 500, None),
    (2, 3, 5, 64, "fp16", "int8", 32, [37, 530], 100, None),
    (2, 2, 7, 64, "bf16", "e4m3", 16, [150, 33], 10, _tree(7, 2)),
    (2, 1, 9, 128, "fp16", "fp16", 64, [140, 0], 1024, _tree(9, 3)),
    (1, 2, 17, 128, "bf16", "int8", 16, [260], 0, None),
    (1, 2, 33, 64, "bf16", "fp16", 256, [257], 5000, _tree(33, 2)),
    (1, 1, 64, 128, "fp16", "e4m3", 16, [100], 64, _tree(64, 1)),
    (1, 1, 130, 64, "fp16", "fp16", 16, [10], 40, None),
    (1, 1, 2, 32, "fp16", "e4m3", 16, [30], 1024, None),
    (2, 2, 3, 64, "fp32", "fp16", 16, [20, 31], 1024, [-1, -1, 1]),
    (1, 1, 1, 256, "bf16", "int8", 16, [25], 8, None),
]


def _dps_check(bt, out, m, alpha, fast, counts=None):
    for b, h, i in bt.rows():
        ctx = bt.contexts[b]
        here = ctx >= 0 and (counts is None or i < counts[b])
        x = bt.seq.values[b][:, h]
        ref = orc.dps_row(bt.q[b, h, i].double(), x[1], x[3], bt.seq.bias[b][h], ctx, i, alpha, None, bt.words) if here else (
            torch.zeros(bt.D).double(), torch.tensor(-math.inf), torch.zeros(bt.D).double(), torch.tensor(0.0))
        _check_result(out[b, h, i], m[b, h, i], ref, bt.dt, bt.D, ctx + bt.n, fast, False, (b, h, i))


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,k_diff,parents", DPS)
def test_dps_decode(B, N, n, D, dtype, code, page, contexts, k_diff, parents, precision):
    bt = Batch(B, N, n, D, dtype, code, page, contexts, dps=True, parents=parents)
    alpha = 1 / math.sqrt(D)
    fast = precision is None and _native.decode_path(_native.OP_DPS_DECODE, D, _native.dtype_code(bt.dt)) == _native.PATH_TCGEN05
    out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, ancestors=bt.ancestors, input_precision=precision)
    ft.check_status(DEV)
    _dps_check(bt, out, m, alpha, fast)
    again = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, ancestors=bt.ancestors, input_precision=precision)
    assert torch.equal(out, again[0]) and torch.equal(m, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,k_diff,parents", DPS)
def test_dps_append(B, N, n, D, dtype, code, page, contexts, k_diff, parents, precision):
    bt = Batch(B, N, n, D, dtype, code, page, contexts, dps=True, parents=parents)
    alpha = 1 / math.sqrt(D)
    fast = precision is None and _native.decode_path(_native.OP_DPS_APPEND, D, _native.dtype_code(bt.dt)) == _native.PATH_TCGEN05
    x = _randn(B, n, 4, N, D, seed=77).to(bt.dt)
    k1, k2, v1, v2 = (x[:, :, i].transpose(1, 2) for i in range(4))
    before = [t.clone() for t in bt.cache]
    ft.dps_append(bt.cache, bt.table, bt.context, *(t.to(DEV) for t in (k1, k2, v1, v2)), alpha, k_diff, ancestors=bt.ancestors,
                  input_precision=precision)
    back = ft.cache_read(bt.cache, bt.table, bt.context, n, torch.float32)
    ft.check_status(DEV)
    held = [orc.quantise(t.double(), bt.code)[2] for t in (k1, k2)]
    gated = back[2].double().cpu()   # (SiLU's codes as they are: test_written_rows has them)
    touched = torch.zeros(before[0].shape[0], before[0].shape[3], dtype=torch.bool)
    grid = {"fp16": 2.0 ** -11, "e4m3": 2.0 ** -4, "int8": 2.0 ** -7}[bt.code]
    for b, h, i in bt.rows():
        ctx = bt.contexts[b]
        if ctx < 0:
            assert float(back[3][b, h, i].abs().max()) == 0
            continue
        at = ctx + i
        touched[bt.table[b, at // bt.seq.page_size].cpu(), at % bt.seq.page_size] = True
        assert torch.equal(back[0][b, h, i].double().cpu(), held[0][b, h, i]) and torch.equal(back[1][b, h, i].double().cpu(), held[1][b, h, i])
        key, val = bt.seq.values[b][0, h].clone(), bt.seq.values[b][2, h].clone()
        key[ctx:], val[ctx:] = held[0][b, h], gated[b, h]
        y, lse, mass, size = orc.dps_row(k2[b, h, i].double(), key, val, None, ctx, i, alpha, k_diff, bt.words)
        w, mass = y * v2[b, h, i].double(), mass * v2[b, h, i].double().abs()
        d = _score_error(D, float(size), fast, False)
        err = (math.expm1(2 * d) + (2.0 ** -10 if fast else 0)) * (mass + w.abs())
        top = float((w.abs() + err).max())
        # a code's rounding: relative, but for int8 and the smallest codes, which count from the row's largest element
        rounding = (grid * w.abs() if bt.code != "int8" else 0) + {"fp16": 2.0 ** -24, "e4m3": 2.0 ** -17, "int8": 2.0 ** -7}[bt.code] * top
        bad = (back[3][b, h, i].double().cpu() - w).abs() - (err * (1 + 2 * grid) + rounding + 1e-30)
        assert float(bad.max()) <= 0, (b, h, i, float(bad.max()))
        assert abs(float(back[4][b, h, i]) - float(lse)) <= d + 2.0 ** -22 * (1 + abs(float(lse)))
    rest = ~touched.to(DEV)
    for new, old in zip(bt.cache, before):
        new, old = new.view(torch.uint8), old.view(torch.uint8)
        if new.dim() == 3:   # lse: [pages, N, rows * 4 bytes]
            new, old = (t.unflatten(2, (-1, 4)).transpose(1, 2) for t in (new, old))
        else:
            new, old = (t.movedim(3, 1) for t in (new, old))
        assert torch.equal(new[rest], old[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
def test_padded_batches_and_free_slots(precision):
    bt = Batch(4, 2, 6, 64, "bf16", "fp16", 16, [30, 0, -1, 100], dps=True)
    counts = [6, 2, 6, 0]
    ct = torch.tensor(counts, dtype=torch.int32, device=DEV)
    out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, counts=ct, input_precision=precision)
    _dps_check(bt, out, m, 0.1, precision is None, counts)
    out, m = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, counts=ct, return_lse=True, input_precision=precision)
    _tdp_check(bt, out, m, (None,) * 4, 0.1, precision is None, counts)
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_are_not_finite_reach_those_that_attend(precision, D):
    """A NaN row (exponent 255) makes the results of the tokens that attend to it NaN, and no others: not those whose window, tree or order
    leaves it out."""
    parents = [-1, 0, 0, 1]
    for part in range(4):
        bt = Batch(2, 2, 4, D, "fp16", "e4m3", 16, [150, 150], dps=True, parents=parents)
        clean = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, 100, 100, ancestors=bt.ancestors, input_precision=precision)
        free, _ = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, ancestors=bt.ancestors, input_precision=precision)
        place = lambda t: (bt.table[0, t // 16].long(), part, 0, t % 16)  # noqa: E731
        bt.cache.exponents[place(151)] = 255     # new token 1 of sequence 0, head 0: tokens 1 and 3 attend to it
        bt.cache.exponents[place(40)] = 255      # behind every window of 100
        out = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, 100, 100, ancestors=bt.ancestors, input_precision=precision)
        hit = torch.zeros(2, 2, 4, dtype=torch.bool, device=DEV)
        hit[0, 0, 1] = hit[0, 0, 3] = True
        assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])
        out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, ancestors=bt.ancestors, input_precision=precision)
        if part in (1, 3):
            hit[0, 0] = True   # (token 40 is in everyone's context)
            assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], free[~hit])
        else:
            assert torch.equal(out, free)
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
def test_places_that_there_are_not(precision):
    """A page that the cache does not have, and tokens past the table: reported, not read or written; the rest of the row's tokens count."""
    bt = Batch(1, 1, 2, 64, "fp16", "fp16", 16, [60], dps=True)
    good = bt.table.clone()
    for page in (1000, -1, 1 << 30):
        bt.table[0, 1] = page
        before = [t.clone() for t in bt.cache]
        out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, input_precision=precision)
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        assert bool(torch.isfinite(out).all())
        for i in range(2):
            x, bias = bt.seq.values[0][:, 0], bt.seq.bias[0][0].clone()
            bias[16:32] = -1e300
            ref = orc.dps_row(bt.q[0, 0, i].double(), x[1], x[3], bias, 60, i, 0.1)
            assert float((out[0, 0, i].double().cpu() - ref[0]).abs().max()) < 2e-3
        assert bool(torch.isfinite(ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, input_precision=precision)).all())
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        ctx = torch.tensor([30], dtype=torch.int32, device=DEV)
        x = torch.ones(1, 1, 2, 64, device=DEV, dtype=torch.float16)
        ft.cache_write(bt.cache, bt.table, ctx, x, x, x, x)          # tokens 30 and 31: on the missing page
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        back = ft.cache_read(bt.cache, bt.table, ctx, 4, torch.float32)   # 30, 31 missing, 32 and 33 there
        with pytest.raises(_native.TrittError, match="place"):
            ft.check_status(DEV)
        assert float(back[0][0, 0, :2].abs().max()) == 0 and float(back[0][0, 0, 2:].abs().min()) >= 0 and float(back[0][0, 0, 2:].abs().max()) > 0
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(bt.cache, before))
    bt.table.copy_(good)
    past = torch.tensor([bt.table.shape[1] * 16 - 1], dtype=torch.int32, device=DEV)   # the second new token is past the table
    before = [t.clone() for t in bt.cache]
    x = torch.full((1, 1, 2, 64), 2.0, device=DEV, dtype=torch.float16)
    ft.dps_append(bt.cache, bt.table, past, x, x, x, x, input_precision=precision)
    with pytest.raises(_native.TrittError, match="place"):
        ft.check_status(DEV)
    changed = sum(int((a.view(torch.uint8) != b.view(torch.uint8)).any(-1).sum()) for a, b in zip(bt.cache[:1], before[:1]))
    assert changed <= 4


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("scale", [1e-3, 6.0])
def test_small_and_large_scores(scale, precision):
    """Rows of 0.001 (soft-max of equals) and of 6 (one pair carries almost all)."""
    for D in (64, 128):
        bt = Batch(1, 2, 3, D, "bf16", "fp16", 16, [140], dps=True, scale=scale)
        a = 1 / math.sqrt(D)
        fast = precision is None
        out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, a, return_lse=True, input_precision=precision)
        _tdp_check(bt, out, lse, (None,) * 4, a, fast)
        out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, a, input_precision=precision)
        _dps_check(bt, out, m, a, fast)
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["fp16", "e4m3", "int8"])
def test_rows_of_very_different_sizes(code):
    """Rows whose exponents differ by up to 2^40 within one tile, and rows of zeros."""
    bt = Batch(1, 2, 2, 64, "fp16", code, 16, [200], dps=True)
    shift = torch.randint(-20, 21, bt.seq.exponents.shape, generator=torch.Generator().manual_seed(3))
    shift[:, :2] = shift[:, :2].clamp(max=0)    # (keys only smaller: scores stay moderate)
    byte = (bt.seq.exponents.int() + shift).clamp(1, 254).to(torch.uint8)
    bt.seq.exponents.copy_(byte)
    bt.cache.exponents.copy_(byte)
    page = bt.seq.page_size
    for t in range(202):
        p = int(bt.table[0, t // page])
        codes = bt.seq.codes[p, :, :, t % page]
        bt.seq.values[0][:, :, t] = orc.values(codes, byte[p, :, :, t % page])
    out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1)
    _dps_check(bt, out, m, 0.1, True)
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, 0.1, return_lse=True)
    _tdp_check(bt, out, lse, (None,) * 4, 0.1, True)
    ft.check_status(DEV)


# ---------------------------------------------------------------- as a program uses them

def _against_whole(dps, code, tol):
    """A sequence token by token, and in chunks, against the whole-sequence kernels."""
    B, N, T, D = 2, 2, 48, 64
    xs = [(_randn(B, N, T, D, seed=i) * 0.7).to(DEV, torch.float16) for i in range(5)]
    q, k1, k2, v1, v2 = xs
    if dps:
        whole, m_whole = ft.TrittentionTriton(softmax_scale=0.125, k_diff=20)(*xs)
    else:
        whole = ft.flash_trittention(*xs, softmax_scale=0.125, k1_window=30, k2_window=None, kk_left=None, kk_right=25)
    table = _table(B, 3, 7).to(DEV)
    for steps in ([1] * T, [13, 1, 20, 14]):
        cache = ft.new_cache(7, 16, N, D, code, DEV, dps=dps)
        at, got = 0, []
        for n in steps:
            ctx = torch.full((B,), at, dtype=torch.int32, device=DEV)
            new = [t[:, :, at: at + n] for t in xs]
            if dps:
                ft.dps_append(cache, table, ctx, *new[1:], 0.125, 20)
                got.append(ft.dps_decode(new[0], cache, table, ctx, 0.125)[0])
            else:
                ft.cache_write(cache, table, ctx, *new[1:])
                got.append(ft.tdp_decode(new[0], cache, table, ctx, 0.125, 30, None, None, 25))
            at += n
        err = (torch.cat(got, 2).float() - whole.float()).norm() / whole.float().norm()
        assert float(err) < tol, float(err)
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dps", [False, True])
def test_token_by_token_against_the_whole_sequence(dps):
    # fp16 codes: nothing of fp16 tensors is lost but SiLU's and W's rounding (2^-11 each, as the whole-sequence kernels round them too)
    _against_whole(dps, torch.float16, 5e-3)
    # e4m3: four rows of a product, each rounded to 2^-4 at most (rms 0.026 each)
    _against_whole(dps, torch.float8_e4m3fn, 0.15)


@pytest.mark.gpu
@pytest.mark.parametrize("dps", [False, True])
def test_drafts_verified_and_written_again(dps):
    """A tree of drafts gives each of its paths what that path gives as a chain; the accepted path, written again, is the new context."""
    B, N, D, n = 2, 3, 64, 7
    parents = [-1, 0, 0, 1, 1, 2, 4]
    words = ft.tree_ancestors(parents, DEV).expand(B, n).contiguous()
    table = _table(B, 4, 9).to(DEV)
    ctx = torch.tensor([25, 14], dtype=torch.int32, device=DEV)
    base = ft.new_cache(9, 16, N, D, torch.float16, DEV, dps=dps)
    old = [(_randn(B, N, 25, D, seed=i)).to(DEV, torch.float16) for i in range(4)]
    start = torch.zeros(B, dtype=torch.int32, device=DEV)
    new = [(_randn(B, N, n, D, seed=20 + i)).to(DEV, torch.float16) for i in range(5)]
    add = (lambda c, t, x, **kw: ft.dps_append(c, table, t, *x, **kw)) if dps else (
        lambda c, t, x, ancestors=None, **kw: ft.cache_write(c, table, t, *x, **kw))
    ask = (lambda q, c, **kw: ft.dps_decode(q, c, table, ctx, **kw)[0]) if dps else (lambda q, c, **kw: ft.tdp_decode(q, c, table, ctx, **kw))
    add(base, start, old, counts=ctx)
    tree = ft.TrittentionCache(*(None if t is None else t.clone() for t in base))
    add(tree, ctx, new[1:], ancestors=words)
    got = ask(new[0], tree, ancestors=words)
    for path in ([0, 1, 4, 6], [0, 2, 5], [0, 1, 3]):
        chain = ft.TrittentionCache(*(None if t is None else t.clone() for t in base))
        part = [t[:, :, path] for t in new]
        add(chain, ctx, part[1:])
        want = ask(part[0], chain)
        # (the same sums in another order: fp16's rounding of p and of the result)
        assert float((got[:, :, path].float() - want.float()).abs().max()) < 4e-3
        add(tree, ctx, part[1:])   # the accepted path over the drafts
        assert torch.equal(ask(part[0], tree), want)
        add(tree, ctx, new[1:], ancestors=words)
    ft.check_status(DEV)


@pytest.mark.gpu
def test_graphs_that_run_at_once_and_another_stream():
    bts = [Batch(2, 4, 3, 64, "bf16", "e4m3", 16, [90, 140], dps=True, seed=s) for s in (0, 50)]

    def step(bt):
        q = bt.q.to(DEV) if not bt.q.is_cuda else bt.q
        ft.dps_append(bt.cache, bt.table, bt.context, q, q, q, q, 0.125, 64)
        return [*ft.dps_decode(q, bt.cache, bt.table, bt.context, 0.125), ft.tdp_decode(q, bt.cache, bt.table, bt.context, 0.125)]

    for bt in bts:
        bt.q = bt.q.to(DEV)
    want = [[t.clone() for t in step(bt)] for bt in bts]
    streams, graphs, outs = [torch.cuda.Stream() for _ in bts], [], []
    torch.cuda.synchronize()
    for bt, s in zip(bts, streams):
        with torch.cuda.stream(s):
            step(bt)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(bt))
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the context moves on without a new capture
    for bt in bts:
        bt.context.sub_(40)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for bt, b in zip(bts, outs):
        assert all(torch.equal(x, y) for x, y in zip(step(bt), b))
    ft.check_status(DEV)


HOST = ("host_norm_rotary", "host_norm_rotary_backward", "host_cache_write", "host_cache_read", "host_decode")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tree", [False, True])
def test_calls_by_the_extension_and_by_the_python_code(dtype, tree, monkeypatch):
    """The same bits; the extension takes every one of these calls, and leaves those that need help."""
    _native.lib()
    _native.status_word(DEV)
    assert _native._host is not None, "the host extension is not built"

    def calls():
        bt = Batch(3, 2, 5, 64, dtype, "e4m3", 16, [20, 0, 33], dps=True, parents=_tree(5, 2) if tree else None)
        q, out = bt.q.to(DEV), []
        ct = torch.tensor([5, 2, 3], dtype=torch.int32, device=DEV)
        kw = dict(counts=ct, ancestors=bt.ancestors)
        out += [ft.tdp_decode(q, bt.cache, bt.table, bt.context, 0.1, 30, None, 20, **kw)]
        out += ft.tdp_decode(q, bt.cache, bt.table, bt.context, 0.1, return_lse=True, input_precision="ieee", **kw)
        ft.cache_write(bt.cache, bt.table, bt.context, q, q * 2, q, q, counts=ct)
        ft.dps_append(bt.cache, bt.table, bt.context, q, q, q, q, 0.1, 20, **kw)
        out += ft.dps_decode(q, bt.cache, bt.table, bt.context, 0.1, **kw)
        out += ft.cache_read(bt.cache, bt.table, bt.context, 5, TYPES[dtype], counts=ct)
        return out + [t.clone() for t in bt.cache]

    taken = []
    for name in HOST:
        f = getattr(_native._host, name[5:])
        monkeypatch.setattr(_native, name, lambda *a, f=f, name=name: taken.append((name, f(*a))) or taken[-1][1])
    fast = calls()
    assert len(taken) == 6 and all(r is not None for _, r in taken)
    for name in HOST:
        monkeypatch.setattr(_native, name, lambda *a: None)
    slow = calls()
    assert len(fast) == len(slow) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(fast, slow))
    ft.check_status(DEV)


@pytest.mark.gpu
def test_calls_that_need_help():
    """Rows that start off 16-byte boundaries or are not contiguous, a table with gaps, another current stream: copied first, the same result."""
    bt = Batch(2, 2, 3, 64, "fp16", "e4m3", 16, [20, 33], dps=True)
    q = bt.q.to(DEV)
    want = ft.tdp_decode(q, bt.cache, bt.table, bt.context, 0.1)
    store = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)
    odd = store[1:].view(q.shape).copy_(q)
    gaps = torch.zeros(2, 2 * bt.table.shape[1], dtype=torch.int32, device=DEV)[:, ::2].copy_(bt.table)
    wide = torch.zeros(2, 9, dtype=torch.int32, device=DEV)
    wide[:, : bt.table.shape[1]] = bt.table
    for x, table, ctx in [(odd, bt.table, bt.context), (q.transpose(2, 3).contiguous().transpose(2, 3), bt.table, bt.context),
                          (q, gaps, bt.context), (q, wide[:, : bt.table.shape[1]], bt.context), (q, bt.table, bt.context.repeat_interleave(2)[::2])]:
        assert torch.equal(ft.tdp_decode(x, bt.cache, table, ctx, 0.1), want)
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            other = ft.tdp_decode(x, bt.cache, table, ctx, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(other, want)
    ft.check_status(DEV)


# ---------------------------------------------------------------- refusals

def test_tree_ancestors():
    assert ft.tree_ancestors([-1, 0, 0, 2]).tolist() == [1, 3, 5, 13]
    assert ft.tree_ancestors([-1, -1]).tolist() == [1, 2]
    assert ft.tree_ancestors(list(range(-1, 63)))[63].item() == -1
    for bad in ([], [0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(ValueError):
            ft.tree_ancestors(bad)


def test_new_cache():
    c = ft.new_cache(3, 16, 2, 64, torch.int8, "cpu", dps=True)
    assert c.codes.shape == (3, 4, 2, 16, 64) and c.exponents.shape == (3, 4, 2, 16) and c.lse.shape == (3, 2, 16)
    assert ft.new_cache(1, 16, 1, 16, device="cpu").lse is None
    for kw in (dict(dtype=torch.float32), dict(page_size=12), dict(page_size=8), dict(head_dim=48)):
        with pytest.raises(ValueError):
            ft.new_cache(**{**dict(pages=1, page_size=16, heads=1, head_dim=64, device="cpu"), **kw})


def test_a_cache_on_the_cpu_is_refused():
    c = ft.new_cache(3, 16, 2, 64, torch.int8, "cpu", dps=True)
    table, ctx, x = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 1, 64)
    for call in (lambda: ft.cache_write(c, table, ctx, x, x, x, x), lambda: ft.cache_read(c, table, ctx, 1),
                 lambda: ft.tdp_decode(x, c, table, ctx), lambda: ft.dps_append(c, table, ctx, x, x, x, x), lambda: ft.dps_decode(x, c, table, ctx)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_refusals():
    c = ft.new_cache(3, 16, 2, 64, torch.int8, DEV)
    d = ft.new_cache(3, 16, 2, 64, torch.int8, DEV, dps=True)
    table, ctx = torch.zeros(1, 3, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 2, 1, 64, device=DEV, dtype=torch.float16)
    words = torch.ones(1, 1, dtype=torch.int64, device=DEV)
    bad = [
        lambda: ft.cache_write((c.codes, c.exponents), table, ctx, x, x, x, x),
        lambda: ft.cache_write(c, table, ctx, x, x, x, x.float()),
        lambda: ft.cache_write(c, table, ctx, x, x, x, x[:, :1]),
        lambda: ft.cache_write(c, table, ctx, x.long(), x.long(), x.long(), x.long()),
        lambda: ft.cache_write(c, table, ctx, *(x.expand(2, 2, 1, 64),) * 4),
        lambda: ft.cache_write(c, table, ctx, *(x[:, :, :0],) * 4),
        lambda: ft.cache_write(c, table.long(), ctx, x, x, x, x),
        lambda: ft.cache_write(c, table[0], ctx, x, x, x, x),
        lambda: ft.cache_write(c, table, ctx.long(), x, x, x, x),
        lambda: ft.cache_write(c, table, ctx.expand(2), x, x, x, x),
        lambda: ft.cache_write(c, table, ctx, x, x, x, x, counts=ctx.float()),
        lambda: ft.cache_read(c, table, ctx, 0),
        lambda: ft.cache_read(c, table, ctx, 1, torch.float64),
        lambda: ft.tdp_decode(x, c, table, ctx, k1_window=-1),
        lambda: ft.tdp_decode(x, c, table, ctx, ancestors=words.int()),
        lambda: ft.tdp_decode(x, c, table, ctx, ancestors=words.expand(1, 2)),
        lambda: ft.tdp_decode(x, c, table, ctx, input_precision="tf32"),
        lambda: ft.tdp_decode(x.expand(1, 2, 65, 64), c, table, ctx, ancestors=words.expand(1, 65)),
        lambda: ft.dps_decode(x, c, table, ctx),
        lambda: ft.dps_append(c, table, ctx, x, x, x, x),
        lambda: ft.dps_append(d, table, ctx, x, x, x, x, k_diff=-1),
        lambda: ft.tdp_decode(x, c._replace(exponents=c.exponents[:2]), table, ctx),
        lambda: ft.tdp_decode(x, c._replace(exponents=c.exponents.int()), table, ctx),
        lambda: ft.tdp_decode(x, c._replace(codes=c.codes.transpose(0, 3).contiguous().transpose(0, 3)), table, ctx),
        lambda: ft.dps_decode(x, d._replace(lse=d.lse.half()), table, ctx),
        lambda: ft.tdp_decode(x, ft.TrittentionCache(c.codes[..., :16, :].float(), c.exponents), table, ctx),
        lambda: ft.tdp_decode(x, ft.TrittentionCache(c.codes[:, :, :, :12].contiguous(), c.exponents[..., :12].contiguous()), table, ctx),
        lambda: ft.tdp_decode(x, ft.TrittentionCache(c.codes[:, :, :, :8].contiguous(), c.exponents[..., :8].contiguous()), table, ctx),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    ft.check_status(DEV)


def test_the_librarys_own_refusals():
    lib, C = _native.lib(), _native.C
    p = 1 << 20
    good = dict(codes=p, exponents=p, lse=p, pages=2, page_size=16, N=2, D=64, code=1, table=p, table_stride=2, table_pages=2, context=p, B=1, n=1)
    rows = (_native.Rows * 4)(*(_native.Rows(p, 64, 64, 64) for _ in range(4)))

    def calls(c, r=rows, ws=p, size=1 << 40, dtype=1, o=p):
        c = C.byref(c)
        return [lib.tritt_cache_write(c, r, dtype, None, None), lib.tritt_tdp_decode(c, r, o, None, dtype, 0.1, 1, 1, 1, 1, ws, size, None, 0, None),
                lib.tritt_dps_append(c, r, dtype, 0.1, 1, ws, size, None, 0, None), lib.tritt_dps_decode(c, r, o, None, dtype, 0.1, ws, size, None, 0, None)]

    for kw, rc in [(dict(B=0), -1), (dict(n=0), -1), (dict(pages=0), -1), (dict(D=48), -2), (dict(code=3), -3), (dict(page_size=12), -14),
                   (dict(page_size=8), -14), (dict(page_size=1 << 20, table_pages=1 << 12), -14), (dict(codes=None), -4), (dict(table=None), -4),
                   (dict(context=None), -4), (dict(codes=p + 8), -5), (dict(ancestors=p, n=65), -15), (dict(B=32768, N=2), -11),
                   (dict(B=8192, N=2, n=1 << 20), -11)]:
        c = _native.Cache(**{**good, **kw})
        assert calls(c) == [rc] * 4, kw
        assert lib.tritt_decode_workspace(_native.OP_TDP_DECODE, C.byref(c), 1, 1, 1, 0) == 0
    c = _native.Cache(**good)
    assert calls(c, dtype=7) == [-3] * 4 and calls(c, r=None) == [-4] * 4
    odd = (_native.Rows * 4)(*(_native.Rows(p, 64, 64, 4) for _ in range(4)))
    assert calls(c, r=odd) == [-5] * 4
    none = C.byref(_native.Cache(**{**good, "lse": None}))
    assert lib.tritt_dps_append(none, rows, 1, 0.1, 1, p, 1 << 40, None, 0, None) == -16
    assert lib.tritt_dps_decode(none, rows, p, None, 1, 0.1, p, 1 << 40, None, 0, None) == -16
    c = C.byref(c)
    wide = C.byref(_native.Cache(**{**good, "page_size": 4096}))   # (what fits in shared memory needs no workspace)
    assert lib.tritt_decode_workspace(_native.OP_TDP_DECODE, wide, 1, 1 << 30, 1 << 30, 0) > 0
    assert lib.tritt_tdp_decode(wide, rows, p, None, 1, 0.1, 9999, 9999, 1, 1, None, 0, None, 0, None) == -6
    assert lib.tritt_tdp_decode(wide, rows, p, None, 1, 0.1, 9999, 9999, 1, 1, p, 8, None, 0, None) == -6
    assert lib.tritt_tdp_decode(c, rows, p, None, 1, 0.1, 1, -1, 1, 1, p, 1 << 40, None, 0, None) == -10
    assert lib.tritt_tdp_decode(c, rows, None, None, 1, 0.1, 1, 1, 1, 1, p, 1 << 40, None, 0, None) == -4
    assert lib.tritt_dps_append(c, rows, 1, 0.1, -1, p, 1 << 40, None, 0, None) == -10
    assert lib.tritt_dps_append(c, rows, 1, 0.1, 1, p, 8, None, 0, None) == -6
    assert lib.tritt_dps_decode(c, rows, p + 4, None, 1, 0.1, p, 1 << 40, None, 0, None) == -5
    assert lib.tritt_cache_read(c, None, None, 1, None, None) == -4
