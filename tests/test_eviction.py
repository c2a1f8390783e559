"""The attention weight of cached tokens, and eviction by it, against the 64-bit definitions (``oracle/serving_oracle.py``).

A token's weight is a sum of p = exp(s - lse), all of them positive, so an error of the exponent's argument by at most d leaves it within d of its value (relative, d small).  A score's is
  (D + 64) 2^-24 (1 + size) for the sum of its D products, whose absolute values add up to `size`;
  2^-22 size for the operand q * K2, which is held in two fp16 numbers (of fp32 queries: rounded to 22 bits);
  2^-22 (1 + size + |lse|) for the factors, the argument (one multiplication and addition) and the exponential;
and the sums add 2^-24 for each addition in a line: a thread adds a column up over every 128th row, the block's and the CTAs' sums follow: at most 256 + (new tokens) (tokens / 128).
"""
import math

import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native, ops
from oracle import serving_oracle as orc
from tests.test_cache import Batch, TYPES, _randn, _table

DEV = "cuda:0"


def _bound(D, n, tokens, size, lse, gain, before):
    d = (D + 64) * 2.0 ** -24 * (1 + size) + 2.0 ** -21 * (1 + size + abs(lse))
    return gain * (math.expm1(float(d)) + (256 + n * (tokens / 128)) * 2.0 ** -24) + 2.0 ** -22 * (before.abs() + gain) + 1e-30


class Weighed(Batch):
    """A batch with weights of before, and each new token's log-sum-exps in 64 bits."""

    def __init__(self, *args, length=None, windows=(None,) * 4, k_diff=None, alpha=None, counts=None, **kw):
        super().__init__(*args, **kw)
        self.alpha, self.windows, self.k_diff = 1 / math.sqrt(self.D) if alpha is None else alpha, windows, k_diff
        self.length = length or max(1, max(self.contexts) + self.n + 3)
        self.counts = counts
        self.before = _randn(self.B, self.N, self.length, seed=5).exp()
        self.k2 = _randn(self.B, self.N, self.n, self.D, seed=6).to(self.dt)
        self.gain = torch.zeros(self.B, self.N, self.length, dtype=torch.float64)
        self.sums = torch.full((self.B, self.N, self.n), -math.inf)
        self.size, self.most = 0.0, 0.0
        for b, h, i in self.rows():
            ctx = self.contexts[b]
            if ctx < 0 or (counts is not None and i >= counts[b]):
                continue
            x, q = self.seq.values[b][:, h], self.q[b, h, i].double()
            if k_diff is None:
                zero = torch.zeros_like(x[2])
                lse = orc.tdp_row(q, x[0], x[1], zero, zero, ctx, i, self.alpha, windows)[1]
                self.sums[b, h, i] = lse
                if lse == -math.inf:
                    continue
                gain, size = orc.tdp_weights(q, x[0], x[1], ctx, i, self.alpha, windows, float(self.sums[b, h, i]))
                self.most = max(self.most, abs(float(lse)))
            else:
                inner = orc.dps_row(self.k2[b, h, i].double(), x[0], x[2], None, ctx, i, self.alpha, k_diff)[1].float()
                at = ctx + i
                self.seq.bias[b][h, at] = inner.double()
                self.cache.lse[int(self.seq.table[b, at // self.seq.page_size]), h, at % self.seq.page_size] = inner.to(DEV)
                m = orc.dps_row(q, x[1], x[3], self.seq.bias[b][h], ctx, i, self.alpha)[1]
                self.sums[b, h, i] = m
                gain, size = orc.dps_weights(q, self.k2[b, h, i].double(), x[0], x[1], self.seq.bias[b][h], ctx, i, self.alpha, k_diff, float(self.sums[b, h, i]))
                self.most = max(self.most, abs(float(m)) + float(self.seq.bias[b][h, :at + 1].abs().max()))
            self.size = max(self.size, float(size))
            self.gain[b, h] += torch.nn.functional.pad(gain, (0, max(0, self.length - gain.shape[0])))[: self.length]

    def run(self, weights=None, out=None, decay=1.0, table=None, **kw):
        weights = self.before.to(DEV) if weights is None else weights
        counts = None if self.counts is None else torch.tensor(self.counts, dtype=torch.int32, device=DEV)
        where = (self.cache, self.table if table is None else table, self.context, self.alpha)
        if self.k_diff is None:
            ft.tdp_weigh(weights, self.q.to(DEV), self.sums.to(DEV), *where, *self.windows, counts=counts, decay=decay, out=out, **kw)
        else:
            ft.dps_weigh(weights, self.q.to(DEV), self.k2.to(DEV), self.sums.to(DEV), *where, self.k_diff, counts=counts, decay=decay, out=out, **kw)
        return weights if out is None else out

    def check(self, got, decay=1.0, before=None, stale=None):
        before = self.before if before is None else before
        stale = before if stale is None else stale
        got = got.double().cpu()
        for b in range(self.B):
            ctx = self.contexts[b]
            end = 0 if ctx < 0 else min(self.length, ctx + (self.n if self.counts is None else max(0, min(self.n, self.counts[b]))))
            assert torch.equal(got[b, :, end:], stale[b, :, end:].double())
            old = decay * before[b].double()
            old[:, max(ctx, 0):] = 0
            want = (old + self.gain[b])[:, :end]
            err, bound = (got[b, :, :end] - want).abs(), _bound(self.D, self.n, max(1, end), self.size, self.most, self.gain[b][:, :end], old[:, :end])
            ok = bool((err <= bound).all())
            assert ok, f"sequence {b}: off by {float((err / bound).max()):.2f} bounds, {float((err - bound).max()):.3e} at {int((err > bound).sum())} of {err.numel()}"


TDP = [  # B N n D dtype code page contexts windows counts
    (1, 1, 1, 64, "fp16", "e4m3", 16, [0], (None,) * 4, None),
    (3, 2, 1, 64, "bf16", "fp16", 16, [1, 40, -1], (None,) * 4, None),
    (2, 3, 5, 64, "fp16", "int8", 32, [37, 130], (None,) * 4, [5, 2]),
    (2, 1, 9, 128, "fp16", "fp16", 64, [140, 0], (20, 50, 10, 3), None),
    (1, 2, 4, 128, "bf16", "int8", 16, [260], (128, 128, 32, 32), None),
    (1, 1, 3, 64, "fp16", "fp16", 16, [300], (None, 0, None, None), None),
    (1, 1, 3, 64, "fp16", "e4m3", 16, [200], (0, None, None, 0), None),
    (1, 2, 2, 64, "bf16", "fp16", 256, [257], (None, None, 0, 0), None),
    (2, 1, 2, 128, "bf16", "e4m3", 128, [129, 127], (60, None, None, 40), None),
    (1, 1, 2, 32, "fp16", "e4m3", 16, [30], (None,) * 4, None),
    (2, 2, 3, 64, "fp32", "fp16", 16, [20, 31], (15, None, 8, None), [0, 3]),
    (1, 1, 1, 256, "bf16", "int8", 16, [25], (None,) * 4, None),
    (1, 2, 2, 256, "fp16", "fp16", 32, [140], (None, 70, None, None), None),
    (2, 2, 3, 16, "fp32", "int8", 16, [50, 3], (None,) * 4, None),
    (2, 1, 2, 128, "fp32", "e4m3", 16, [131, 15], (None,) * 4, None),
    (1, 1, 66, 64, "bf16", "fp16", 16, [10], (None,) * 4, None),
    (1, 1, 150, 64, "fp16", "int8", 16, [0], (40, None, None, 7), None),
    (1, 2, 1, 64, "bf16", "e4m3", 64, [900], (None,) * 4, None),
    (2, 1, 2, 128, "fp16", "int8", 64, [700, 383], (None,) * 4, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,windows,counts", TDP)
def test_tdp_weigh(B, N, n, D, dtype, code, page, contexts, windows, counts, monkeypatch):
    bt = Weighed(B, N, n, D, dtype, code, page, contexts, windows=windows, counts=counts)
    got = bt.run()
    ft.check_status(DEV)
    bt.check(got)
    # to another place, laid out in another way, older weights fading; a table that is much longer
    out = torch.full((N, B, bt.length), 7.0, device=DEV).transpose(0, 1)
    before = bt.before.to(DEV)
    wide = torch.nn.functional.pad(bt.table, (0, 40), value=0)
    bt.run(before, out, 0.75, wide)
    ft.check_status(DEV)
    assert torch.equal(before.cpu(), bt.before)
    bt.check(out, 0.75, stale=torch.full_like(bt.before, 7.0))
    # nothing of before counts, whatever it is; the same bits again, and without the host extension
    again = [bt.run(torch.full_like(before, math.nan), torch.zeros_like(before), 0.0)]
    bt.check(again[0], 0.0, stale=torch.zeros_like(bt.before))
    monkeypatch.setattr(_native, "host_weigh", lambda *a: None)
    again.append(bt.run(torch.full_like(before, math.nan), torch.zeros_like(before), 0.0))
    assert torch.equal(*again)


DPS = [  # B N n D dtype code page contexts k_diff counts
    (1, 1, 1, 64, "fp16", "e4m3", 16, [0], 1024, None),
    (3, 2, 1, 64, "bf16", "fp16", 16, [1, 40, -1], 20, None),
    (2, 3, 5, 64, "fp16", "int8", 32, [37, 130], 1000, [5, 2]),
    (2, 1, 9, 128, "fp16", "fp16", 64, [140, 0], 0, None),
    (1, 2, 4, 128, "bf16", "int8", 16, [260], 128, None),
    (1, 1, 2, 32, "fp16", "e4m3", 16, [30], 5, None),
    (2, 2, 3, 64, "fp32", "fp16", 16, [20, 31], 15, [0, 3]),
    (1, 1, 1, 256, "bf16", "int8", 16, [25], 9, None),
    (1, 2, 70, 256, "fp32", "fp16", 32, [140], 100, None),
    (2, 2, 3, 16, "fp32", "int8", 16, [50, 3], 30, None),
    (1, 2, 11, 16, "bf16", "fp16", 16, [50], 30, None),
    (2, 1, 33, 256, "fp16", "e4m3", 16, [100, 15], 64, [33, 17]),
    (1, 1, 130, 64, "bf16", "fp16", 16, [10], 40, None),
    (1, 2, 1, 64, "bf16", "e4m3", 64, [2900], 1024, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,k_diff,counts", DPS)
def test_dps_weigh(B, N, n, D, dtype, code, page, contexts, k_diff, counts, monkeypatch):
    bt = Weighed(B, N, n, D, dtype, code, page, contexts, dps=True, k_diff=k_diff, counts=counts)
    got = bt.run()
    ft.check_status(DEV)
    bt.check(got)
    out = torch.full((N, B, bt.length), 7.0, device=DEV).transpose(0, 1)
    before = bt.before.to(DEV)
    bt.run(before, out, 0.75, torch.nn.functional.pad(bt.table, (0, 40), value=0))
    ft.check_status(DEV)
    bt.check(out, 0.75, stale=torch.full_like(bt.before, 7.0))
    again = [bt.run(torch.full_like(before, math.nan), torch.zeros_like(before), 0.0)]
    bt.check(again[0], 0.0, stale=torch.zeros_like(bt.before))
    monkeypatch.setattr(_native, "host_weigh", lambda *a: None)
    again.append(bt.run(torch.full_like(before, math.nan), torch.zeros_like(before), 0.0))
    assert torch.equal(*again)


FORMS = [dict(k_diff=None, dps=False), dict(k_diff=50, dps=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scale,alpha", [(1e-3, None), (3.0, None), (1.0, -0.3), (1.0, 0.0)])
def test_small_large_and_negative_scores(form, scale, alpha, D):
    bt = Weighed(1, 2, 3, D, "fp16", "fp16", 16, [150], scale=scale, alpha=alpha, **form)
    bt.check(bt.run())
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("code", ["fp16", "e4m3", "int8"])
def test_rows_of_very_different_sizes(code, D):
    """Exponents far apart in one tile, in both factors: a score's error is that of its own row."""
    bt = Batch(1, 1, 2, D, "fp16", code, 16, [200])
    x = _randn(4, 1, 202, D, seed=3).double()
    power = torch.randint(-90, 1, (202,), generator=torch.Generator().manual_seed(1)).double()
    x[0] *= torch.exp2(power)[None, :, None]
    x[1] *= torch.exp2(-power.flip(0))[None, :, None] * 2.0 ** -60
    x[1] *= torch.where(power.flip(0) < -60, 2.0 ** -50, 1.0)[None, :, None]
    seq = orc.Sequences([x], code, 16, bt.seq.codes.shape[0], bt.seq.table)
    k1, k2 = seq.values[0][0, 0], seq.values[0][1, 0]
    cache = ft.TrittentionCache(seq.codes.to(DEV), seq.exponents.to(DEV))
    sums, gain, most, size = torch.zeros(1, 1, 2), torch.zeros(202, dtype=torch.float64), 0.0, 0.0
    for i in range(2):
        q, zero = bt.q[0, 0, i].double(), torch.zeros_like(k1)
        sums[0, 0, i] = orc.tdp_row(q, k1, k2, zero, zero, 200, i, 0.1)[1]
        one, s = orc.tdp_weights(q, k1, k2, 200, i, 0.1, (None,) * 4, float(sums[0, 0, i]))
        gain, most, size = gain + one, max(most, abs(float(sums[0, 0, i]))), max(size, float(s))
    out = torch.zeros(1, 1, 202, device=DEV)
    ft.tdp_weigh(out, bt.q.to(DEV), sums.to(DEV), cache, bt.table, bt.context, 0.1)
    ft.check_status(DEV)
    err = (out[0, 0].double().cpu() - gain).abs()
    assert bool((err <= _bound(D, 2, 202, size, most, gain, 0 * gain)).all()), float((err / gain).max())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("form", FORMS)
def test_rows_and_queries_that_are_not_finite(form, D):
    bt = Weighed(2, 2, 2, D, "bf16", "e4m3", 16, [100, 60], **form)
    place = lambda t: (int(bt.seq.table[0, t // 16]), t % 16)  # noqa: E731
    page, row = place(101)
    for part in (0, 1):
        bt.cache.exponents[page, part, 0, row] = 255   # of the last new token: only it attends to the row
    got = bt.run().cpu()
    ft.check_status(DEV)
    assert bool(got[0, 0, :102].isnan().any())          # (what attends to it is NaN ...)
    ok = got.clone()
    ok[0, 0, :102] = (bt.before[0, 0, :102] * (torch.arange(102) < 100) + bt.gain[0, 0, :102]).float()   # (... other heads and sequences are as ever)
    bt.check(ok)
    bt.cache.exponents[page, :2, 0, row] = 127
    # hidden by counts, the same row changes nothing
    hidden = Weighed(2, 2, 2, D, "bf16", "e4m3", 16, [100, 60], counts=[1, 2], **form)
    hidden.cache.exponents[page, :2, 0, row] = 255
    hidden.check(hidden.run())
    ft.check_status(DEV)
    bad = Weighed(1, 2, 2, D, "bf16", "e4m3", 16, [40], **form)
    bad.q = bad.q.clone()
    bad.q[0, 1, 0, 3] = math.inf
    got = bad.run()
    assert bool(got[0, 1, :41].isnan().all()) and not bool(got[0, 0].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("form", FORMS)
def test_nothing_attended_missing_places_and_short_weights(form, D):
    bt = Weighed(2, 1, 3, D, "fp16", "int8", 16, [70, 20], **form)
    sums = bt.sums.clone()
    bt.sums[:] = -math.inf                      # tokens that attend to nothing add nothing
    if bt.k_diff is not None:
        for b, i in ((0, 0), (0, 1), (0, 2), (1, 0), (1, 1), (1, 2)):
            at = bt.contexts[b] + i
            bt.cache.lse[int(bt.seq.table[b, at // 16]), 0, at % 16] = -math.inf
    got = bt.run().cpu()
    ft.check_status(DEV)
    for b, c in enumerate(bt.contexts):
        assert torch.equal(got[b, 0, :c], bt.before[b, 0, :c]) and float(got[b, 0, c:c + 3].abs().max()) == 0
    # a page that there is not: its tokens keep their weights, the others' come from the pairs that there are
    bt = Weighed(2, 1, 3, D, "fp16", "int8", 16, [70, 20], **form)
    table = bt.table.clone()
    table[0, 1] = -1
    full, part = bt.run().cpu(), bt.run(table=table).cpu()
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    assert torch.equal(part[0, 0, 16:32], bt.before[0, 0, 16:32])
    rest = torch.cat((torch.arange(16), torch.arange(32, 70)))
    assert bool((part[0, 0, rest] <= full[0, 0, rest] * (1 + 1e-5)).all()) and bool((part[0, 0, rest] > bt.before[0, 0, rest]).all())
    assert torch.equal(part[1], full[1])
    # weights for fewer tokens than there are
    bt = Weighed(2, 1, 3, D, "fp16", "int8", 16, [70, 20], length=50, **form)
    bt.check(bt.run())
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    # a table that ends before the tokens do
    bt = Weighed(1, 1, 3, D, "fp16", "int8", 16, [70], **form)
    got = bt.run(table=bt.table[:, :4].contiguous()).cpu()
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    assert not bool(got.isnan().any())


def _longer(bt, pages=256):
    """A table with room for so many tokens more that the tiles of a call's kernel do not stay in shared memory."""
    return torch.nn.functional.pad(bt.table, (0, pages), value=0)


WINDOWS = [  # B N n D dtype code page contexts windows counts
    (2, 3, 1, 64, "bf16", "int8", 16, [500, 130], (128, 128, 32, 32), None),
    (1, 2, 16, 64, "fp16", "e4m3", 64, [333], (128, 128, 32, 32), None),
    (3, 1, 37, 64, "bf16", "fp16", 16, [200, 0, -1], (64, 64, 64, 64), [37, 20, 5]),
    (1, 1, 5, 64, "fp32", "fp16", 16, [300], (40, 150, 5, 9), None),
    (1, 1, 5, 64, "fp16", "int8", 32, [300], (150, 40, 9, 5), None),
    (2, 2, 3, 64, "bf16", "e4m3", 16, [90, 15], (0, 0, 0, 0), None),
    (2, 1, 9, 64, "fp16", "fp16", 128, [255, 256], (7, 120, 0, 3), [9, 0]),
    (1, 2, 16, 128, "bf16", "fp16", 16, [222], (128, 128, 32, 32), None),
    (2, 1, 3, 128, "fp32", "e4m3", 32, [300, 31], (100, 64, 20, 0), None),
    (1, 3, 21, 128, "fp16", "int8", 16, [140], (31, 33, None, 10), None),
    (40, 8, 1, 64, "bf16", "int8", 16, [b * 29 % 210 for b in range(40)], (100, 100, None, None), None),
    (1, 1, 2, 64, "bf16", "int8", 256, [1500], (1200, 1200, 16, 16), None),
    (1, 1, 60, 64, "fp16", "fp16", 16, [100], (90, 90, 20, 20), None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,n,D,dtype,code,page,contexts,windows,counts", WINDOWS)
def test_tdp_weigh_under_windows(B, N, n, D, dtype, code, page, contexts, windows, counts):
    """All that a head's tokens attend to stays in shared memory: one kernel.  The table's length is of no account."""
    bt = Weighed(B, N, n, D, dtype, code, page, contexts, windows=windows, counts=counts)
    before = _native.lib().tritt_kernel_launches()
    got = bt.run()
    assert _native.lib().tritt_kernel_launches() - before == 1
    ft.check_status(DEV)
    bt.check(got)
    out = torch.full((N, B, bt.length), 7.0, device=DEV).transpose(0, 1)
    bt.run(bt.before.to(DEV), out, 0.75, _longer(bt))
    bt.check(out, 0.75, stale=torch.full_like(bt.before, 7.0))
    again = [bt.run(torch.full_like(got, math.nan), torch.zeros_like(got), 0.0) for _ in range(2)]
    ft.check_status(DEV)
    bt.check(again[0], 0.0, stale=torch.zeros_like(bt.before))
    assert torch.equal(*again)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_queries_whose_elements_are_far_apart(dtype, D):
    """Large ones meet zeros of K2; small ones, some of them less than fp16 has next to those, make the scores."""
    bt = Batch(1, 1, 3, D, dtype, "fp16", 16, [150])
    x = _randn(4, 1, 153, D, seed=3).double()
    x[1, :, :, : D // 2] = 0
    q = _randn(1, 1, 3, D, seed=4)
    q[..., D // 2:] *= 2.0 ** -12
    bt.q = q.to(bt.dt)
    seq = orc.Sequences([x], "fp16", 16, bt.seq.codes.shape[0], bt.seq.table)
    k1, k2 = seq.values[0][0, 0], seq.values[0][1, 0]
    cache = ft.TrittentionCache(seq.codes.to(DEV), seq.exponents.to(DEV))
    alpha = 2.0 ** 9
    for windows, table in (((None,) * 4, bt.table), ((100, 100, 20, 20), bt.table), ((None,) * 4, _longer(bt))):
        sums, gain, most, size = torch.zeros(1, 1, 3), torch.zeros(153, dtype=torch.float64), 0.0, 0.0
        for i in range(3):
            qi, zero = bt.q[0, 0, i].double(), torch.zeros_like(k1)
            sums[0, 0, i] = orc.tdp_row(qi, k1, k2, zero, zero, 150, i, alpha, windows)[1]
            one, s = orc.tdp_weights(qi, k1, k2, 150, i, alpha, windows, float(sums[0, 0, i]))
            gain, most, size = gain + torch.nn.functional.pad(one, (0, 153 - one.shape[0])), max(most, abs(float(sums[0, 0, i]))), max(size, float(s))
        out = torch.zeros(1, 1, 153, device=DEV)
        ft.tdp_weigh(out, bt.q.to(DEV), sums.to(DEV), cache, table, bt.context, alpha, *windows)
        ft.check_status(DEV)
        err = (out[0, 0].double().cpu() - gain).abs()
        assert bool((err <= _bound(D, 3, 153, size, most, gain, 0 * gain)).all()), float((err / gain).max())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("windows", [(None,) * 4, (60, 60, 20, 20)])
@pytest.mark.parametrize("long", [False, True])
def test_odd_rows_and_places_under_windows_and_long_tables(windows, long, D):
    """A row that is not finite, a page that there is not, and a table that ends before the tokens do, in each of the kernels."""
    def batch(**kw):
        bt = Weighed(2, 2, 3, D, "bf16", "e4m3", 16, [100, 60], windows=windows, **kw)
        return bt, (_longer(bt) if long else bt.table)
    bt, table = batch()
    page, row = int(bt.seq.table[0, 6]), 102 % 16
    bt.cache.exponents[page, :2, 0, row] = 255     # of the last new token of the first head
    got = bt.run(table=table).cpu()
    ft.check_status(DEV)
    assert bool(got[0, 0, 90:103].isnan().all()) and not bool(got[0, 1].isnan().any()) and not bool(got[1].isnan().any())
    hidden, table = batch(counts=[2, 3])
    hidden.cache.exponents[page, :2, 0, row] = 255
    hidden.check(hidden.run(table=table))
    ft.check_status(DEV)
    bt, table = batch()
    full = bt.run(table=table).cpu()
    table = table.clone()
    table[0, 5] = -1
    part = bt.run(table=table).cpu()
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    assert torch.equal(part[0, :, 80:96], bt.before[0, :, 80:96]) and torch.equal(part[1], full[1])
    assert bool((part[0, :, :103] <= full[0, :, :103] * (1 + 1e-5)).all()) and bool((part[0, :, 96:100] > bt.before[0, :, 96:100]).all())
    got = bt.run(table=bt.table[:, :6].contiguous()).cpu()
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    assert not bool(got.isnan().any())
    bt.sums[:] = -math.inf
    got = bt.run(table=_longer(bt) if long else bt.table).cpu()
    ft.check_status(DEV)
    for b, c in enumerate(bt.contexts):
        assert torch.equal(got[b, :, :c], bt.before[b, :, :c]) and float(got[b, :, c:c + 3].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 32])
def test_a_table_far_longer_than_the_sequences(D):
    """Scratch for all of a table's tokens: a call takes some sequences at a time."""
    B = 40
    bt = Weighed(B, 2, 1, D, "fp16", "int8", 256, [b * 31 % 90 - 1 for b in range(B)], strided=False)
    table = torch.nn.functional.pad(bt.table, (0, 1024 - bt.table.shape[1]), value=0)
    c = _native.Cache(codes=bt.cache.codes.data_ptr(), exponents=bt.cache.exponents.data_ptr(), pages=bt.cache.codes.shape[0], page_size=256, N=2, D=D, code=2,
                      table=table.data_ptr(), table_stride=1024, table_pages=1024, context=bt.context.data_ptr(), B=B, n=1)
    whole = (148 + 2 * B) * 5 * 256 * 1024 * 4
    assert 0 < _native.lib().tritt_tdp_weigh_workspace(c, 1 << 30, 1 << 30) < min(whole, 1 << 30)
    bt.check(bt.run(table=table))
    ft.check_status(DEV)


@pytest.mark.gpu
def test_weights_that_share_places_are_refused():
    bt = Weighed(2, 2, 1, 64, "bf16", "e4m3", 16, [20, 10])
    for w in (torch.zeros(1, 2, 40, device=DEV).expand(2, 2, 40), torch.zeros(2, 1, 40, device=DEV).expand(2, 2, 40), torch.zeros(400, device=DEV).as_strided((2, 2, 40), (39, 80, 1))):
        with pytest.raises(ValueError):
            bt.run(weights=torch.zeros(2, 2, 40, device=DEV), out=w)
    out = torch.zeros(400, device=DEV).as_strided((2, 2, 40), (50, 100, 1))   # (sequences within heads)
    bt.run(weights=bt.before.to(DEV), out=out[:, :, : bt.length])
    bt.check(out[:, :, : bt.length], stale=torch.zeros_like(bt.before))


@pytest.mark.gpu
def test_many_sequences_and_heads():
    """More sequences than a block has threads, most of them short or unused: the line over all of them."""
    B = 700
    contexts = [(-1 if b % 3 == 1 else b * 37 % 50) for b in range(B)]
    contexts[B - 1] = 300
    bt = Weighed(B, 1, 1, 64, "bf16", "e4m3", 16, contexts, strided=False)
    bt.check(bt.run())
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 32])
@pytest.mark.parametrize("form", FORMS)
def test_in_graphs_that_run_at_once_and_on_another_stream(form, D):
    first, second = (Weighed(2, 3, 2, D, "bf16", "int8", 16, c, **form) for c in ([200, 90], [33, 301]))
    want = [bt.run() for bt in (first, second)]
    calls = []
    for bt in (first, second):
        q, k2, sums = bt.q.to(DEV), bt.k2.to(DEV), bt.sums.to(DEV)
        before, out = bt.before.to(DEV), bt.before.to(DEV)
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            if bt.k_diff is None:
                ft.tdp_weigh(before, q, sums, bt.cache, bt.table, bt.context, bt.alpha, out=out)
            else:
                ft.dps_weigh(before, q, k2, sums, bt.cache, bt.table, bt.context, bt.alpha, bt.k_diff, out=out)
        calls.append((graph, side, out, (q, k2, sums, before)))
    for _ in range(3):
        for graph, side, out, _ in calls:
            with torch.cuda.stream(side):
                out.zero_()
                graph.replay()
    torch.cuda.synchronize()
    ft.check_status(DEV)
    for (_, _, out, _), w, bt in zip(calls, want, (first, second)):
        for b, c in enumerate(bt.contexts):
            assert torch.equal(out[b, :, : c + 2], w[b, :, : c + 2]) and float(out[b, :, c + 2:].abs().max()) == 0


# ---------------------------------------------------------------- eviction

class Full(Batch):
    """A cache with weights; what is left of it after an eviction, from the definition."""

    def __init__(self, B, N, D, code, page, contexts, length=None, dps=False, seed=0):
        super().__init__(B, N, 1, D, "fp16", code, page, [c if c < 0 else c - 1 if c else 0 for c in contexts], dps=dps, seed=seed)
        self.contexts = contexts
        self.context = torch.tensor(contexts, dtype=torch.int32, device=DEV)
        self.length = length or max(max(contexts), 1)
        w = _randn(B, N, self.length, seed=seed + 3).exp()
        w[:, :, ::3] = w[:, :, ::3].round()   # (ties)
        w[:, :, 5::11] = -0.0
        w[:, :, 10::11] = 0.0
        self.weights = w

    def rows(self, table, count):
        """Codes, exponents and log-sum-exps of tokens 0 .. count - 1 as bytes, [B, 4, N, count, bytes], [B, 4, N, count], [B, N, count]."""
        page = self.seq.page_size
        t = torch.arange(count)
        at = table.cpu().long()[:, t // page]
        codes = self.cache.codes.view(torch.uint8).cpu()
        byte = self.cache.exponents.cpu()
        out = [codes[at, :, :, t % page].permute(0, 2, 3, 1, 4), byte[at, :, :, t % page].permute(0, 2, 3, 1)]
        return out + ([] if self.cache.lse is None else [self.cache.lse.cpu()[at, :, t % page].permute(0, 2, 1)])


EVICT = [  # B N D code page contexts keep first recent dps
    (1, 1, 64, "e4m3", 16, [40], 20, 2, 5, False),
    (3, 2, 64, "fp16", 16, [100, 30, -1], 30, 0, 0, True),
    (2, 3, 128, "int8", 32, [333, 200], 199, 4, 195, False),
    (2, 2, 128, "fp16", 64, [129, 64], 128, 0, 1, True),
    (1, 2, 16, "int8", 16, [600], 555, 7, 100, False),
    (1, 2, 16, "fp16", 16, [300], 1, 0, 0, False),
    (2, 1, 32, "e4m3", 16, [77, 0], 50, 50, 0, True),
    (1, 3, 256, "fp16", 32, [190], 97, 1, 1, False),
    (1, 2, 256, "int8", 16, [190], 100, 0, 32, True),
    (1, 1, 64, "fp16", 256, [5000], 2600, 4, 64, False),
    (1, 1, 16, "e4m3", 256, [40000], 9000, 4, 640, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("elsewhere,host", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("B,N,D,code,page,contexts,keep,first,recent,dps", EVICT)
def test_evict(B, N, D, code, page, contexts, keep, first, recent, dps, elsewhere, host, monkeypatch):
    _native.lib()
    if not host:
        monkeypatch.setattr(_native, "host_evict", lambda *a: None)
    bt = Full(B, N, D, code, page, contexts, length=max(max(contexts), keep) + 2, dps=dps)
    most = max(contexts)
    before = bt.rows(bt.table, most)
    codes_before = bt.cache.codes.view(torch.uint8).cpu()
    weights, table_out, weights_out = bt.weights.to(DEV), None, None
    if elsewhere:
        few = -(-keep // page)
        old = bt.cache.codes.shape[0]
        more = lambda t: None if t is None else torch.cat((t.view(torch.uint8) if t.element_size() == 1 else t, torch.full(  # noqa: E731
            (B * few, *t.shape[1:]), 3, dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device=DEV))).view(t.dtype)
        bt.cache = ft.TrittentionCache(*(more(t) for t in bt.cache))
        table_out = (old + torch.randperm(B * few, generator=torch.Generator().manual_seed(2))).view(B, few).int().to(DEV)
        weights_out = torch.full((N, B, keep + 1), 9.0, device=DEV).transpose(0, 1)
    context, kept = ft.cache_evict(weights, bt.cache, bt.table, bt.context, keep, first, recent, table_out=table_out, weights_out=weights_out)
    ft.check_status(DEV)
    assert context.tolist() == [min(c, keep) for c in contexts] and kept.dtype == torch.int32
    after, table = bt.rows(table_out if elsewhere else bt.table, min(keep, (table_out if elsewhere else bt.table).shape[1] * page)), (table_out if elsewhere else bt.table)
    got_w = (weights_out if elsewhere else weights).cpu()
    for b in range(B):
        for h in range(N):
            want = orc.evicted(bt.weights[b, h].tolist(), max(0, contexts[b]), keep, first, recent)
            c = len(want)
            assert kept[b, h].tolist() == want + [-1] * (keep - c)
            for x, y in zip(before, after):
                x, y = (x[b, h], y[b, h]) if x.dim() == 3 else (x[b, :, h].transpose(0, 1), y[b, :, h].transpose(0, 1))
                assert torch.equal(y[:c], x[want])
            assert torch.equal(got_w[b, h, :c], bt.weights[b, h, want])
            assert torch.equal(got_w[b, h, c:], torch.full((keep + 1 - c,), 9.0) if elsewhere else bt.weights[b, h, c:])
    if elsewhere:   # what was there stays
        assert torch.equal(bt.cache.codes.view(torch.uint8)[:old].cpu(), codes_before) and torch.equal(weights.cpu(), bt.weights)
    else:           # rows behind the kept ones, and pages of nobody, stay
        touched = torch.zeros(codes_before.shape[0], page, dtype=torch.bool)
        for b in range(B):
            for t in range(max(0, min(contexts[b], keep))):
                touched[int(bt.table[b, t // page]), t % page] = True
        assert torch.equal(bt.cache.codes.view(torch.uint8).cpu().permute(0, 3, 1, 2, 4)[~touched], codes_before.permute(0, 3, 1, 2, 4)[~touched])


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,D,ctx,keep", [(1, 1, 64, 9000, 6000), (1, 2, 16, 40000, 30000), (2, 2, 128, 700, 600)])
@pytest.mark.parametrize("table_too", [False, True])
def test_rows_to_other_pages_and_weights_in_place(B, N, D, ctx, keep, table_too):
    """Few heads and many tokens: several blocks move one head's rows.  A table that is the one for reading is a call in place."""
    bt = Full(B, N, D, "fp16", 64, [ctx] * B, length=ctx + 3)
    few = -(-keep // 64)
    old = bt.cache.codes.shape[0]
    bt.cache = ft.TrittentionCache(*(None if t is None else torch.cat((t, torch.zeros((B * few, *t.shape[1:]), dtype=t.dtype, device=DEV))) for t in bt.cache))
    table_out = bt.table if table_too else torch.arange(old, old + B * few, device=DEV).view(B, few).int()
    before, weights = bt.rows(bt.table, ctx), bt.weights.to(DEV)
    left, kept = ft.cache_evict(weights, bt.cache, bt.table, bt.context, keep, 2, 7, table_out=table_out)
    ft.check_status(DEV)
    after = bt.rows(table_out, keep)
    for b in range(B):
        for h in range(N):
            want = orc.evicted(bt.weights[b, h].tolist(), ctx, keep, 2, 7)
            assert int(left[b]) == keep and kept[b, h].tolist() == want
            assert torch.equal(weights[b, h].cpu(), torch.cat((bt.weights[b, h, want], bt.weights[b, h, keep:])))
            assert all(torch.equal(y[b, :, h], x[b, :, h][:, want]) for x, y in zip(before, after))


@pytest.mark.gpu
@pytest.mark.parametrize("ctx", [300, 30000])
def test_order_of_weights(ctx):
    """Infinities, NaN, zeros of either sign, negative ones, numbers next to one another; one CTA and a cluster."""
    bt = Full(1, 2, 16, "int8", 256, [ctx])
    w = bt.weights
    w[0, 0] = 1.0 + torch.randint(0, 3, (ctx,), generator=torch.Generator().manual_seed(1)) * 2.0 ** -23
    special = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, -1.0, 1e-45, -1e-45, 1e38, -math.nan])
    w[0, 1] = special[torch.randint(0, 10, (ctx,), generator=torch.Generator().manual_seed(2))]
    for keep in (1, 40, ctx // 2, ctx - 1):
        bt2 = Full(1, 2, 16, "int8", 256, [ctx])
        _, kept = ft.cache_evict(w.to(DEV), bt2.cache, bt2.table, bt2.context, keep)
        for h in range(2):
            assert kept[0, h].tolist() == orc.evicted(w[0, h].tolist(), ctx, keep, 0, 0)
    ft.check_status(DEV)


@pytest.mark.gpu
def test_shared_pages_and_places_that_there_are_not():
    bt = Full(2, 2, 64, "e4m3", 16, [100, 100])
    bt.table[1, :3] = bt.table[0, :3]                   # a shared prefix
    before, weights = bt.rows(bt.table, 100), bt.weights.to(DEV)
    spare = ft.new_cache(bt.cache.codes.shape[0] + 6, 16, 2, 64, torch.float8_e4m3fn, DEV)
    for new, old in zip(spare[:2], bt.cache[:2]):
        new.view(torch.uint8)[: old.shape[0]] = old.view(torch.uint8)
    bt.cache = spare
    out = torch.arange(bt.cache.codes.shape[0] - 6, bt.cache.codes.shape[0], dtype=torch.int32, device=DEV).view(2, 3)
    _, kept = ft.cache_evict(weights, bt.cache, bt.table, bt.context, 48, 4, 10, table_out=out, weights_out=torch.zeros(2, 2, 48, device=DEV))
    ft.check_status(DEV)
    after = bt.rows(out, 48)
    for b in range(2):
        for h in range(2):
            assert torch.equal(after[0][b, :, h], before[0][b, :, h][:, kept[b, h].long().cpu()])
    # a page that there is not: its rows are left out, the others move
    table = bt.table.clone()
    table[0, 2] = 10 ** 6
    bt.cache.codes.view(torch.uint8)[out.long()] = 85
    _, again = ft.cache_evict(weights, bt.cache, table, bt.context, 48, 4, 10, table_out=out, weights_out=torch.zeros(2, 2, 48, device=DEV))
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    assert torch.equal(again, kept)
    rows = bt.rows(out, 48)
    for h in range(2):
        numbers = kept[0, h].long().cpu()
        there = numbers // 16 != 2
        assert torch.equal(rows[0][0, :, h][:, there], after[0][0, :, h][:, there]) and bool((rows[0][0, :, h][:, ~there] == 85).all())
    assert torch.equal(rows[0][1], after[0][1])


@pytest.mark.gpu
def test_eviction_with_weights_for_fewer_tokens():
    bt = Full(1, 2, 64, "int8", 16, [100], length=60)
    _, kept = ft.cache_evict(bt.weights.to(DEV), bt.cache, bt.table, bt.context, 20, 2, 3)
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    for h in range(2):
        assert kept[0, h].tolist() == orc.evicted(bt.weights[0, h].tolist(), 60, 20, 2, 3)


@pytest.mark.gpu
def test_evict_in_a_graph_and_again():
    """Captured, replayed while contexts and weights change; twice in a row, in place."""
    bt = Full(2, 2, 64, "fp16", 16, [90, 50], dps=True)
    start = [t.clone() for t in bt.cache]
    weights, context = bt.weights.to(DEV), bt.context.clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        left, kept = ft.cache_evict(weights, bt.cache, bt.table, context, 40, 3, 9)
    for contexts in ([90, 50], [41, 40], [70, -1]):
        for t, s in zip(bt.cache, start):
            t.copy_(s)
        weights.copy_(bt.weights.flip(2))
        context.copy_(torch.tensor(contexts))
        before = bt.rows(bt.table, 90)
        graph.replay()
        torch.cuda.synchronize()
        after = bt.rows(bt.table, 40)
        assert left.tolist() == [min(c, 40) for c in contexts]
        for b in range(2):
            for h in range(2):
                want = orc.evicted(bt.weights.flip(2)[b, h].tolist(), max(0, contexts[b]), 40, 3, 9)
                assert kept[b, h].tolist() == want + [-1] * (40 - len(want))
                assert all(torch.equal((y[b, h] if y.dim() == 3 else y[b, :, h].transpose(0, 1))[: len(want)], (x[b, h] if x.dim() == 3 else x[b, :, h].transpose(0, 1))[want])
                           for x, y in zip(before, after))
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dps", [False, True])
def test_generation_with_a_short_cache(dps):
    """Tokens are written, attended to, weighed and evicted, with positions of two axes: each step against the definition over the rows that each head has kept."""
    B, N, D, page, keep, most, alpha, k_diff = 2, 2, 64, 16, 24, 32, 0.15, 12
    cache = ft.new_cache(B * 3, page, N, D, torch.float16, DEV, dps=dps)
    table = torch.randperm(B * 3, generator=torch.Generator().manual_seed(0)).view(B, 3).int().to(DEV)
    axes = ft.rotary_axes((8, 8), mixed=True)
    cos, sin = ft.rotary_tables(100, 32, device=DEV)
    weights, context = torch.zeros(B, N, 3 * page, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    rows = [[torch.zeros(4, 0, D, dtype=torch.float64) for _ in range(N)] for _ in range(B)]          # the definition's cache, of each head
    biases = [[torch.zeros(0, dtype=torch.float64) for _ in range(N)] for _ in range(B)]
    expected = [[torch.zeros(0, dtype=torch.float64) for _ in range(N)] for _ in range(B)]
    number = 0
    for step, n in enumerate([20, 1, 7, 1, 4, 8, 1, 8]):
        x = torch.randn(B, n, 5, N, D, generator=torch.Generator().manual_seed(step)).to(DEV, torch.bfloat16)
        q, k1, k2, v1, v2 = (t.transpose(1, 2) for t in x.unbind(2))
        at = number + torch.arange(n, device=DEV)
        q, k1, k2 = ft.qk_norm_rotary(q, k1, k2, None, None, None, cos, sin, torch.stack((at // 8, at % 8)), axes=axes)
        number += n
        old = int(context[0])
        if dps:
            ft.dps_append(cache, table, context, k1, k2, v1, v2, alpha, k_diff)
            o, sums = ft.dps_decode(q, cache, table, context, alpha)
            ft.dps_weigh(weights, q, k2, sums, cache, table, context, alpha, k_diff, decay=0.9)
        else:
            ft.cache_write(cache, table, context, k1, k2, v1, v2)
            o, sums = ft.tdp_decode(q, cache, table, context, alpha, return_lse=True)
            ft.tdp_weigh(weights, q, sums, cache, table, context, alpha, decay=0.9)
        new = ft.cache_read(cache, table, context, n, torch.float32)
        for b in range(B):
            for h in range(N):
                part = torch.stack([t[b, h].double().cpu() for t in new[:4]])
                rows[b][h] = torch.cat((rows[b][h], part), 1)
                k1_, k2_, v1_, w_ = rows[b][h]
                biases[b][h] = torch.cat((biases[b][h], new[4][b, h].double().cpu() if dps else torch.zeros(n)))
                gain = torch.zeros(old + n, dtype=torch.float64)
                for i in range(n):
                    qi, s = q[b, h, i].double().cpu(), float(sums[b, h, i])
                    if dps:
                        ref = orc.dps_row(qi, k2_, w_, biases[b][h], old, i, alpha)
                        gain += orc.dps_weights(qi, k2[b, h, i].double().cpu(), k1_, k2_, biases[b][h], old, i, alpha, k_diff, s)[0]
                    else:
                        ref = orc.tdp_row(qi, k1_, k2_, v1_, w_, old, i, alpha)
                        gain += orc.tdp_weights(qi, k1_, k2_, old, i, alpha, (None,) * 4, s)[0]
                    # (bf16 results: half a step, and the kernel's 2^-9 of its terms)
                    assert bool(((o[b, h, i].double().cpu() - ref[0]).abs() <= 2.0 ** -8 * ref[0].abs() + 2.0 ** -8 * ref[2] + 1e-6).all())
                expected[b][h] = torch.cat((0.9 * expected[b][h], torch.zeros(n))) + gain
                got = weights[b, h, : old + n].double().cpu()
                assert bool(((got - expected[b][h]).abs() <= 1e-4 * expected[b][h] + 1e-7).all())
                expected[b][h] = got   # (from here on the kernel's own, so that a tie is one for both)
        context += n
        if int(context[0]) > most - 8:
            context, kept = ft.cache_evict(weights, cache, table, context, keep - 8, 2, 6)
            for b in range(B):
                for h in range(N):
                    want = orc.evicted(expected[b][h].tolist(), rows[b][h].shape[1], keep - 8, 2, 6)
                    assert kept[b, h].tolist() == want
                    rows[b][h], biases[b][h], expected[b][h] = rows[b][h][:, want], biases[b][h][want], expected[b][h][want]
    ft.check_status(DEV)


@pytest.mark.gpu
def test_library_operators_and_compiled_calls():
    ns = torch.ops.flash_trittention
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    for form in FORMS:
        bt = Weighed(2, 2, 2, 64, "bf16", "fp16", 16, [40, 21], **form)
        q, k2, sums, w = bt.q.to(DEV), bt.k2.to(DEV), bt.sums.to(DEV), bt.before.to(DEV)
        codes, exponents, lse = bt.cache
        if bt.k_diff is None:
            torch.library.opcheck(ns.tdp_weigh.default, (w.clone(), w, q, sums, codes, exponents, bt.table, bt.context, 0.1, None, 9, None, None, None, 0.5), test_utils=checks)
        else:
            torch.library.opcheck(ns.dps_weigh.default, (w.clone(), None, q, k2, sums, codes, exponents, lse, bt.table, bt.context, 0.1, 50, None, 1.0), test_utils=checks)
        torch.library.opcheck(ns.cache_evict.default, (codes, exponents, lse, w.clone(), None, bt.table, bt.context, 10, 1, 2, None), test_utils=checks)

        def step(weights, q, k2, sums, codes, exponents, lse, table, context):
            cache = ft.TrittentionCache(codes, exponents, lse)
            if bt.k_diff is None:
                ft.tdp_weigh(weights, q, sums, cache, table, context, 0.1)
            else:
                ft.dps_weigh(weights, q, k2, sums, cache, table, context, 0.1, 50)
            return (*ft.cache_evict(weights, cache, table, context + 2, 10, 1, 2), weights * 1.0)

        out = []
        for f in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
            args = [w.clone(), q, k2, sums, *(None if t is None else t.clone() for t in bt.cache), bt.table, bt.context]
            out.append([*f(*args), args[0], args[4], args[5]])
        assert all(torch.equal(a, b) for a, b in zip(*out))
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_queries_that_want_gradients_and_results_elsewhere(form):
    """While a model is trained its queries have a history, of which the weights know nothing; eager and compiled, with new weights and rows in other places."""
    bt = Weighed(2, 2, 2, 64, "bf16", "int8", 16, [60, 21], **form)
    sums, table = bt.sums.to(DEV), bt.table
    few = 2
    old = bt.cache.codes.shape[0]
    cache = [None if t is None else torch.cat((t, torch.zeros((2 * few, *t.shape[1:]), dtype=t.dtype, device=DEV))) for t in bt.cache]
    table_out = torch.arange(old, old + 2 * few, device=DEV).view(2, few).int()

    def step(x, y, weights, out, short, codes, exponents, lse):
        q, k2, c = x * 1.0, y * 1.0, ft.TrittentionCache(codes, exponents, lse)
        if bt.k_diff is None:
            ft.tdp_weigh(weights, q, sums, c, table, bt.context, bt.alpha, out=out)
        else:
            ft.dps_weigh(weights, q, k2, sums, c, table, bt.context, bt.alpha, bt.k_diff, out=out)
        return (*ft.cache_evict(out, c, table, bt.context + 2, 20, 1, 2, table_out, short), (q * q).sum())

    got = []
    for f in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        x, y = bt.q.to(DEV).requires_grad_(True), bt.k2.to(DEV).requires_grad_(True)
        args = [bt.before.to(DEV), torch.zeros(2, 2, bt.length, device=DEV), torch.full((2, 2, 25), 3.0, device=DEV), *(None if t is None else t.clone() for t in cache)]
        left, kept, loss = f(x, y, *args)
        loss.backward()
        assert torch.equal(x.grad, 2 * x.detach()) and torch.equal(args[0].cpu(), bt.before)
        bt.check(args[1].detach(), stale=torch.zeros_like(bt.before))
        got.append([left, kept, *(t.detach() for t in args if t is not None)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert float(got[0][4][:, :, 20:].min()) == 3.0
    ft.check_status(DEV)


# ---------------------------------------------------------------- refusals, on the CPU

def _cpu(dps=False):
    cache = ft.new_cache(4, 16, 2, 64, torch.int8, "cpu", dps=dps)
    return cache, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)


def test_shapes_on_the_meta_device():
    cache = ft.new_cache(4, 16, 2, 64, torch.int8, "meta")
    table, context = torch.empty(1, 2, dtype=torch.int32, device="meta"), torch.empty(1, dtype=torch.int32, device="meta")
    left, kept = ops.cache_evict(*cache, torch.empty(1, 2, 32, device="meta"), None, table, context, 9, 1, 2, None)
    assert left.shape == (1,) and kept.shape == (1, 2, 9) and left.dtype == kept.dtype == torch.int32


def test_refusals(monkeypatch):
    """What the Python layer refuses, with the check that tensors are on a GPU left out."""
    from flash_trittention import eviction

    described = _native.Cache(B=1, N=2, n=3, D=64, page_size=16, table_pages=2)
    monkeypatch.setattr(eviction, "_describe", lambda *a: (described, ()))
    calls = []
    monkeypatch.setattr(_native, "tdp_weigh", lambda *a: calls.append("tdp"))
    monkeypatch.setattr(_native, "dps_weigh", lambda *a: calls.append("dps"))
    monkeypatch.setattr(_native, "cache_evict", lambda *a: calls.append("evict"))
    cache, table, ctx = _cpu(True)
    q, w, m = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 32), torch.zeros(1, 2, 3)
    tdp = lambda w=w, q=q, m=m, **kw: ft.tdp_weigh(w, q, m, cache, table, ctx, **kw)  # noqa: E731
    dps = lambda w=w, q=q, k2=q, m=m, cache=cache, **kw: ft.dps_weigh(w, q, k2, m, cache, table, ctx, **kw)  # noqa: E731
    evict = lambda w=w, keep=9, **kw: ft.cache_evict(w, cache, table, ctx, keep, **kw)  # noqa: E731
    tdp(), dps(), evict(), evict(table_out=table), evict(weights_out=torch.zeros(1, 2, 9))
    assert calls == ["tdp", "dps", "evict", "evict", "evict"]
    bad = [w[:, :1], w[0], w.double(), torch.zeros(1, 2, 32, 2)[..., 0], w.clone().requires_grad_(True), torch.zeros(1, 2, 0)]
    for call in (tdp, dps, evict):
        for x in bad:
            with pytest.raises(ValueError):
                call(w=x)
    for call in (tdp, dps):
        for kw in (dict(m=m[:, :, :2]), dict(m=m.double()), dict(q=q[:, :1]), dict(q=q.int()), dict(decay=-1.0), dict(decay=math.nan), dict(decay=math.inf),
                   dict(out=w[:, :1]), dict(w=torch.zeros(1, 2, 64)[:, :, :32], out=None, q=q[0])):
            with pytest.raises(ValueError):
                call(**kw)
    with pytest.raises(ValueError):
        tdp(k1_window=-1)
    with pytest.raises(ValueError):
        dps(k_diff=-1)
    with pytest.raises(ValueError):
        dps(cache=_cpu()[0])
    with pytest.raises(ValueError):
        dps(k2=q[:, :, :2])
    base = torch.zeros(2 * 40)
    with pytest.raises(ValueError):   # one place, two layouts
        tdp(w=base[:64].view(1, 2, 32), out=base.view(1, 2, 40))
    for x in (torch.zeros(1, 1, 32).expand(1, 2, 32), base.as_strided((1, 2, 32), (80, 20, 1))):   # one place, several tokens
        for call in (tdp, dps, evict):
            with pytest.raises(ValueError):
                call(w=x)
    for kw in (dict(keep=0), dict(first=-1), dict(recent=-1), dict(first=5, recent=5), dict(keep=33), dict(weights_out=torch.zeros(1, 2, 8)),
               dict(table_out=table.long()), dict(table_out=torch.zeros(2, 2, dtype=torch.int32)), dict(keep=17, table_out=table[:, :1]),
               dict(table_out=table[0]), dict(keep=1 << 40)):
        with pytest.raises(ValueError):
            evict(**kw)
    for call in (tdp, dps, evict):   # not a cache
        with pytest.raises(ValueError):
            ft.tdp_weigh(w, q, m, tuple(cache), table, ctx)
    assert len(calls) == 5


def test_tensors_must_be_on_a_gpu():
    cache, table, ctx = _cpu(True)
    q, w, m = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 32), torch.zeros(1, 2, 3)
    for call in (lambda: ft.tdp_weigh(w, q, m, cache, table, ctx), lambda: ft.dps_weigh(w, q, q, m, cache, table, ctx), lambda: ft.cache_evict(w, cache, table, ctx, 9)):
        with pytest.raises(RuntimeError):
            call()


def test_the_library_refuses():
    import ctypes as C

    L = _native.lib()
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 255) // 256 * 256
    good = dict(codes=p, exponents=p, lse=p, pages=2, page_size=16, N=1, D=64, code=2, table=p, table_stride=0, table_pages=1, context=p, B=1, n=2)
    weights = dict(before=p, after=p, before_length=16, after_length=16, decay=1.0)
    rows = _native.Rows(p, 0, 0, 64)

    def tdp(c={}, w={}, lse=p, alpha=0.1, win=(0, 0, 0, 0), ws=p, size=1 << 30, q=rows):  # noqa: B006
        return L.tritt_tdp_weigh(_native.Cache(**{**good, **c}), _native.Weights(**{**weights, **w}), q, lse, 1, alpha, *win, ws, size, None, None)

    def dps(c={}, w={}, m=p, alpha=0.1, k_diff=0, k2=rows):  # noqa: B006
        return L.tritt_dps_weigh(_native.Cache(**{**good, **c}), _native.Weights(**{**weights, **w}), rows, k2, m, 1, alpha, k_diff, None, None)

    def evict(c={}, w={}, out=(0, 0, 0), keep=9, first=0, recent=0, left=p + 64, kept=p):  # noqa: B006
        return L.tritt_cache_evict(_native.Cache(**{**good, **c}), _native.Weights(**{**weights, **w}), *out, keep, first, recent, left, kept, None, None)

    for call in (tdp, dps, evict):
        assert call(w=dict(before=None)) == -4 and call(w=dict(after=p + 2)) == -5 and call(w=dict(after_length=0)) == -1
        assert call(w=dict(decay=-0.5)) == -14 and call(w=dict(decay=math.nan)) == -14
        assert call(c=dict(ancestors=p)) == -15 and call(c=dict(D=48)) < 0 and call(c=dict(page_size=24)) < 0
    assert tdp(lse=None) == -4 and tdp(lse=p + 1) == -5 and tdp(alpha=math.inf) == -14 and tdp(win=(0, -1, 0, 0)) == -10
    assert tdp(ws=None) == -6 and tdp(size=100) == -6 and tdp(ws=p + 8) == -6 and tdp(q=_native.Rows(p + 8, 0, 0, 64)) == -5
    assert dps(m=None) == -4 and dps(alpha=math.nan) == -14 and dps(k_diff=-1) == -10 and dps(c=dict(lse=None)) == -16 and dps(k2=_native.Rows(None, 0, 0, 64)) == -4
    assert evict(keep=0) == -10 and evict(first=5, recent=5) == -10 and evict(first=-1) == -10 and evict(keep=17) == -1 and evict(left=None) == -4
    assert evict(left=p) == -4 and evict(kept=p + 2) == -5 and evict(out=(p, 0, 0)) == -12 and evict(out=(p, 0, 1), keep=17, w=dict(after_length=32)) == -12
    assert L.tritt_tdp_weigh_workspace(_native.Cache(**good), -1, 0) == 0
    # a small table; of 148 CTAs and a head five sums of one tile of 128 tokens
    assert L.tritt_tdp_weigh_workspace(_native.Cache(**good), 1 << 30, 0) == 256 + 149 * 5 * 128 * 4
