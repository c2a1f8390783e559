"""The attention weight of cached tokens beside rows of any size: rows next to zero, and rows that a token does not attend to and that are larger than its own by any power of two.

Tolerances: ``_bound`` of ``test_eviction``, counted from the arithmetic there."""
import math

import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from oracle import serving_oracle as orc
from tests.test_cache import Batch, _randn
from tests.test_eviction import DEV, Weighed, _bound, _longer

K1, K2 = 0, 1
CODES = ["fp16", "e4m3", "int8"]


def _gains(bt, alpha, windows, silent=()):
    """Log-sum-exps of the new tokens (-inf of the silent ones, which add nothing), what the others add, the largest |lse| and the largest sum of |products|."""
    sums = torch.full((bt.B, bt.N, bt.n), -torch.inf)
    tokens = max(c + bt.n for c in bt.contexts)
    gain, most, size = torch.zeros(bt.B, bt.N, tokens, dtype=torch.float64), 0.0, 0.0
    for b, h, i in bt.rows():
        if i in silent:
            continue
        ctx, q = bt.contexts[b], bt.q[b, h, i].double()
        x = bt.seq.values[b][:, h]
        zero = torch.zeros_like(x[K1])
        seen = torch.arange(x.shape[1]) <= ctx + i
        k1, k2 = (torch.where(seen[:, None], x[part], 0.0) for part in (K1, K2))
        sums[b, h, i] = orc.tdp_row(q, torch.nan_to_num(k1), torch.nan_to_num(k2), zero, zero, ctx, i, alpha, windows)[1]
        one, s = orc.tdp_weights(q, k1, k2, ctx, i, alpha, windows, float(sums[b, h, i]))
        gain[b, h, : one.shape[0]] += one
        most, size = max(most, abs(float(sums[b, h, i]))), max(size, float(s))
    return sums, gain, most, size


def _check(bt, alpha, windows, table, launches, silent=()):
    sums, gain, most, size = _gains(bt, alpha, windows, silent)
    out = torch.zeros(gain.shape, device=DEV)
    before = _native.lib().tritt_kernel_launches()
    ft.tdp_weigh(out, bt.q.to(DEV), sums.to(DEV), bt.cache, table, bt.context, alpha, *windows)
    if launches is not None:   # (which of the kernels it was)
        assert _native.lib().tritt_kernel_launches() - before == launches
    ft.check_status(DEV)
    got = out.double().cpu()
    for b in range(bt.B):
        end = bt.contexts[b] + bt.n
        err, bound = (got[b, :, :end] - gain[b, :, :end]).abs(), _bound(bt.D, bt.n, end, size, most, gain[b, :, :end], 0 * gain[b, :, :end])
        assert bool((err <= bound).all()), f"sequence {b}: {float((err / bound).max()):.3g} bounds, {float(err.max()):.3e} off"


def _put(bt, b, token, part, rows):
    """Rows [N, D] in 64 bits in the place of a token's, quantised, in the pages and in the 64-bit values."""
    codes, byte, value = orc.quantise(rows, bt.code)
    page, row = int(bt.seq.table[b, token // bt.seq.page_size]), token % bt.seq.page_size
    as_bytes = lambda t: t if t.element_size() > 1 else t.view(torch.uint8)  # noqa: E731
    as_bytes(bt.seq.codes)[page, part, :, row] = as_bytes(codes)
    bt.seq.exponents[page, part, :, row] = byte
    bt.seq.values[b][part, :, token] = value
    bt.cache = ft.TrittentionCache(bt.seq.codes.to(DEV), bt.seq.exponents.to(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D,long", [(64, False), (64, True), (128, False), (128, True), (32, True), (256, True)])
@pytest.mark.parametrize("part", [K1, K2])
def test_rows_next_to_zero(part, D, long, code):
    """Some rows are so small that their exponent byte is 1, the least, but their codes are not zeros; others are zeros.  Their scores are nothing beside the ordinary ones'."""
    bt = Batch(1, 2, 3, D, "bf16", code, 16, [200], seed=41)
    for token in range(4, 203, 7):
        size = (1e-37 if code == "int8" else 1e-36) if token % 3 else 0.0
        _put(bt, 0, token, part, _randn(2, D, seed=token).double() * size)
    page, row = int(bt.seq.table[0, 0]), 4
    assert int(bt.seq.exponents[page, part, 0, row]) == 1 and bool((bt.seq.codes[page, part, 0, row].float() != 0).any())
    _check(bt, 0.2, (None,) * 4, _longer(bt) if long else bt.table, 2 if long else None)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D,long", [(64, False), (64, True), (128, True), (32, True)])
def test_rows_next_to_zero_whose_partners_are_large(D, long, code):
    """Pairs of a token with itself alone: a row of 1e-36 meets one of 1e36, and the score is an ordinary one; so are the other pairs', whose rows are ordinary."""
    bt = Batch(1, 2, 2, D, "bf16", code, 16, [200], seed=43)
    for token in range(5, 202, 9):
        for part, size in ((K1, 1e36), (K2, 1e-36)) if token % 2 else ((K1, 1e-36), (K2, 1e36)):
            _put(bt, 0, token, part, _randn(2, D, seed=token + part).clamp(-3, 3).double() * size)
    windows = (None, None, 0, 0)
    _check(bt, 0.2, windows, _longer(bt) if long else bt.table, None)


def _enlarge(bt, b, token, part, by):
    """A token's rows times 2^by (None: not finite), in the pages and in the 64-bit values."""
    page, row = int(bt.seq.table[b, token // bt.seq.page_size]), token % bt.seq.page_size
    old = bt.seq.exponents[page, part, :, row].int()
    byte = torch.full_like(old, 255) if by is None else (old + by).clamp(2, 254)
    bt.seq.exponents[page, part, :, row] = byte.to(torch.uint8)
    bt.seq.values[b][part, :, token] = orc.values(bt.seq.codes[page, part, :, row], byte)
    bt.cache.exponents.copy_(bt.seq.exponents)


BY = [12, 30, 100, 200, None]
KERNELS = [(64, False), (64, True), (128, False), (128, True), (32, True)]   # D, a long table: each of the kernels


@pytest.mark.gpu
@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("part", [K1, K2])
@pytest.mark.parametrize("windows", [(None,) * 4, (100, 100, 20, 20)])
@pytest.mark.parametrize("D,long", KERNELS)
def test_later_tokens_that_are_larger(D, long, windows, part, by):
    """The new tokens before it do not attend to the last one, whatever it holds; it adds nothing itself (its log-sum-exp is -inf)."""
    bt = Batch(1, 2, 4, D, "bf16", "e4m3", 16, [150], seed=45)
    _enlarge(bt, 0, 153, part, by)
    _check(bt, 0.2, windows, _longer(bt) if long else bt.table, None, silent=(3,))


@pytest.mark.gpu
@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("windows,hidden,part", [((20, 100, 8, 8), 70, K2), ((100, 20, 8, 8), 70, K1), ((40, 60, None, None), 61, K2), ((60, 40, None, None), 61, K1),
                                                 ((40, 40, 16, 16), 45, K1), ((40, 40, 16, 16), 45, K2), ((20, None, 8, 8), 31, K2), ((None, 20, 8, 8), 31, K1)])
@pytest.mark.parametrize("D,long", KERNELS)
def test_tokens_outside_the_windows_or_the_band(D, long, windows, hidden, part, code, by):
    """A row of the context that no pair of the windows and the band has, but that lies among those that are looked at."""
    bt = Batch(1, 1, 2, D, "fp16", code, 16, [190], seed=47)
    _enlarge(bt, 0, 191 - hidden, part, by)
    if hidden == 61:
        assert 191 - hidden >= 190 - 60   # (the first new token attends to it; it adds nothing)
    _check(bt, 0.2, windows, _longer(bt) if long else bt.table, None, silent=(0,) if hidden == 61 else ())


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,queries", [(2.0 ** 100, 2.0 ** -100), (2.0 ** -100, 2.0 ** 100), (2.0 ** 60, 2.0 ** -60)])
@pytest.mark.parametrize("D,n,form", [(64, 2, "tdp"), (64, 60, "tdp"), (128, 2, "tdp"), (32, 2, "tdp"), (64, 2, "dps"), (128, 9, "dps"), (32, 3, "dps"), (256, 2, "dps")])
def test_queries_and_rows_of_opposite_sizes(form, D, n, rows, queries, dtype, code):
    """The scores are ordinary ones: all rows (of K1 in the triple product) are times a power of two, the queries, and the new tokens' k2, times its inverse."""
    kw = dict(k_diff=50, dps=True) if form == "dps" else {}
    bt = Weighed(1, 1, n, D, dtype, code, 16, [150], **kw)   # (of ordinary sizes: scaled by powers of two all scores keep their values)
    for part in (K1, K2) if form == "dps" else (K1,):
        for token in range(150 + n):
            _enlarge(bt, 0, token, part, round(math.log2(rows)))
    bt.q, bt.k2 = bt.q * queries, bt.k2 * queries
    bt.check(bt.run())
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("part", [K1, K2])
@pytest.mark.parametrize("D,n,code", [(64, 4, "e4m3"), (64, 9, "fp16"), (128, 4, "int8"), (32, 3, "fp16"), (256, 4, "e4m3")])
def test_later_tokens_that_are_larger_in_the_dot_product_sum(D, n, code, part, by):
    """The new tokens before it do not attend to the last one, whatever it holds."""
    kw = dict(dps=True, k_diff=40)
    bt, kept = (Weighed(1, 2, n, D, "bf16", code, 16, [130], counts=c, **kw) for c in (None, [n - 1]))
    bt.gain, bt.sums, bt.cache, bt.size, bt.most = kept.gain, kept.sums, kept.cache, kept.size, kept.most
    page, row = int(bt.seq.table[0, (130 + n - 1) // 16]), (130 + n - 1) % 16
    bt.cache.lse[page, :, row] = -math.inf
    _enlarge(bt, 0, 130 + n - 1, part, by)
    bt.check(bt.run())
    ft.check_status(DEV)
