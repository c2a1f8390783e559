"""Attention over the cache beside rows that a new token does not attend to, and that are larger than its own by any power of two: another branch of a
tree (a padded draft, say), a token outside the window or the band.  The result is that of the attended rows alone, as exact as without them."""
import math

import pytest
import torch

import flash_trittention as ft
from oracle import serving_oracle as orc
from test_cache import DEV, Batch, _check_result, _kernel_of_windows, _score_error, _tree, _widened

K1, K2, V1, V2 = range(4)


def _enlarge(bt, b, token, parts, by):
    """The rows of a token (every head) times 2^by, in the pages and in the 64-bit values."""
    at = int(bt.table[b, token // bt.seq.page_size]), token % bt.seq.page_size
    for part in parts:
        byte = (bt.seq.exponents[at[0], part, :, at[1]].int() + by).clamp(2, 254)
        bt.seq.exponents[at[0], part, :, at[1]] = byte.to(torch.uint8)
        bt.seq.values[b][part, :, token] = orc.values(bt.seq.codes[at[0], part, :, at[1]], byte)
    bt.cache.exponents.copy_(bt.seq.exponents)


def _sees(bt, b, i, token, window):
    """Whether new token i attends to a token, at a distance up to the window."""
    ctx = bt.contexts[b]
    rows, pos, at = orc._tokens(ctx, i, bt.words)
    found = (rows == token).nonzero()
    return len(found) > 0 and (window is None or at - int(pos[found[0, 0]]) <= window)


TREES = [  # D dtype code n contexts parents hidden windows: hidden are (sequence, new token) or (sequence, token of the context)
    (64, "fp16", "e4m3", 5, [40, 21], [-1, 0, 0, 1, 2], [(0, 42), (1, 22)], (None,) * 4),
    (64, "bf16", "fp16", 7, [100], _tree(7, 2), [(0, 106), (0, 103)], (None,) * 4),
    (64, "fp16", "int8", 16, [130, 300], _tree(16, 2), [(0, 130 + 9), (1, 300 + 14)], (100, 100, 32, 32)),
    (128, "fp16", "fp16", 6, [70], [-1, 0, 0, 2, 1, 4], [(0, 72)], (None,) * 4),
    (128, "bf16", "e4m3", 9, [60, 90], _tree(9, 3), [(0, 62), (1, 98)], (50, 70, 20, 40)),
    (128, "bf16", "int8", 3, [200], [-1, -1, -1], [(0, 201)], (64, 64, None, None)),
]


def _tdp(bt, table, windows):
    alpha = 1 / math.sqrt(bt.D)
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, *windows, ancestors=bt.ancestors, return_lse=True)
    ft.check_status(DEV)
    return out, lse, alpha


def _tdp_rows(bt, out, lse, windows, alpha, rows):
    """Those rows against the definition, as the tests of the cache compare them (but for p below the kernels' range, which counts from the largest p
    of the row's own tokens)."""
    for b, h, i in rows:
        ctx, x = bt.contexts[b], bt.seq.values[b][:, h]
        ref = orc.tdp_row(bt.q[b, h, i].double(), x[0], x[1], x[2], x[3], ctx, i, alpha, windows, bt.words)
        _check_result(out[b, h, i], lse[b, h, i], ref, bt.dt, bt.D, (ctx + bt.n) ** 2, True, True, (b, h, i))


@pytest.mark.gpu
@pytest.mark.parametrize("by", [18, 26, 40, 100, 200])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,dtype,code,n,contexts,parents,hidden,windows", TREES)
def test_tdp_other_branches(D, dtype, code, n, contexts, parents, hidden, windows, wide, by):
    bt = Batch(len(contexts), 2, n, D, dtype, code, 16, contexts, parents=parents, seed=21)
    table = _widened(bt.table, 8192, 16) if wide else bt.table
    if all(w is None for w in windows):
        assert _kernel_of_windows(bt, table, windows) != wide   # (either kernel)
    for b, token in hidden:
        _enlarge(bt, b, token, range(4), by)
    out, lse, alpha = _tdp(bt, table, windows)
    again = _tdp(bt, table, windows)
    blind = [(b, h, i) for b, h, i in bt.rows() if not any(s == b and _sees(bt, b, i, t, None) for s, t in hidden)]
    assert len(blind) > 2 and len(blind) < len(contexts) * 2 * n
    assert all(torch.equal(out[at], again[0][at]) and torch.equal(lse[at], again[1][at]) for at in blind)
    _tdp_rows(bt, out, lse, windows, alpha, blind)


@pytest.mark.gpu
@pytest.mark.parametrize("by", [18, 26, 40, 100, 200])
@pytest.mark.parametrize("D,dtype,code", [(64, "fp16", "e4m3"), (64, "bf16", "int8"), (128, "fp16", "fp16"), (128, "bf16", "e4m3")])
@pytest.mark.parametrize("windows", [(40, 60, None, None), (300, 300, 20, 8)])
def test_tdp_tokens_outside_the_window_of_some(D, dtype, code, windows, by):
    """A chain: the token is behind the windows of the later new tokens, in those of the first ones.  (Window kernel and the other.)"""
    ctx, n = 330, 9
    at = ctx + 3 - max(windows[:2]) - 1   # the new tokens before number 3 see it
    bt = Batch(1, 2, n, D, dtype, code, 16, [ctx], seed=23)
    for part in range(4):
        _enlarge(bt, 0, at, [part], by)
    out, lse, alpha = _tdp(bt, _widened(bt.table, 8192, 16), windows)
    blind = [(b, h, i) for b, h, i in bt.rows() if not _sees(bt, b, i, at, max(windows[:2]))]
    assert len(blind) == 2 * (n - 3)
    _tdp_rows(bt, out, lse, windows, alpha, blind)


@pytest.mark.gpu
@pytest.mark.parametrize("by", [12, 16, 19, 21, 23, 25])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,dtype,code", [(64, "fp16", "fp16"), (64, "fp16", "e4m3"), (128, "fp16", "int8"), (128, "bf16", "fp16")])
def test_tdp_small_elements_beside_a_larger_row(D, dtype, code, wide, by):
    """A later token of the chain is larger; the first one attends to itself alone, and gets its own values' product, each element as the type rounds it
    (bfloat16: times a row's other half step)."""
    bt = Batch(2, 2, 4, D, dtype, code, 16, [0, 0], seed=33)
    for token in (2, 3):
        _enlarge(bt, 0, token, range(4), by)
    table = _widened(bt.table, 8192, 16) if wide else bt.table
    out, lse, alpha = _tdp(bt, table, (None,) * 4)
    for b in range(2):
        for h in range(2):
            want = bt.seq.values[b][V1, h, 0] * bt.seq.values[b][V2, h, 0]
            err = (out[b, h, 0].double().cpu() - want).abs()
            # (P of a single pair is a power of two; elements of fp16 codes below 2^-14 of their row's largest lose bits: 2^-25 of it)
            top = bt.seq.values[b][V1, h, 0].abs().max() * bt.seq.values[b][V2, h, 0].abs()
            least = 2.0 ** -25 if bt.dt == torch.float16 else 0.0
            assert bool((err <= torch.finfo(bt.dt).eps / 2 * want.abs() * (1 + 2.0 ** -10) + least + 2.0 ** -24 * top).all()), (b, h, float(err.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("by", [26, 60])
@pytest.mark.parametrize("D,dtype,code,windows", [(64, "fp16", "e4m3", (128, 128, 16, 16)), (128, "bf16", "fp16", (96, 96, 16, 16)),
                                                  (64, "fp16", "fp16", (None, None, 16, 16)), (128, "fp16", "int8", (None, None, 8, 16))])
def test_tdp_large_keys_that_are_attended(D, dtype, code, windows, by):
    """A K1 row 2^by larger, of a sign that gives its pairs a score of no weight: the other rows' scores keep their bits."""
    ctx = 200
    bt = Batch(1, 1, 1, D, dtype, code, 16, [ctx], seed=25)
    at = ctx - 30
    x, q, alpha = bt.seq.values[0][:, 0], bt.q[0, 0, 0].double(), 1 / math.sqrt(D)
    # among rows k of the band around it, all of one sign: K2 rows there equal
    page = bt.seq.page_size
    src = int(bt.table[0, at // page]), at % page
    for t in range(at - 16, at + 17):
        to = int(bt.table[0, t // page]), t % page
        bt.seq.codes.view(torch.uint8)[to[0], K2, :, to[1]] = bt.seq.codes.view(torch.uint8)[src[0], K2, :, src[1]]
        bt.seq.exponents[to[0], K2, :, to[1]] = bt.seq.exponents[src[0], K2, :, src[1]]
        x[K2, t] = x[K2, at]
    if float((q * x[K1, at] * x[K2, at]).sum()) > 0:
        codes = bt.seq.codes[src[0], K1, 0, src[1]]
        bt.seq.codes[src[0], K1, 0, src[1]] = (-codes.float()).to(codes.dtype)
        x[K1, at] = -x[K1, at]
    bt.cache.codes.view(torch.uint8).copy_(bt.seq.codes.view(torch.uint8))
    _enlarge(bt, 0, at, [K1], by)
    out, lse, alpha = _tdp(bt, _widened(bt.table, 4096, 16), windows)
    # (the score's error counts from the sum of |products| of the pairs that carry weight: those without that row)
    y = x.clone()
    y[K1, at] = 0
    plain = orc.tdp_row(q, y[0], y[1], y[2], y[3], ctx, 0, alpha, windows)
    ref = orc.tdp_row(q, x[0], x[1], x[2], x[3], ctx, 0, alpha, windows)
    assert float(ref[3]) > 2 ** 20
    _check_result(out[0, 0, 0], lse[0, 0, 0], (ref[0], ref[1], ref[2], plain[3]), bt.dt, D, (ctx + 1) ** 2, True, True, windows)


@pytest.mark.gpu
@pytest.mark.parametrize("by", [14, 26, 40, 100, 200])
@pytest.mark.parametrize("D,dtype,code,n,contexts,parents,hidden,windows", TREES)
def test_dps_other_branches(D, dtype, code, n, contexts, parents, hidden, windows, by):
    bt = Batch(len(contexts), 2, n, D, dtype, code, 16, contexts, dps=True, parents=parents, seed=27)
    alpha = 1 / math.sqrt(D)
    for b, token in hidden:
        _enlarge(bt, b, token, range(4), by)
    out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, ancestors=bt.ancestors)
    ft.check_status(DEV)
    again = ft.dps_decode(bt.q.to(DEV), bt.cache, bt.table, bt.context, alpha, ancestors=bt.ancestors)
    for b, h, i in bt.rows():
        if any(s == b and _sees(bt, b, i, t, None) for s, t in hidden):
            continue
        assert torch.equal(out[b, h, i], again[0][b, h, i]) and torch.equal(m[b, h, i], again[1][b, h, i])
        x = bt.seq.values[b][:, h]
        ref = orc.dps_row(bt.q[b, h, i].double(), x[K2], x[V2], bt.seq.bias[b][h], contexts[b], i, alpha, None, bt.words)
        _check_result(out[b, h, i], m[b, h, i], ref, bt.dt, D, contexts[b] + n, True, False, (b, h, i))


@pytest.mark.gpu
@pytest.mark.parametrize("by", [14, 26, 40, 100])
@pytest.mark.parametrize("D,dtype,code", [(64, "fp16", "fp16"), (64, "bf16", "e4m3"), (128, "fp16", "int8"), (128, "bf16", "fp16")])
def test_append_tokens_outside_the_window_of_some(D, dtype, code, by):
    """The inner attention's window ends inside a tile: the rows before it are loaded with it."""
    ctx, n, k_diff = 200, 11, 100
    at = ctx + 4 - k_diff   # new tokens up to 4 see it
    bt = Batch(1, 2, n, D, dtype, code, 16, [ctx], dps=True, seed=29)
    _enlarge(bt, 0, at, [K1, V1], by)
    x = torch.randn(1, n, 4, 2, D, generator=torch.Generator().manual_seed(5)).to(bt.dt)
    k1, k2, v1, v2 = (x[:, :, i].transpose(1, 2) for i in range(4))
    alpha = 1 / math.sqrt(D)
    ft.dps_append(bt.cache, bt.table, bt.context, *(t.to(DEV) for t in (k1, k2, v1, v2)), alpha, k_diff)
    back = [t.double().cpu() for t in ft.cache_read(bt.cache, bt.table, bt.context, n, torch.float32)]
    ft.check_status(DEV)
    grid = {"fp16": 2.0 ** -11, "e4m3": 2.0 ** -4, "int8": 2.0 ** -7}[code]
    for h in range(2):
        key, val = bt.seq.values[0][K1, h].clone(), bt.seq.values[0][V1, h].clone()
        key[ctx:], val[ctx:] = back[0][0, h], back[2][0, h]
        for i in range(4, n):
            y, lse, mass, size = orc.dps_row(k2[0, h, i].double(), key, val, None, ctx, i, alpha, k_diff)
            if i == 4:
                assert float(size) > 2.0 ** by / 8   # (it sees the row)
                continue
            w, mass = y * v2[0, h, i].double(), mass * v2[0, h, i].double().abs()
            d = _score_error(D, float(size), True, False)
            err = (math.expm1(2 * d) + 2.0 ** -10) * (mass + w.abs())
            top = float((w.abs() + err).max())
            rounding = (grid * w.abs() if code != "int8" else 0) + {"fp16": 2.0 ** -24, "e4m3": 2.0 ** -17, "int8": 2.0 ** -7}[code] * top
            bad = (back[3][0, h, i] - w).abs() - (err * (1 + 2 * grid) + rounding + 1e-30)
            assert float(bad.max()) <= 0, (h, i, float(bad.max()))
            assert abs(float(back[4][0, h, i]) - float(lse)) <= d + 2.0 ** -22 * (1 + abs(float(lse)))


def test_the_oracle_counts_only_what_is_attended():
    """(Of the tests themselves: a row that is hidden changes no reference, one that is not changes it.)"""
    bt_values = torch.randn(4, 12, 16, generator=torch.Generator().manual_seed(0)).double()
    words = ft.tree_ancestors([-1, 0, 0, 1])
    q = torch.randn(16, generator=torch.Generator().manual_seed(1)).double()
    row = lambda v, i: orc.tdp_row(q, *v, 8, i, 0.25, (None,) * 4, words)[0]  # noqa: E731
    big = bt_values.clone()
    big[:, 10] *= 2.0 ** 30   # new token 2
    assert torch.equal(row(bt_values, 3), row(big, 3)) and torch.equal(row(bt_values, 1), row(big, 1)) and not torch.equal(row(bt_values, 2), row(big, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,code", [(64, "fp16"), (64, "e4m3"), (128, "int8")])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e13])
def test_scores_of_which_32_bits_hold_no_fraction(D, code, size, wide, precision):
    """The largest score's pair has p = 1, however large it is: a mean of the attended products comes out, and that score as the log-sum-exp (whose
    relative error is A's rounding and the sums')."""
    bt = Batch(2, 2, 3, D, "bf16", code, 16, [90, 40], seed=31)
    bt.q = (bt.q.float() * size).to(torch.bfloat16)
    alpha = 1 / math.sqrt(D)
    table = _widened(bt.table, 8192, 16) if wide else bt.table
    out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, return_lse=True, input_precision=precision)
    ft.check_status(DEV)
    for b, h, i in bt.rows():
        x, ctx = bt.seq.values[b][:, h], bt.contexts[b]
        _, want, _, scores = orc.tdp_row(bt.q[b, h, i].double(), *x, ctx, i, alpha)
        most = (x[V1, : ctx + i + 1].abs().amax(0) * x[V2, : ctx + i + 1].abs().amax(0))
        assert bool((out[b, h, i].double().cpu().abs() <= most * (1 + 2.0 ** -7)).all()), (b, h, i)
        assert abs(float(lse[b, h, i]) - float(want)) <= (2.0 ** -11 + (D + 64) * 2.0 ** -24) * float(scores), (b, h, i)
