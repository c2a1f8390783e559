"""Calls at the edges of the cache's operators and of the norms: sizes that 32 bits do not hold, derivatives that there are not, bad pointers."""
import math

import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from test_cache import DEV, Batch


# ---------------------------------------------------------------- more than the kernels count

@pytest.mark.gpu
def test_a_sequence_of_more_groups_than_can_be_numbered_is_reported():
    """65536 new tokens behind a million: 65536 * 34816 groups of 32 rows, more than 2^31.  Reported, the sequence without results; the others' are
    theirs.  (All of the table's places are those of one page: the sequence is not looked at.)"""
    n, page, D = 65536, 256, 64
    bt = Batch(1, 1, 3, D, "fp16", "e4m3", page, [40], seed=2)
    pages = (1 << 20) // page + n // page
    table = torch.zeros(3, pages, dtype=torch.int32, device=DEV)
    table[1, : bt.table.shape[1]] = bt.table[0]
    q = torch.zeros(3, 1, n, D, dtype=torch.float16, device=DEV)
    q[1, :, :3] = bt.q.to(DEV)[0]
    q[2] = q[1]
    context = torch.tensor([1 << 20, 40, 0], dtype=torch.int32, device=DEV)
    counts = torch.tensor([n, 3, 0], dtype=torch.int32, device=DEV)
    assert n * ((1 << 20) + n) // 32 > 2 ** 31
    out, lse = ft.tdp_decode(q, bt.cache, table, context, 0.125, counts=counts, return_lse=True)
    with pytest.raises(_native.TrittError, match="triple-dot-product attention over a cache"):
        ft.check_status(DEV)
    long = torch.zeros(1, pages, dtype=torch.int32, device=DEV)
    long[0, : bt.table.shape[1]] = bt.table[0]
    want, want_lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, long, bt.context, 0.125, return_lse=True)
    ft.check_status(DEV)
    # (the same pairs, perhaps cut at other places: fp32 sums in another order, P's and the result's rounding to fp16)
    assert float((out[1, :, :3].float() - want[0].float()).abs().max()) <= 2.0 ** -9 * float(want.float().abs().max())
    assert float((lse[1, :, :3] - want_lse[0]).abs().max()) <= 1e-5
    empty = torch.ones(3, 1, n, dtype=torch.bool, device=DEV)
    empty[1, :, :3] = False
    assert not bool(out[empty].any()) and bool((lse[empty] == -math.inf).all())


# ---------------------------------------------------------------- pointers and sizes that the C entries refuse

P = 1 << 20


def _cache_calls(**kw):
    lib, C = _native.lib(), _native.C
    out, m = kw.pop("out", P), kw.pop("m", P)
    c = C.byref(_native.Cache(**{**dict(codes=P, exponents=P, lse=P, pages=2, page_size=16, N=2, D=64, code=1, table=P, table_stride=2, table_pages=2,
                                        context=P, B=1, n=1), **kw}))
    rows, parts = (_native.Rows * 4)(*(_native.Rows(P, 64, 64, 64) for _ in range(4))), (C.c_void_p * 4)(P, P, P, P)
    return dict(write=lambda: lib.tritt_cache_write(c, rows, 1, None, None), read=lambda: lib.tritt_cache_read(c, parts, m, 1, None, None),
                tdp=lambda: lib.tritt_tdp_decode(c, rows, out, m, 1, 0.1, 1, 1, 1, 1, P, 1 << 40, None, 0, None),
                append=lambda: lib.tritt_dps_append(c, rows, 1, 0.1, 1, P, 1 << 40, None, 0, None),
                dps=lambda: lib.tritt_dps_decode(c, rows, out, m, 1, 0.1, P, 1 << 40, None, 0, None))


# (every call below is refused before anything is launched: there is no GPU in it)
@pytest.mark.parametrize("field,off", [("counts", 2), ("counts", 1), ("ancestors", 4), ("ancestors", 1), ("table", 2), ("context", 2)])
def test_the_caches_pointers_that_are_not_aligned_are_refused(field, off):
    for name, call in _cache_calls(**{field: P + off}).items():
        assert call() == -5, name


@pytest.mark.parametrize("off", [1, 2])
def test_log_sum_exps_that_are_not_aligned_are_refused(off):
    calls = _cache_calls(m=P + off)
    assert [calls[name]() for name in ("read", "tdp", "dps")] == [-5] * 3


def _norm_args(**kw):
    rows = lambda: (_native.Rows * 3)(*(_native.Rows(P, 64, 64, 64) for _ in range(3)))  # noqa: E731
    return _native.NormRotary(**{**dict(x=rows(), y=rows(), dx=rows(), B=1, N=1, T=1, D=64, dtype=1), **kw})


@pytest.mark.parametrize("wide,off", [(0, 2), (0, 1), (1, 4), (1, 2)])
def test_positions_that_are_not_aligned_are_refused(wide, off):
    lib, C = _native.lib(), _native.C
    a = _norm_args(rot=16, cos=P, sin=P, table=4, positions=P + off, positions64=wide)
    assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == -5
    assert lib.tritt_qk_norm_rotary_bwd(C.byref(a), P, 1 << 40, None, None) == -5


@pytest.mark.parametrize("kw,backward", [(dict(N=2 ** 31 - 1, T=64), False), (dict(N=2 ** 31 - 1, T=64), True), (dict(N=2 ** 31 - 3, B=64), False),
                                         (dict(N=90000), True), (dict(N=65536, weight_heads=1, weight_dtype=1), True)])
def test_more_heads_than_a_grid_has_are_refused(kw, backward):
    lib, C = _native.lib(), _native.C
    a = _norm_args(**kw)
    if backward:
        a.w[0] = a.dw[0] = P
        assert lib.tritt_qk_norm_rotary_bwd(C.byref(a), P, 1 << 60, None, None) == -11
    else:
        assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == -11


def test_the_workspace_of_very_many_heads_is_counted():
    """(Their groups were counted in 32 bits, which ended the process with a division by zero.)"""
    lib, C = _native.lib(), _native.C
    a = _norm_args(N=2 ** 31 - 1)
    a.w[0] = a.dw[0] = P
    assert lib.tritt_qk_norm_rotary_workspace(C.byref(a)) >= 3 * (2 ** 31 - 1) * 64 * 4
