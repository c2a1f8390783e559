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
