"""Eviction with tables whose entries do not lie next to one another: kept transposed, or every second column of a wider one."""
import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from oracle import serving_oracle as orc
from tests.test_eviction import DEV, Full

LAYOUTS = {
    "transposed": lambda t: t.t().contiguous().t(),
    "every second column": lambda t: torch.stack((t, torch.full_like(t, -1)), -1).flatten(1)[:, ::2],
    "a column of many": lambda t: torch.stack((torch.full_like(t, -1), t), -1)[..., 1],
}


def test_a_table_out_that_is_the_table_is_a_call_in_place(monkeypatch):
    from flash_trittention import eviction

    seen = []
    monkeypatch.setattr(eviction, "_describe", lambda *a: (_native.Cache(B=2, N=2, n=1, D=64, page_size=16, table_pages=4), ()))
    monkeypatch.setattr(_native, "cache_evict", lambda c, w, table_out, *a: seen.append(table_out))
    cache = ft.new_cache(9, 16, 2, 64, torch.int8, "cpu")
    table, context, weights = torch.arange(8, dtype=torch.int32).view(2, 4), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64)
    for layout in LAYOUTS.values():
        t = layout(table)
        assert t.stride(1) != 1 and torch.equal(t, table)
        for out, in_place in ((t, True), (t[:], True), (t[:, :3], True), (t.clone(), False), (table, False), (t[:, 1:], False)):
            ft.cache_evict(weights, cache, t, context, 20, table_out=out)
            assert (seen[-1] is None) == in_place
            assert in_place or (seen[-1].stride(1) == 1 and torch.equal(seen[-1], out))
    wide = layout(table)
    ft.cache_evict(weights, cache, wide[:, ::2], context, 20, table_out=wide)   # (starts where the table does, and has other pages)
    assert seen[-1] is not None
    one = torch.arange(4, dtype=torch.int32).view(4, 1).t()                     # one sequence: how far apart rows are is of no account
    ft.cache_evict(weights[:1], cache, one, context[:1], 20, table_out=one.as_strided((1, 4), (99, 1)))
    assert seen[-1] is None


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("where", ["in place", "the table", "other pages"])
@pytest.mark.parametrize("B,N,D,code,ctx,keep", [(1, 1, 64, "fp16", 9000, 6000), (1, 2, 16, "int8", 40000, 30000), (2, 2, 128, "fp16", 700, 600), (3, 1, 64, "e4m3", 333, 100)])
def test_rows_move_by_strided_tables(B, N, D, code, ctx, keep, where, layout):
    """(The first three: several blocks move a head's rows.)"""
    bt = Full(B, N, D, code, 64, [ctx] * B, length=ctx + 3)
    few, old = -(-keep // 64), bt.cache.codes.shape[0]
    grown = lambda t: torch.cat((t, torch.zeros((B * few, *t.shape[1:]), dtype=t.dtype, device=DEV)))  # noqa: E731
    bt.cache = ft.TrittentionCache(grown(bt.cache.codes.view(torch.uint8)).view(bt.cache.codes.dtype), grown(bt.cache.exponents))
    table = LAYOUTS[layout](bt.table)
    out = {"in place": None, "the table": table, "other pages": LAYOUTS[layout](torch.arange(old, old + B * few, device=DEV).view(B, few).int())}[where]
    before, weights = bt.rows(bt.table, ctx), bt.weights.to(DEV)
    left, kept = ft.cache_evict(weights, bt.cache, table, bt.context, keep, 2, 7, table_out=out)
    ft.check_status(DEV)
    after = bt.rows(bt.table if out is None else out, keep)
    for b in range(B):
        for h in range(N):
            want = orc.evicted(bt.weights[b, h].tolist(), ctx, keep, 2, 7)
            assert int(left[b]) == keep and kept[b, h].tolist() == want
            assert torch.equal(weights[b, h].cpu(), torch.cat((bt.weights[b, h, want], bt.weights[b, h, keep:])))
            assert all(torch.equal(y[b, :, h], x[b, :, h][:, want]) for x, y in zip(before, after))
