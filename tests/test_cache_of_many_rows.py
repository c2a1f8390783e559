"""Weights and eviction in a cache that has more rows than 32 bits number: the last pages hold what the first ones of a small cache do, and give the same bits."""
import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from tests.test_eviction import DEV, Weighed


def test_a_page_of_too_many_rows_is_refused():
    import ctypes as C

    L = _native.lib()
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 255) // 256 * 256
    cache = dict(codes=p, exponents=p, pages=1, page_size=1 << 28, N=2, D=64, code=2, table=p, table_stride=0, table_pages=1, context=p, B=1, n=2)
    weights = _native.Weights(before=p, after=p, before_length=16, after_length=16, decay=1.0)
    call = lambda **kw: L.tritt_tdp_weigh(_native.Cache(**{**cache, **kw}), weights, _native.Rows(p, 0, 0, 64), p, 1, 0.1, *(1 << 30,) * 4, p, 1 << 62, None, None)  # noqa: E731
    assert call() == -11 and call(D=128, code=0) == -11


@pytest.mark.gpu
def test_the_last_pages_of_a_large_cache():
    N, D, page, rows = 16, 64, 64, 2 ** 31 + 2 ** 20
    pages = -(-rows // (4 * N * page))
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < pages * 4 * N * page * (D + 1) + (8 << 30):
        pytest.skip("less free memory than the cache needs")
    bts = [Weighed(2, N, 3, D, "bf16", "e4m3", page, [300, 150]), Weighed(2, N, 3, D, "bf16", "e4m3", page, [300, 150], dps=True, k_diff=50)]
    codes = torch.empty(pages, 4, N, page, D, dtype=torch.float8_e4m3fn, device=DEV)
    exponents, lse = torch.empty(pages, 4, N, page, dtype=torch.uint8, device=DEV), torch.empty(pages, N, page, device=DEV)
    try:
        for bt in bts:
            few = bt.cache.codes.shape[0]
            got = []
            for cache, first in ((ft.TrittentionCache(*(None if t is None else t.clone() for t in bt.cache)), 0),
                                 (ft.TrittentionCache(codes, exponents, None if bt.cache.lse is None else lse), pages - few)):
                if first:
                    for large, small in zip(cache, bt.cache):
                        if large is not None:
                            (large.view(torch.uint8) if large.element_size() == 1 else large)[first:] = small.view(torch.uint8) if small.element_size() == 1 else small
                small, bt.cache = bt.cache, cache
                table = torch.nn.functional.pad(bt.table + first, (0, 64), value=first)   # (too long for the rows to stay in shared memory)
                weights = [bt.run(table=table)]
                if bt.k_diff is None:
                    weights.append(bt.run(table=bt.table + first))
                context, kept = ft.cache_evict(weights[0].clone(), cache, bt.table + first, bt.context, 100, 3, 20)
                bt.cache = small
                got.append([*weights, context, kept, cache.codes.view(torch.uint8)[first: first + few].clone(), cache.exponents[first: first + few].clone()])
            assert all(torch.equal(a, b) for a, b in zip(*got))
            bt.check(got[1][0])
        ft.check_status(DEV)
    finally:
        del codes, exponents, lse, cache, large
        torch.cuda.empty_cache()
