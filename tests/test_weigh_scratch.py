"""Scratch of the weights of the triple product, as it is documented."""
import ctypes as C

import pytest

from flash_trittention import _native


def _bytes(**kw):
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 255) // 256 * 256
    good = dict(codes=p, exponents=p, pages=2, page_size=64, N=16, D=64, code=2, table=p, table_stride=0, table_pages=1, context=p, B=1, n=1)
    windows = kw.pop("windows", (1 << 30, 1 << 30))
    return _native.lib().tritt_tdp_weigh_workspace(_native.Cache(**{**good, **kw}), *windows)


@pytest.mark.parametrize("D,each", [(16, 8), (32, 8), (64, 20), (128, 20), (256, 8)])
def test_bytes_for_each_token_block_and_head(D, each):
    assert _bytes(D=D, page_size=64, table_pages=2048) == 256 + (148 + 16) * each * 2 ** 17
    assert _bytes(D=D, page_size=64, table_pages=2 ** 14) == 256 + (148 + 16) * each * 2 ** 20          # (one sequence: as much as it takes)
    assert _bytes(D=D, page_size=64, table_pages=2 ** 14, windows=(100, 300)) == 256 + (148 + 16) * each * 512   # 300 + 1 + 127 tokens, in tiles
    for B, N in ((1, 1), (7, 3), (500, 16), (65535, 1)):
        want = 256 * -(-8 * (B + 1) // 256)
        most = max(1, min(B, (2 ** 30 // (each * 2 ** 14) - 148) // N))
        assert _bytes(D=D, B=B, N=N, page_size=64, table_pages=256) == want + (148 + most * N) * each * 2 ** 14
        assert most in (1, B) or _bytes(D=D, B=B, N=N, page_size=64, table_pages=256) <= 2 ** 30 + want


def test_the_figures_of_the_documents():
    assert 425e6 < _bytes(table_pages=2 ** 11) < 435e6 and 3.35e9 < _bytes(table_pages=2 ** 14) < 3.45e9
