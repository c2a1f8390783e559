"""Weights of a sequence whose last new tokens have no place, because its table ends before them: the call reports it, and writes the weights of those tokens all the same."""
import math

import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from tests.test_eviction import DEV, Weighed

FORMS = [dict(k_diff=None, dps=False), dict(k_diff=50, dps=True), dict(k_diff=1000, dps=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("places,missing", [(256, 1), (128, 2), (256, 3), (512, 2), (144, 1), (128, 5)])
@pytest.mark.parametrize("n", [5, 9])
@pytest.mark.parametrize("D,code", [(64, "e4m3"), (128, "fp16"), (32, "int8")])
@pytest.mark.parametrize("form", FORMS)
def test_tokens_behind_the_table(form, D, code, n, places, missing):
    """The tokens that are there get what the new ones that are there add."""
    ctx = places - n + missing
    bt = Weighed(1, 2, n, D, "bf16", code, 16, [ctx], **form)
    lost = range(n - missing, n)
    kept = Weighed(1, 2, n, D, "bf16", code, 16, [ctx], counts=[n - missing], **form)
    bt.gain, bt.sums = kept.gain, kept.sums.clone()   # (tokens that are not there have no log-sum-exp: they add nothing)
    assert all(float(bt.sums[0, h, i]) == -math.inf for h in range(2) for i in lost)
    bt.cache = kept.cache
    table = bt.table[:, : places // 16].contiguous()
    got = bt.run(table=table)
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    bt.check(got)
    assert float(got[:, :, places: ctx + n].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 3])
@pytest.mark.parametrize("D,page", [(64, 256), (16, 16), (256, 16)])
@pytest.mark.parametrize("form", FORMS)
def test_one_page_and_a_token_too_many(form, D, page, n):
    ctx = 256 - n + 1
    bt = Weighed(1, 1, n, D, "fp16", "int8", page, [ctx], **form)
    kept = Weighed(1, 1, n, D, "fp16", "int8", page, [ctx], counts=[n - 1], **form)
    bt.gain, bt.sums, bt.cache = kept.gain, kept.sums.clone(), kept.cache
    got = bt.run(table=bt.table[:, : 256 // page].contiguous())
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    bt.check(got)
