"""Prompts and chunks of prompts over the cache against the whole-sequence kernels, and calls that the documentation allows beside the usual ones: any
softmax_scale, prefixes that sequences share, two streams at once."""
import pytest
import torch

import flash_trittention as ft
from test_cache import DEV, Batch, _dps_check, _randn, _table, _tdp_check, _widened


def _close(got, want, tol):
    err = (got.float() - want.float()).norm(dim=-1) / want.float().norm(dim=-1).clamp_min(1e-3)
    assert bool(torch.isfinite(got.float()).all()) and float(err.max()) < 4 * tol and float(err.square().mean().sqrt()) < tol, (float(err.max()), float(err.mean()))


# Float16 codes of fp16 tensors: the whole-sequence kernels round SiLU(V1), P and Y V2 to fp16 (2^-11 each), the cache's kernels A, P and W; a row's norm is off
# by less than these four's sum in the mean (2e-3), single rows, whose terms cancel, by a few times that.
TOL = 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,steps,k_diff", [(1100, 64, [1100], 300), (1100, 128, [700, 1, 399], 5000), (2500, 64, [1024, 1024, 452], 1024),
                                              (777, 128, [777], 64)])
def test_dps_prompts(T, D, steps, k_diff):
    B, N, page = 2, 2, 64
    xs = [(_randn(B, N, T, D, seed=i) * 0.7).to(DEV, torch.float16) for i in range(5)]
    whole, m = ft.TrittentionTriton(softmax_scale=0.1, k_diff=k_diff)(*xs)
    each = -(-T // page)
    table = _table(B, each, B * each + 1).to(DEV)
    cache = ft.new_cache(B * each + 1, page, N, D, torch.float16, DEV, dps=True)
    at = 0
    for n in steps:
        ctx = torch.full((B,), at, dtype=torch.int32, device=DEV)
        ft.dps_append(cache, table, ctx, *(t[:, :, at: at + n] for t in xs[1:]), 0.1, k_diff)
        o, lse = ft.dps_decode(xs[0][:, :, at: at + n], cache, table, ctx, 0.1)
        _close(o, whole[:, :, at: at + n], TOL)
        assert float((lse - m[:, :, at: at + n]).abs().max()) < 2e-2   # (its inner log-sum-exp of fp16 products, then the outer one)
        at += n
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,steps,windows", [(500, 64, [500], (None,) * 4), (300, 128, [300], (None,) * 4), (900, 64, [512, 388], (128, 128, 32, 32)),
                                               (700, 128, [130, 300, 270], (96, 200, None, 40)), (1300, 64, [1300], (60, 60, None, None))])
def test_tdp_chunks(T, D, steps, windows):
    B, N, page = 1, 2, 32
    xs = [(_randn(B, N, T, D, seed=i) * 0.7).to(DEV, torch.float16) for i in range(5)]
    k1w, k2w, kkl, kkr = windows
    whole = ft.flash_trittention(*xs, softmax_scale=0.1, k1_window=k1w, k2_window=k2w, kk_left=kkl, kk_right=kkr)
    each = -(-T // page)
    table = _table(B, each, each + 1).to(DEV)
    cache = ft.new_cache(each + 1, page, N, D, torch.float16, DEV)
    at = 0
    for n in steps:
        ctx = torch.full((B,), at, dtype=torch.int32, device=DEV)
        ft.cache_write(cache, table, ctx, *(t[:, :, at: at + n] for t in xs[1:]))
        _close(ft.tdp_decode(xs[0][:, :, at: at + n], cache, table, ctx, 0.1, *windows), whole[:, :, at: at + n], TOL)
        at += n
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("alpha", [-0.2, 0.0, 1e-30, -3.0])
def test_any_scale(alpha, wide, precision):
    for D, code in ((64, "e4m3"), (128, "fp16")):
        bt = Batch(2, 1, 4, D, "fp16", code, 16, [70, 3], dps=True, parents=[-1, 0, 0, 1], seed=41)
        table, fast = _widened(bt.table, 8192, 16) if wide else bt.table, precision is None
        out, lse = ft.tdp_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, 40, None, ancestors=bt.ancestors, return_lse=True, input_precision=precision)
        _tdp_check(bt, out, lse, (40, None, None, None), alpha, fast)
        out, m = ft.dps_decode(bt.q.to(DEV), bt.cache, table, bt.context, alpha, ancestors=bt.ancestors, input_precision=precision)
        _dps_check(bt, out, m, alpha, fast)
    ft.check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dps", [False, True])
def test_sequences_that_share_a_prefix(dps):
    """Two sequences whose tables name the same first pages, and go on in pages of their own."""
    N, D, page, n = 3, 64, 16, 2
    cache = ft.new_cache(8, page, N, D, torch.float16, DEV, dps=dps)
    table = torch.tensor([[5, 2, 0, 1], [5, 2, 7, 3]], dtype=torch.int32, device=DEV)
    start, at = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((2,), 32, dtype=torch.int32, device=DEV)
    prefix = [_randn(1, N, 32, D, seed=i).to(DEV, torch.float16) for i in range(5)]
    new = [_randn(2, N, n, D, seed=10 + i).to(DEV, torch.float16) for i in range(5)]
    alone = [ft.TrittentionCache(*(None if t is None else t.clone() for t in cache)) for _ in range(2)]
    write = (lambda c, t, at, x: ft.dps_append(c, t, at, *x[1:], 0.1, 20)) if dps else (lambda c, t, at, x: ft.cache_write(c, t, at, *x[1:]))
    ask = (lambda c, t, at, x: ft.dps_decode(x[0], c, t, at, 0.1)[0]) if dps else (lambda c, t, at, x: ft.tdp_decode(x[0], c, t, at, 0.1))
    write(cache, table[:1], start, prefix)
    write(cache, table, at, new)
    both = ask(cache, table, at, new)
    for b in range(2):
        own, one = table[b: b + 1], [t[b: b + 1] for t in new]
        write(alone[b], own, start, prefix)
        write(alone[b], own, at[:1], one)
        # (the line of steps is cut at other places: fp32 sums in another order, then fp16's rounding)
        assert float((both[b].float() - ask(alone[b], own, at[:1], one)[0].float()).abs().max()) <= 2.0 ** -9
    ft.check_status(DEV)


@pytest.mark.gpu
def test_two_streams_at_once_and_inference_mode():
    """Calls of two streams over one cache, each with its own workspace; tensors of inference mode; queries that are views of one head."""
    bt = Batch(3, 4, 2, 64, "bf16", "e4m3", 16, [900, 333, 50], dps=True, seed=43)
    q, table = bt.q.to(DEV), _widened(bt.table, 4096, 16)
    one = q[:, :1].expand(3, 4, 2, 64)
    calls = [lambda x: ft.tdp_decode(x, bt.cache, table, bt.context, 0.1), lambda x: ft.dps_decode(x, bt.cache, table, bt.context, 0.1)[0],
             lambda x: ft.tdp_decode(x, bt.cache, table, bt.context, 0.1, 50, 60, 8, 8)]
    want = [f(x) for f in calls for x in (q, one, one.contiguous())]
    assert all(torch.equal(want[i + 1], want[i + 2]) for i in (0, 3, 6))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s), torch.inference_mode():
                got.append([f(x) for f in calls for x in (q, one, one.contiguous())])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))
    ft.check_status(DEV)
