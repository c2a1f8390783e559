"""Calls at the edges of the cache's operators and of the norms: sizes that 32 bits do not hold, derivatives that there are not, bad pointers."""
import ctypes
import importlib
import math

import pytest
import torch
from torch.autograd import forward_ad

import flash_trittention as ft
from flash_trittention import _native, ops  # noqa: F401  (the operators, registered)
from oracle import serving_oracle as orc
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


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["ieee", None])
def test_a_sequence_without_new_tokens_may_have_any_context(precision):
    bt = Batch(3, 2, 4, 64, "bf16", "e4m3", 16, [30, 17, 21], dps=True, seed=8)
    q = bt.q.to(DEV)
    counts = torch.tensor([4, 0, -3], dtype=torch.int32, device=DEV)
    table = torch.cat([bt.table, torch.full((3, 300), -1, dtype=torch.int32, device=DEV)], 1)   # (and the kernels of long tables)

    def calls(context, table):
        out = [ft.tdp_decode(q, bt.cache, table, context, 0.1, counts=counts, input_precision=precision)]
        ft.cache_write(bt.cache, table, context, q, q, q, q, counts=counts)
        ft.dps_append(bt.cache, table, context, q, q, q, q, 0.1, 20, counts=counts, input_precision=precision)
        out += ft.dps_decode(q, bt.cache, table, context, 0.1, counts=counts, input_precision=precision)
        out += ft.cache_read(bt.cache, table, context, 4, torch.float32, counts=counts)
        ft.check_status(DEV)
        return [t.clone() for t in out]

    for t in (bt.table, table):
        want = calls(bt.context, t)
        again = calls(torch.tensor([30, 1 << 20, 2 ** 31 - 1], dtype=torch.int32, device=DEV), t)
        assert all(torch.equal(a, b) for a, b in zip(want[1:], again[1:])) and torch.equal(want[0][1:], again[0][1:])


# ---------------------------------------------------------------- derivatives that there are not

def _norm_on_cpu(monkeypatch):
    """The norm's two calls by torch operations in the place of the kernels."""
    module = importlib.import_module("flash_trittention.norm_rotary")

    def forward(xs, ws, cos, sin, positions, eps, interleaved):
        return tuple(orc.norm_rotary(x.detach(), w.detach(), None, None, None, eps) for x, w in zip(xs, ws))

    def backward(xs, ws, cos, sin, positions, eps, interleaved, dys, weights_too):
        grads = []
        for x, w, dy in zip(xs, ws, dys):
            with torch.enable_grad():
                x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
                y = orc.norm_rotary(x, w, None, None, None, eps)
            grads.append([torch.zeros_like(x), torch.zeros_like(w)] if dy is None else torch.autograd.grad(y, [x, w], dy.detach()))
        return (*(g[0] for g in grads), *(g[1] if want else None for g, want in zip(grads, weights_too)))

    monkeypatch.setattr(module, "norm_rotary_forward", forward)
    monkeypatch.setattr(module, "norm_rotary_backward", backward)


def _leaves(shape, dtype=torch.float64, device="cpu"):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(shape, generator=g).to(device, dtype).requires_grad_(True) for _ in range(3)], [
        (torch.rand(shape[-1], generator=g) + 0.5).to(device, dtype).requires_grad_(True) for _ in range(3)]


def _second_derivatives_raise(f, leaves, like, what):
    """``f``'s gradients with create_graph: as without, and nothing that depends on them can be differentiated, whatever else the loss has."""
    plain = torch.autograd.grad(f(), leaves, torch.ones_like(like))
    for dy in (torch.ones_like(like), torch.ones_like(like).requires_grad_(True)):   # (of a linear loss, and of any other)
        grads = torch.autograd.grad(f(), leaves, dy, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        for g in grads:
            with pytest.raises(RuntimeError, match=what):
                (g.float().square().sum() + sum(t.float().square().sum() for t in leaves)).backward(retain_graph=True)


def test_a_second_derivative_of_the_norms_raises(monkeypatch):
    _norm_on_cpu(monkeypatch)
    xs, ws = _leaves((1, 2, 5, 16))
    like = torch.empty(1, 2, 5, 16, dtype=torch.float64)
    _second_derivatives_raise(lambda: sum(ft.qk_norm_rotary(*xs, *ws)), xs + ws, like, "qk_norm_rotary")
    # frozen weights, and a result that the loss does not have
    y = ft.qk_norm_rotary(*xs, *(w.detach() for w in ws))
    grads = torch.autograd.grad(y[1].sum(), xs, create_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="qk_norm_rotary"):
        (grads[1].sum() + xs[1].square().sum()).backward()


@pytest.mark.gpu
def test_a_second_derivative_of_the_norms_kernels_raises():
    xs, ws = _leaves((2, 3, 20, 64), torch.float32, DEV)
    _second_derivatives_raise(lambda: sum(ft.qk_norm_rotary(*xs, *ws)), xs + ws, xs[0].detach(), "qk_norm_rotary")


def _layouts(dtype, device):
    """[2, 3, 20, 64] tensors: plain, parts of a projection, rows that are not contiguous, expanded over heads, off 16-byte boundaries."""
    g = torch.Generator().manual_seed(4)
    new = lambda *shape: torch.randn(shape, generator=g).to(device, dtype)  # noqa: E731
    return {"plain": new(2, 3, 20, 64), "projection": new(2, 20, 5, 3, 64)[:, :, 1].transpose(1, 2), "columns": new(2, 3, 64, 20).transpose(2, 3),
            "expanded": new(2, 1, 20, 64).expand(2, 3, 20, 64), "every other": new(2, 3, 20, 128)[..., ::2], "heads last": new(2, 64, 20, 3).transpose(1, 3),
            "odd": new(2 * 3 * 20 * 64 + 1)[1:].view(2, 3, 20, 64)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gradients_of_the_norms_have_the_declared_layout(dtype, monkeypatch):
    """A compiler is told that the inputs' gradients are laid out as ``empty_like`` would.  (The kernel's place is taken by one that writes a
    number for each tensor into every row that it is given.)"""
    module = importlib.import_module("flash_trittention.norm_rotary")

    def kernel(a, dev, backward):
        for i in range(3):
            r, size = a.dx[i], dtype.itemsize
            for b in range(a.B):
                for n in range(a.N):
                    for t in range(a.T):
                        at = r.p + size * (b * r.stride_b + n * r.stride_n + t * r.stride_t)
                        ctypes.memmove(at, (ctypes.c_char * (size * a.D)).from_buffer_copy(torch.full((a.D,), i + 1.0).to(dtype).view(torch.uint8).numpy()),
                                       size * a.D)

    monkeypatch.setattr(_native, "host_norm_rotary_backward", lambda *a: None)
    monkeypatch.setattr(_native, "norm_rotary", kernel)
    layouts = _layouts(dtype, "cpu")
    for name, x in layouts.items():
        xs = (x, layouts["plain"], layouts["columns"])
        out = module.norm_rotary_backward(xs, (None,) * 3, None, None, None, 1e-6, False, (layouts["plain"],) * 3, (False,) * 3)
        for i, (dx, of) in enumerate(zip(out, xs)):
            assert dx.stride() == torch.empty_like(of).stride(), name
            assert bool((dx == i + 1).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_norms_operators_on_other_layouts(dtype):
    """Declared and real layouts, of the forward and of the backward; and the same numbers as of contiguous tensors."""
    ns, layouts = torch.ops.flash_trittention, _layouts(dtype, DEV)
    w = torch.rand(64, device=DEV) + 0.5
    cos, sin = ft.rotary_tables(20, 32, device=DEV)
    dys = [torch.randn(2, 3, 20, 64, device=DEV).to(dtype) for _ in range(3)]
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    for name, x in layouts.items():
        xs = [x, layouts["plain"], x]
        args = (*xs, w, None, w, cos, sin, None, 1e-6, False)
        torch.library.opcheck(ns.norm_rotary.default, args, test_utils=checks)
        torch.library.opcheck(ns.norm_rotary_bwd.default, (*args, *dys, [True, False, True]), test_utils=checks)
        got = ns.norm_rotary_bwd(*args, *dys, [True, False, True])
        want = ns.norm_rotary_bwd(*(t.contiguous() for t in xs), *args[3:], *dys, [True, False, True])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    ft.check_status(DEV)


def test_a_tangent_through_the_norms_raises(monkeypatch):
    _norm_on_cpu(monkeypatch)
    xs, ws = _leaves((1, 2, 5, 16))
    xs, ws = [x.detach() for x in xs], [w.detach() for w in ws]
    want = ft.qk_norm_rotary(*xs, *ws)
    with forward_ad.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(want, ft.qk_norm_rotary(*xs, *ws)))   # (no tensor with a tangent)
        for i in range(6):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(xs + ws)]
            with pytest.raises(RuntimeError, match="jvp"):
                ft.qk_norm_rotary(*args)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: ft.qk_norm_rotary(x, *xs[1:], *ws)[0], (xs[0],), (xs[0],))


def _decodes(cache, table, ctx):
    return {"tdp_decode": lambda q: ft.tdp_decode(q, cache, table, ctx, 0.1), "tdp_decode with lse": lambda q: ft.tdp_decode(q, cache, table, ctx, 0.1,
            return_lse=True)[0], "dps_decode": lambda q: ft.dps_decode(q, cache, table, ctx, 0.1)[0]}


def _decode_derivatives_raise(calls, q):
    for name, call in calls.items():
        want = call(q)
        assert not want.requires_grad
        leaf = q.clone().requires_grad_(True)
        with torch.no_grad():
            assert not call(leaf).requires_grad
        o = call(leaf)
        assert torch.equal(o.detach(), want)
        with pytest.raises(RuntimeError, match=name[:10]):
            (o.float().sum() + leaf.float().sum()).backward()
        call(leaf).mul_(2)   # (a result like any other)
        with forward_ad.dual_level():
            assert torch.equal(call(q), want)
            with pytest.raises(RuntimeError, match="jvp"):
                call(forward_ad.make_dual(q, q))


def test_derivatives_of_the_attention_over_a_cache_raise(monkeypatch):
    """(With another call in the place of the kernels'.)"""
    cache = ft.new_cache(1, 16, 2, 64, device="cpu", dps=True)
    monkeypatch.setattr(_native, "host_decode", lambda op, *a: (a[9].detach() * 2, a[9].detach().sum(-1)))
    q = torch.randn(1, 2, 3, 64)
    _decode_derivatives_raise(_decodes(cache, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)), q)


@pytest.mark.gpu
def test_derivatives_of_the_attention_over_a_cache_raise_on_the_gpu():
    bt = Batch(1, 2, 3, 64, "fp16", "e4m3", 16, [20], dps=True)
    _decode_derivatives_raise(_decodes(bt.cache, bt.table, bt.context), bt.q.to(DEV))
    ft.check_status(DEV)


def _attentions():
    return (("flash_trittention", lambda xs: ft.flash_trittention(*xs, 0.125, None, None, None, None)),
            ("TrittentionTriton", lambda xs: ft.TrittentionTriton(softmax_scale=0.125)(*xs)[0]))


@pytest.mark.parametrize("which", [0, 1])
def test_a_second_derivative_of_the_attentions_raises(which, monkeypatch):
    """(With other calls in the place of the kernels': what is looked at is what autograd makes of their results.)"""
    name, attend = _attentions()[which]
    like = torch.empty(1, 2, 5, 16, dtype=torch.float64)
    monkeypatch.setattr(_native, "host_forward", lambda op, q, k1, k2, v1, v2, *a: (q * k1 + k2 * v1 * v2, q.sum(-1), None)[: 2 + which])
    monkeypatch.setattr(_native, "host_backward", lambda op, q, k1, k2, v1, v2, o, do, *a: (do * k1, do * q, do * v1 * v2, do * k2 * v2, do * k2 * v1))
    xs = [torch.randn(like.shape, dtype=torch.float64).requires_grad_(True) for _ in range(5)]
    _second_derivatives_raise(lambda: attend(xs), xs, like, name)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_a_second_derivative_of_the_attentions_kernels_raises(which):
    name, attend = _attentions()[which]
    xs = [(0.5 * torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(i))).to(DEV, torch.float32).requires_grad_(True) for i in range(5)]
    got = torch.autograd.grad(attend(xs).sum(), xs, create_graph=True)
    for g in got:
        with pytest.raises(RuntimeError, match=name):
            (g.sum() + xs[0].square().sum()).backward(retain_graph=True)
    for a, b in zip(got, torch.autograd.grad(attend(xs).sum(), xs)):   # (the kernels' sums may be in another order)
        assert float((a - b).abs().max()) <= 1e-3 * float(b.abs().max())


# ---------------------------------------------------------------- pointers and sizes that the C entries refuse

P = 1 << 20


def _cache_calls(**kw):
    lib, C = _native.lib(), _native.C
    out, m, alpha = kw.pop("out", P), kw.pop("m", P), kw.pop("alpha", 0.1)
    c = C.byref(_native.Cache(**{**dict(codes=P, exponents=P, lse=P, pages=2, page_size=16, N=2, D=64, code=1, table=P, table_stride=2, table_pages=2,
                                        context=P, B=1, n=1), **kw}))
    rows, parts = (_native.Rows * 4)(*(_native.Rows(P, 64, 64, 64) for _ in range(4))), (C.c_void_p * 4)(P, P, P, P)
    return dict(write=lambda: lib.tritt_cache_write(c, rows, 1, None, None), read=lambda: lib.tritt_cache_read(c, parts, m, 1, None, None),
                tdp=lambda: lib.tritt_tdp_decode(c, rows, out, m, 1, alpha, 1, 1, 1, 1, P, 1 << 40, None, 0, None),
                append=lambda: lib.tritt_dps_append(c, rows, 1, alpha, 1, P, 1 << 40, None, 0, None),
                dps=lambda: lib.tritt_dps_decode(c, rows, out, m, 1, alpha, P, 1 << 40, None, 0, None))


# (every call below is refused before anything is launched: there is no GPU in it)
@pytest.mark.parametrize("field,off", [("counts", 2), ("counts", 1), ("ancestors", 4), ("ancestors", 1), ("table", 2), ("context", 2)])
def test_the_caches_pointers_that_are_not_aligned_are_refused(field, off):
    for name, call in _cache_calls(**{field: P + off}).items():
        assert call() == -5, name


@pytest.mark.parametrize("off", [1, 2])
def test_log_sum_exps_that_are_not_aligned_are_refused(off):
    calls = _cache_calls(m=P + off)
    assert [calls[name]() for name in ("read", "tdp", "dps")] == [-5] * 3


@pytest.mark.parametrize("alpha", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_not_finite_is_refused(alpha):
    calls = _cache_calls(alpha=alpha)
    assert [calls[name]() for name in ("tdp", "append", "dps")] == [-10] * 3


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


# ---------------------------------------------------------------- which kernel

@pytest.mark.parametrize("B,N,n,D,dtype,window,windows_kernel", [
    (32, 16, 1, 128, _native.BF16, 100, False), (8, 16, 16, 128, _native.F16, 100, False), (4, 8, 1, 128, _native.F16, 100, True),
    (32, 16, 1, 128, _native.F16, 64, True), (8, 16, 16, 128, _native.BF16, 128, True), (32, 16, 1, 128, _native.BF16, 160, False),
    (32, 16, 1, 64, _native.BF16, 160, True), (8, 16, 16, 64, _native.F16, 160, False), (8, 16, 16, 64, _native.F16, 128, True),
    (4, 8, 1, 64, _native.BF16, 200, False)])
def test_the_kernel_that_was_measured_to_be_faster_is_taken(B, N, n, D, dtype, window, windows_kernel):
    lib, C = _native.lib(), _native.C
    c = C.byref(_native.Cache(codes=P, exponents=P, pages=2, page_size=16, N=N, D=D, code=2, table=P, table_stride=256, table_pages=256, context=P, B=B, n=n))
    # (the kernel of windows needs no workspace)
    assert (lib.tritt_decode_workspace(_native.OP_TDP_DECODE, c, dtype, window, window, 0) == 0) == windows_kernel
