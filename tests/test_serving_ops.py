"""The ``torch.library`` operators of the norms and the cache: schemas, shapes on the meta device, and functions compiled without a graph break."""
import pytest
import torch

import flash_trittention as ft
from flash_trittention import ops

DEV = "cuda:0"
CHECKS = ("test_schema", "test_faketensor", "test_autograd_registration")


def test_operators_are_registered_with_schemas():
    ns = torch.ops.flash_trittention
    for name in ("norm_rotary", "norm_rotary_bwd", "cache_write", "cache_read", "tdp_decode", "dps_append", "dps_decode"):
        assert hasattr(ns, name)
    assert str(ns.dps_append.default._schema).count("!") == 3 and str(ns.cache_write.default._schema).count("!") == 2
    assert "!" not in str(ns.tdp_decode.default._schema)


def test_shapes_propagate_on_the_meta_device():
    x = [torch.empty(2, 3, 10, 64, device="meta", dtype=torch.bfloat16, requires_grad=True) for _ in range(3)]
    w = torch.empty(64, device="meta", requires_grad=True)
    cos = torch.empty(10, 16, device="meta")
    y = ops.norm_rotary(*x, w, None, w, cos, cos, None, 1e-6, False)
    assert all(t.shape == x[0].shape and t.dtype == x[0].dtype for t in y)
    sum(t.sum() for t in y).backward()
    assert all(t.grad.shape == t.shape for t in (*x, w)) and w.grad.dtype == w.dtype
    with pytest.raises(ValueError):
        ops.norm_rotary(*x, w[:32], None, None, None, None, None, 1e-6, False)
    c = ft.new_cache(5, 16, 3, 64, device="meta", dps=True)
    table, ctx = torch.empty(2, 2, dtype=torch.int32, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
    parts = ops.cache_read(*c, table, ctx, 4, torch.float16, None)
    assert [t.shape for t in parts] == [(2, 3, 4, 64)] * 4 + [(2, 3, 4)]
    q = x[0].detach()
    for o, m in (ops.tdp_decode(q, c.codes, c.exponents, table, ctx, 0.1, None, 5, None, None, None, None, None),
                 ops.dps_decode(q, *c, table, ctx, 0.1, None, None, None)):
        assert o.shape == q.shape and o.dtype == q.dtype and m.shape == q.shape[:3] and m.dtype == torch.float32


def test_cpu_tensors_have_no_implementation():
    x = torch.zeros(1, 1, 8, 16)
    with pytest.raises(NotImplementedError):
        ops.norm_rotary(x, x, x, None, None, None, None, None, None, 1e-6, False)


def _inputs(B=2, N=2, n=3, D=64, dtype=torch.bfloat16, dps=True):
    g = torch.Generator().manual_seed(0)
    cache = ft.new_cache(7, 16, N, D, torch.float16, DEV, dps=dps)
    table = torch.arange(6, dtype=torch.int32, device=DEV).view(B, 3)
    ctx = torch.tensor([20, 7], dtype=torch.int32, device=DEV)
    xs = [torch.randn(B, N, n, D, generator=g).to(DEV, dtype) for _ in range(5)]
    old = [torch.randn(B, N, 20, D, generator=g).to(DEV, dtype) for _ in range(4)]
    if dps:
        ft.dps_append(cache, table, ctx * 0, *old, counts=ctx)
    else:
        ft.cache_write(cache, table, ctx * 0, *old, counts=ctx)
    return cache, table, ctx, xs


@pytest.mark.gpu
def test_opcheck():
    ns = torch.ops.flash_trittention
    x = [torch.randn(1, 2, 20, 32, device=DEV, requires_grad=True) for _ in range(3)]
    w = torch.randn(2, 32, device=DEV, requires_grad=True)
    cos, sin = ft.rotary_tables(20, 16, device=DEV)
    torch.library.opcheck(ns.norm_rotary.default, (*x, w, None, w, cos, sin, None, 1e-6, True), test_utils=CHECKS)
    cache, table, ctx, (q, *new) = _inputs()
    codes, exponents, lse = cache
    for op, args in ((ns.cache_write, (codes, exponents, table, ctx, None, *new)), (ns.cache_read, (codes, exponents, lse, table, ctx, 3, torch.float32, ctx)),
                     (ns.tdp_decode, (q, codes, exponents, table, ctx, 0.1, None, 9, None, None, None, None, None)),
                     (ns.dps_append, (codes, exponents, lse, table, ctx, *new, 0.1, 100, None, None, None)),
                     (ns.dps_decode, (q, codes, exponents, lse, table, ctx, 0.1, None, None, "ieee"))):
        torch.library.opcheck(op.default, args, test_utils=CHECKS)
    ft.check_status(DEV)


@pytest.mark.gpu
def test_a_compiled_training_function_has_no_graph_break():
    B, N, T, D = 2, 2, 64, 64
    cos, sin = ft.rotary_tables(T, 32, device=DEV)
    x = torch.randn(B, T, 5, N, D, device=DEV, dtype=torch.bfloat16)
    w = [torch.rand(D, device=DEV) + 0.5 for _ in range(3)]
    dz = torch.randn(B, N, T, D, device=DEV, dtype=torch.bfloat16)

    def f(x, w):
        q, k1, k2, v1, v2 = (t.transpose(1, 2) for t in (x * 1.0).unbind(2))
        q, k1, k2 = ft.qk_norm_rotary(q, k1, k2, *w, cos, sin)
        return ft.flash_trittention(q, k1, k2, v1, v2, softmax_scale=0.1, kk_left=None, kk_right=None, k1_window=None, k2_window=20, causal=True)

    out = []
    for run in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        leaves = [x.clone().requires_grad_(True), *(t.clone().requires_grad_(True) for t in w)]
        y = run(leaves[0], leaves[1:])
        y.backward(dz)
        out.append([y.detach(), *(t.grad for t in leaves)])
    assert torch.equal(out[0][0], out[1][0])
    for a, b in zip(out[0][1:], out[1][1:]):   # (the attention's backward adds in an order that changes: one bf16 step of the largest element)
        assert float((a.float() - b.float()).abs().max()) <= 8e-3 * float(a.float().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dps", [False, True])
def test_a_compiled_decoding_step_has_no_graph_break(dps):
    def f(cache, table, ctx, q, k1, k2, v1, v2, w, cos, sin, at):
        q, k1, k2 = ft.qk_norm_rotary(q, k1, k2, w, w, w, cos, sin, at)
        if dps:
            ft.dps_append(cache, table, ctx, k1, k2, v1, v2, 0.1, 100)
            out = ft.dps_decode(q, cache, table, ctx, 0.1)
        else:
            ft.cache_write(cache, table, ctx, k1, k2, v1, v2)
            out = ft.tdp_decode(q, cache, table, ctx, 0.1, 30, None, return_lse=True)
        return (*out, *ft.cache_read(cache, table, ctx, 3, torch.float32))

    got = []
    cos, sin = ft.rotary_tables(64, 32, device=DEV)
    w = torch.linspace(0.5, 1.5, 64, device=DEV)
    for run in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        cache, table, ctx, xs = _inputs(dps=dps)
        at = ctx[:, None] + torch.arange(3, device=DEV, dtype=torch.int32)
        got.append([*run(cache, table, ctx, *xs, w, cos, sin, at), *(t for t in cache if t is not None)])
    assert len(got[0]) == len(got[1]) and all(torch.equal(a, b) for a, b in zip(*got))
    ft.check_status(DEV)
