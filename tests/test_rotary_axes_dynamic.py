"""Calls of the norms, the weights and the eviction in graphs whose sizes are symbols, traced without a GPU on the meta device."""
import pytest
import torch

import flash_trittention as ft


def _traced(f, *args):
    """What f returns when it is traced with symbols for its tensors' sizes, and how many graphs it was traced into."""
    graphs = []
    torch._dynamo.reset()

    def backend(graph, inputs):
        graphs.append(graph)
        return graph.forward

    out = torch.compile(f, fullgraph=True, dynamic=True, backend=backend)(*args)
    return out, len(graphs)


def _rows(B, N, T, D, count):
    return [torch.empty(B, N, T, D, dtype=torch.bfloat16, device="meta") for _ in range(count)]


@pytest.mark.parametrize("batched", [False, True])
@pytest.mark.parametrize("given", ["closure", "argument"])
def test_axes_of_positions(given, batched):
    B, N, T, D = 3, 5, 33, 64
    axes = ft.rotary_axes((8, 4, 4), mixed=True)
    tables = [torch.empty(99, 16, device="meta") for _ in range(2)]
    positions = torch.empty(*((3, B, T) if batched else (3, T)), dtype=torch.int64, device="meta")

    def f(q, k1, k2, cos, sin, positions, axes=axes):
        return ft.qk_norm_rotary(q, k1, k2, None, None, None, cos, sin, positions, axes=axes)

    out, graphs = _traced(f, *_rows(B, N, T, D, 3), *tables, positions, *((axes,) if given == "argument" else ()))
    assert graphs == 1 and [t.shape for t in out] == [(B, N, T, D)] * 3


def test_axes_with_gradients():
    B, N, T, D = 3, 5, 33, 64
    axes = ft.rotary_axes((8, 4, 4))
    q, k1, k2 = (t.requires_grad_(True) for t in _rows(B, N, T, D, 3))
    weight = torch.empty(D, device="meta", requires_grad=True)
    positions, tables = torch.empty(3, T, dtype=torch.int32, device="meta"), [torch.empty(99, 16, device="meta") for _ in range(2)]
    torch._dynamo.reset()
    f = torch.compile(lambda *a: ft.qk_norm_rotary(*a[:3], weight, weight, None, *tables, a[3], axes=axes), fullgraph=True, dynamic=True, backend="aot_eager")
    out = f(q, k1, k2, positions)
    torch.autograd.backward(out, [torch.empty_like(o) for o in out])
    assert q.grad.shape == k2.grad.shape == (B, N, T, D) and weight.grad.shape == (D,)


def test_axes_that_do_not_fit_are_refused_as_ever():
    q, k1, k2 = _rows(1, 2, 9, 64, 3)
    positions, tables = torch.empty(2, 9, dtype=torch.int32, device="meta"), [torch.empty(99, 16, device="meta") for _ in range(2)]
    for axes in ((0,) * 15, (0,) * 17, (0,) * 15 + (4,), (0,) * 15 + (-1,), ()):
        with pytest.raises(ValueError):
            ft.qk_norm_rotary(q, k1, k2, None, None, None, *tables, positions, axes=axes)
    with pytest.raises(ValueError):
        ft.qk_norm_rotary(q, k1, k2, axes=(0,) * 16)


def test_weights_and_eviction():
    B, N, n, D = 3, 5, 2, 64
    cache = ft.new_cache(40, 16, N, D, torch.int8, "meta", dps=True)
    q, k2 = _rows(B, N, n, D, 2)
    sums, weights = torch.empty(B, N, n, device="meta"), torch.empty(B, N, 90, device="meta")
    table, context = torch.empty(B, 6, dtype=torch.int32, device="meta"), torch.empty(B, dtype=torch.int32, device="meta")

    def f(weights, q, k2, sums, codes, exponents, lse, table, context):
        c = ft.TrittentionCache(codes, exponents, lse)
        ft.tdp_weigh(weights, q, sums, c, table, context, 0.1, 20)
        ft.dps_weigh(weights, q, k2, sums, c, table, context, 0.1, 50)
        return ft.cache_evict(weights, c, table, context + n, weights.shape[2] // 3, 1, 2)

    (left, kept), graphs = _traced(f, weights, q, k2, sums, *cache, table, context)
    assert graphs == 1 and left.shape == (B,) and kept.shape == (B, N, 30)


@pytest.mark.gpu
@pytest.mark.parametrize("dynamic", [None, True])
def test_axes_compiled_for_several_lengths(dynamic):
    """One function for sequences of several lengths: results and gradients as without it."""
    axes = ft.rotary_axes((8, 4, 4), mixed=True)
    cos, sin = ft.rotary_tables(99, 32, device="cuda:0")
    step = lambda q, k1, k2, w, at: ft.qk_norm_rotary(q, k1, k2, w, None, w, cos, sin, at, axes=axes)  # noqa: E731
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, dynamic=dynamic, backend="aot_eager")
    for B, T in ((2, 33), (2, 40), (3, 7)):
        got = []
        for f in (step, compiled):
            g = torch.Generator().manual_seed(T)
            q, k1, k2 = (torch.randn(B, 4, T, 64, generator=g).to("cuda:0", torch.bfloat16).requires_grad_(True) for _ in range(3))
            w = torch.randn(64, generator=g).to("cuda:0").requires_grad_(True)
            out = f(q, k1, k2, w, torch.randint(0, 99, (3, B, T), generator=g).to("cuda:0"))
            torch.autograd.backward(out, [torch.ones_like(o) for o in out])
            got.append([*(o.detach() for o in out), q.grad, k1.grad, k2.grad, w.grad])
        assert all(torch.equal(a, b) for a, b in zip(*got))
    ft.check_status("cuda:0")
