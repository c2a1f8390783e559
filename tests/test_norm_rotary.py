"""Norms of q, k1, k2 with the position rotation, against the 64-bit formula and, for gradients, against its differences."""
import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native
from oracle import serving_oracle as orc

DEV = "cuda:0"
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def _inputs(B, N, T, D, dtype, weights, rot, seed=0, strided=False, table=64, wtype=None):
    g = torch.Generator().manual_seed(seed)
    if strided:   # the parts of one projection
        x = torch.randn(B, T, 5, N, D, generator=g).to(dtype)
        xs = [x[:, :, i].transpose(1, 2) for i in (0, 1, 3)]
    else:
        xs = [torch.randn(B, N, T, D, generator=g).to(dtype) for _ in range(3)]
    shape = {"none": None, "shared": (D,), "heads": (N, D)}[weights]
    ws = [None if shape is None else (1 + 0.3 * torch.randn(shape, generator=g)).to(wtype or dtype) for _ in range(3)]
    cos = sin = None
    if rot:
        cos, sin = ft.rotary_tables(table, rot)
    return xs, ws, cos, sin


def _bound(dtype, ref, largest):
    """Result rounded once (half a step of its value); before that a dozen fp32 operations on numbers up to `largest`, the sum of D squares
    (relative error below D 2^-24 / 2 after the root, in a tree much less) and rsqrt of two units: 64 half steps of fp32 cover them."""
    return HALF_STEP[dtype] * ref.abs() + 64 * 2.0 ** -24 * largest + 1e-30


def _close(got, ref, bound):
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f"off by {float((err - bound).max()):.3e} over the bound at {int((err > bound).sum())} of {err.numel()}"


def _dev(t):
    return None if t is None else t.to(DEV)


CASES = [  # B N T D dtype weights rot interleaved strided positions
    (1, 1, 1, 64, torch.bfloat16, "shared", 64, False, False, None),
    (2, 5, 33, 64, torch.float16, "heads", 32, True, True, None),
    (3, 4, 17, 128, torch.bfloat16, "shared", 128, False, True, "batch"),
    (2, 3, 40, 16, torch.float32, "heads", 16, False, False, "shared"),
    (1, 7, 9, 256, torch.float16, "none", 256, True, True, "batch32"),
    (2, 9, 21, 32, torch.float32, "shared", 0, False, True, None),
    (1, 16, 64, 128, torch.float16, "heads", 48, False, False, "batch"),
    (4, 2, 5, 256, torch.float32, "shared", 16, False, True, "shared"),
    (1, 2, 50, 64, torch.bfloat16, "none", 0, False, False, None),
]


def _positions(kind, B, T, table):
    if kind is None:
        return None
    g = torch.Generator().manual_seed(3)
    p = torch.randint(0, table, (T,) if kind == "shared" else (B, T), generator=g)
    return p.int() if kind == "batch32" else p


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,T,D,dtype,weights,rot,inter,strided,pos", CASES)
@pytest.mark.parametrize("wide_weights", [False, True])
def test_forward_and_gradients(B, N, T, D, dtype, weights, rot, inter, strided, pos, wide_weights):
    xs, ws, cos, sin = _inputs(B, N, T, D, dtype, weights, rot, strided=strided, wtype=torch.float32 if wide_weights else None)
    positions = _positions(pos if rot else None, B, T, 64)
    dys = [torch.randn(B, N, T, D, generator=torch.Generator().manual_seed(9 + i)).to(dtype) for i in range(3)]
    leaves = [x.to(DEV).requires_grad_(True) for x in xs]
    wl = [None if w is None else w.to(DEV).requires_grad_(True) for w in ws]
    out = ft.qk_norm_rotary(*leaves, *wl, _dev(cos), _dev(sin), _dev(positions), interleaved=inter)
    given = [w for w in wl if w is not None]
    grads = torch.autograd.grad(out, leaves + given, [d.to(DEV) for d in dys])
    with torch.no_grad():   # the direct call: the same kernel
        again = ft.qk_norm_rotary(*leaves, *wl, _dev(cos), _dev(sin), _dev(positions), interleaved=inter)
    for i in range(3):
        assert out[i].is_contiguous() and torch.equal(out[i], again[i])
        x = xs[i].double().requires_grad_(True)
        w = None if ws[i] is None else ws[i].double().requires_grad_(True)
        ref = orc.norm_rotary(x, w, cos, sin, positions, interleaved=inter)
        want = torch.autograd.grad(ref, [x] + ([w] if w is not None else []), dys[i].double())
        _close(out[i], ref.detach(), _bound(dtype, ref.detach(), ref.detach().abs().amax(-1, keepdim=True)))
        # dx = r (g - h mean(g h)): sums of D terms as large as |g|, |h| times a row's
        r = (x.detach().pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
        g = dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * (1 if w is None else float(w.detach().abs().max()))
        h = (x.detach() * r).abs().amax(-1, keepdim=True)
        assert grads[i].shape == xs[i].shape
        _close(grads[i], want[0], _bound(dtype, want[0], r * g * (1 + h * h)))
        if w is not None:
            # a sum over rows: fp32, its error below 2^-24 times the rows' absolute sum times the additions in a line (64 at most here)
            size = (dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * h).expand(B, N, T, D).sum((0, 2) if w.dim() == 2 else (0, 1, 2))
            _close(grads[3 + i], want[1], HALF_STEP[ws[i].dtype] * want[1].abs() + 64 * 2.0 ** -24 * size + 1e-30)


@pytest.mark.gpu
def test_gradient_against_differences():
    xs, ws, cos, sin = _inputs(1, 2, 3, 16, torch.float32, "heads", 16)
    leaves = [t.to(DEV).requires_grad_(True) for t in xs + ws]
    out = ft.qk_norm_rotary(*leaves, cos.to(DEV), sin.to(DEV))
    dys = [torch.randn(o.shape, generator=torch.Generator().manual_seed(i)).to(DEV) for i, o in enumerate(out)]
    grads = torch.autograd.grad(out, leaves, dys)
    for k, leaf in enumerate(leaves):
        step = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(50 + k))
        moved = [t.detach().double().cpu() for t in leaves]
        f = lambda e: sum((orc.norm_rotary(moved[i] + (e * step.double() if k == i else 0), moved[3 + i] + (e * step.double() if k == 3 + i else 0),  # noqa: E731
                                           cos, sin, None) * dys[i].double().cpu()).sum() for i in range(3))
        slope = float((f(1e-4) - f(-1e-4)) / 2e-4)
        assert abs(slope - float((grads[k].double().cpu() * step.double()).sum())) < 1e-4 * (1 + float((grads[k].double().cpu() * step.double()).abs().sum()))


@pytest.mark.gpu
def test_a_gradient_that_is_missing_or_expanded():
    xs, ws, cos, sin = _inputs(2, 3, 11, 64, torch.float32, "shared", 64)
    leaves = [t.to(DEV).requires_grad_(True) for t in xs + ws]
    out = ft.qk_norm_rotary(*leaves, cos.to(DEV), sin.to(DEV))
    got = torch.autograd.grad(out[1].sum(), leaves, allow_unused=True)   # (an expanded gradient; none for the other two results)
    x, w = xs[1].double().requires_grad_(True), ws[1].double().requires_grad_(True)
    ref = torch.autograd.grad(orc.norm_rotary(x, w, cos, sin, None).sum(), [x, w])
    _close(got[1], ref[0], 2.0 ** -14 * (1 + ref[0].abs()))
    _close(got[4], ref[1], 2.0 ** -14 * (1 + ref[1].abs()))
    assert all(float(got[i].abs().max()) == 0 for i in (0, 2, 3, 5))


@pytest.mark.gpu
def test_rows_that_are_zero_infinite_or_tiny():
    x = torch.randn(1, 2, 6, 64, generator=torch.Generator().manual_seed(0))
    x[0, 0, 0] = 0
    x[0, 0, 1, 5] = float("inf")
    x[0, 1, 2, 7] = float("nan")
    x[0, 1, 3] *= 1e-12
    y = ft.qk_norm_rotary(*(x.to(DEV),) * 3)[2].cpu()
    assert float(y[0, 0, 0].abs().max()) == 0
    assert bool(torch.isnan(y[0, 0, 1, 5])) and bool(torch.isnan(y[0, 1, 2]).all())
    rest = torch.ones(1, 2, 6, dtype=torch.bool)
    rest[0, 0, 1] = rest[0, 1, 2] = False
    ref = orc.norm_rotary(x.double(), None, None, None, None)
    _close(y[rest], ref[rest], 2.0 ** -18 * (1e-9 + ref[rest].abs()))


@pytest.mark.gpu
def test_a_position_outside_the_tables_is_reported():
    xs, ws, cos, sin = _inputs(1, 1, 4, 32, torch.float16, "none", 32, table=8)
    at = torch.tensor([0, 8, -1, 7], device=DEV)
    out = ft.qk_norm_rotary(*(x.to(DEV) for x in xs), cos=cos.to(DEV), sin=sin.to(DEV), positions=at)
    with pytest.raises(_native.TrittError, match="position"):
        ft.check_status(DEV)
    kept = ft.qk_norm_rotary(*(x.to(DEV) for x in xs), cos=cos.to(DEV), sin=sin.to(DEV), positions=torch.tensor([0, 7, 0, 7], device=DEV))
    ft.check_status(DEV)
    assert all(torch.equal(a, b) for a, b in zip(out, kept))


@pytest.mark.gpu
def test_repeats_itself_and_is_captured():
    xs, ws, cos, sin = _inputs(2, 6, 300, 64, torch.bfloat16, "heads", 64, table=300)
    args = [t.to(DEV).requires_grad_(True) for t in xs + ws]
    tables = cos.to(DEV), sin.to(DEV)
    dys = [torch.randn(2, 6, 300, 64, device=DEV).bfloat16() for _ in range(3)]

    def step():
        return torch.autograd.grad(ft.qk_norm_rotary(*args, *tables), args, dys)

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    del want
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for t in args:
            t.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_calls_by_the_extension_and_by_the_python_code(dtype, monkeypatch):
    _native.lib()
    _native.status_word(DEV)
    assert _native._host is not None, "the host extension is not built"
    xs, ws, cos, sin = _inputs(2, 3, 20, 64, dtype, "heads", 32, strided=True)
    args = [t.to(DEV).requires_grad_(True) for t in xs] + [torch.nn.Parameter(w.to(DEV)) for w in ws]
    positions = torch.arange(40, device=DEV).view(2, 20)
    dys = [torch.randn(2, 20, 3, 64, device=DEV).to(dtype).transpose(1, 2) for _ in range(3)]

    def calls():
        y = ft.qk_norm_rotary(*args, cos.to(DEV), sin.to(DEV), positions, interleaved=True)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, args, dys))

    taken = []
    for name in ("host_norm_rotary", "host_norm_rotary_backward"):
        f = getattr(_native._host, name[5:])
        monkeypatch.setattr(_native, name, lambda *a, f=f: taken.append(f(*a)) or taken[-1])
    fast = calls()
    assert len(taken) == 2 and all(r is not None for r in taken)
    for name in ("host_norm_rotary", "host_norm_rotary_backward"):
        monkeypatch.setattr(_native, name, lambda *a: None)
    slow = calls()
    assert all(torch.equal(a, b) and a.stride() == b.stride() for a, b in zip(fast, slow))
    # rows off 16-byte boundaries are copied, their gradients come back in their own layout
    store = torch.empty(xs[0].numel() + 1, dtype=dtype, device=DEV)
    odd = store[1:].view(2, 20, 3, 64).copy_(xs[0].to(DEV).transpose(1, 2)).transpose(1, 2).requires_grad_(True)
    y = ft.qk_norm_rotary(odd, *args[1:], cos.to(DEV), sin.to(DEV), positions, interleaved=True)
    again = torch.autograd.grad(y, [odd], dys)[0]
    assert torch.equal(y[0], fast[0]) and torch.equal(again, fast[3])


@pytest.mark.gpu
def test_in_front_of_both_attentions():
    """One training step of norm, rotation and attention: gradients reach the projections' parts."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(2, 40, 5, 3, 64, generator=g, device=DEV).half().requires_grad_(True)
    w = torch.ones(64, device=DEV, dtype=torch.float16, requires_grad=True)
    cos, sin = ft.rotary_tables(40, 64, device=DEV)
    for attend in (lambda *a: ft.flash_trittention(*a, 1 / 8, None, None, None, None), lambda *a: ft.TrittentionTriton()(*a)[0]):
        q, k1, k2, v1, v2 = x.transpose(1, 3).unbind(2)
        o = attend(*ft.qk_norm_rotary(q, k1, k2, w, w, w, cos, sin), v1, v2)
        dx, dw = torch.autograd.grad(o.float().square().sum(), [x, w])
        assert dx.shape == x.shape and bool(torch.isfinite(dx).all()) and float(dw.abs().max()) > 0


def test_refusals():
    x = torch.zeros(1, 2, 4, 64)
    cos, sin = ft.rotary_tables(4, 64)
    ok = dict(cos=cos, sin=sin)
    for args, kw, what in [
        ((x[0], x[0], x[0]), {}, "expected"), ((x, x, x[:, :1]), {}, "k2"), ((x, x.half(), x), {}, "k1"),
        ((x[..., :48],) * 3, {}, "head_dim"), ((x, x, x, torch.ones(32)), {}, "weights"),
        ((x, x, x, torch.ones(64), torch.ones(2, 64)), {}, "weights"), ((x, x, x, torch.ones(64).half()), {}, "weights"),
        ((x, x, x), dict(cos=cos), "together"), ((x, x, x), dict(cos=cos[:2], sin=sin[:2]), "sequence"),
        ((x, x, x), dict(cos=cos.double(), sin=sin.double()), "float32"), ((x, x, x), dict(cos=cos[:, :4], sin=sin[:, :4]), "multiple of 16"),
        ((x, x, x), dict(positions=torch.zeros(4).long()), "without"), ((x, x, x), dict(positions=torch.zeros(4), **ok), "positions"),
        ((x, x, x), dict(positions=torch.zeros(2, 4).long(), **ok), "positions"), ((x, x, x), dict(eps=float("nan")), "eps"),
        ((x, x, x), dict(eps=-1), "eps"), ((x[:, :, :0],) * 3, {}, "empty"),
    ]:
        with pytest.raises(ValueError, match=what):
            ft.qk_norm_rotary(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        ft.qk_norm_rotary(x, x, x, **ok)
    for length, rot in ((0, 64), (4, 0), (4, 8)):
        with pytest.raises(ValueError):
            ft.rotary_tables(length, rot)


def test_tables_of_far_positions():
    cos, sin = ft.rotary_tables(200001, 16, base=10000.0)
    import math
    for i in range(8):
        angle = 200000 * 10000.0 ** (-i / 8)
        assert abs(float(cos[200000, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[200000, i]) - math.sin(angle)) < 1e-7


def test_the_librarys_own_refusals():
    lib, C = _native.lib(), _native.C
    p = 1 << 20
    rows = lambda: (_native.Rows * 3)(*(_native.Rows(p, 64, 64, 64) for _ in range(3)))  # noqa: E731
    good = lambda **kw: _native.NormRotary(**{**dict(x=rows(), y=rows(), dx=rows(), B=1, N=1, T=1, D=64, dtype=1), **kw})  # noqa: E731
    for kw, rc in [(dict(B=0), -1), (dict(D=48), -2), (dict(dtype=5), -3), (dict(weight_dtype=2), -3), (dict(rot=8), -13),
                   (dict(rot=128), -13), (dict(rot=16), -13), (dict(rot=16, cos=p, sin=p, table=0), -13), (dict(cos=p, sin=p, rot=16, table=1, T=2), -13)]:
        a = good(**kw)
        assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == rc, kw
    a = good()
    a.x[1].p = None
    assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == -4
    a = good()
    a.y[2].stride_n = 4
    assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == -5
    a = good()
    a.w[0] = p + 8
    assert lib.tritt_qk_norm_rotary_fwd(C.byref(a), None, None) == -5
    a = good()
    a.w[0] = a.dw[0] = p
    assert lib.tritt_qk_norm_rotary_workspace(C.byref(a)) > 0
    assert lib.tritt_qk_norm_rotary_bwd(C.byref(a), None, 0, None, None) == -6
    assert lib.tritt_qk_norm_rotary_fwd(None, None, None) == -1
