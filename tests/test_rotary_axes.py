"""The rotation by positions of several axes, against the 64-bit formula and, for gradients, against its differences."""
import pytest
import torch

import flash_trittention as ft
from flash_trittention import _native, norm_rotary as nr, ops
from oracle import serving_oracle as orc
from tests.test_norm_rotary import HALF_STEP, _bound, _close, _dev, _inputs

DEV = "cuda:0"

CASES = [  # B N T D dtype weights axes interleaved strided positions' shape
    (1, 1, 1, 64, torch.bfloat16, "shared", ft.rotary_axes((8, 12, 12)), False, False, "shared"),
    (2, 5, 33, 64, torch.float16, "heads", ft.rotary_axes((8, 8)), True, True, "batch"),
    (3, 4, 17, 128, torch.bfloat16, "shared", ft.rotary_axes((24, 20, 20), mixed=True), False, True, "batch"),
    (2, 3, 40, 16, torch.float32, "heads", ft.rotary_axes((1, 3, 2, 2)), False, False, "shared"),
    (1, 7, 9, 256, torch.float16, "none", ft.rotary_axes((33, 0, 95), mixed=True), True, True, "batch32"),
    (4, 2, 5, 256, torch.float32, "shared", (3, 0, 3, 2, 1, 1, 0, 0), False, True, "shared"),
    (2, 3, 6, 32, torch.bfloat16, "shared", (0,) * 8, False, False, "batch"),
]


def _positions(kind, count, B, T, table):
    p = torch.randint(0, table, (count, T) if kind == "shared" else (count, B, T), generator=torch.Generator().manual_seed(3))
    return p.int() if kind == "batch32" else p


def test_axes_of_pairs():
    assert ft.rotary_axes((2, 3)) == (0, 0, 1, 1, 1)
    assert ft.rotary_axes((4, 2, 2), mixed=True) == (0, 1, 2, 0, 1, 2, 0, 0)
    assert ft.rotary_axes((0, 8)) == (1,) * 8
    for bad in ((), (0, 0), (1, -1), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError):
            ft.rotary_axes(bad)
    packed = nr._pack_axes((3, 0, 3, 2, 1), 5)
    assert packed[0] == 4 and packed[1] == 3 | 3 << 4 | 2 << 6 and packed[2] == 1 and len(packed) == 33


def test_tables_of_axes():
    axes = ft.rotary_axes((4, 4))
    cos, sin = ft.rotary_tables(20, 16, axes=axes)
    one, _ = ft.rotary_tables(20, 16)
    assert torch.equal(cos[:, :4], cos[:, 4:]) and torch.equal(cos[:, 1], one[:, 2])   # four speeds 10000^(-r / 4), the second and each other of eight
    with pytest.raises(ValueError):
        ft.rotary_tables(20, 16, axes=(0,) * 7)


def test_refusals():
    xs, ws, cos, sin = _inputs(2, 3, 10, 64, torch.float32, "shared", 32)
    axes, p = ft.rotary_axes((8, 8)), torch.zeros(2, 10, dtype=torch.int64)
    call = lambda c=cos, s=sin, at=p, a=axes: ft.qk_norm_rotary(*xs, *ws, c, s, at, axes=a)  # noqa: E731
    for kw in (dict(a=axes[:15]), dict(a=(0,) * 15 + (4,)), dict(a=(0,) * 15 + (-1,)), dict(at=None), dict(at=p[0]), dict(at=p[:1]), dict(at=p[:, :9]),
               dict(at=torch.zeros(5, 10, dtype=torch.int64)), dict(at=p.float()), dict(at=torch.zeros(2, 3, 10, dtype=torch.int32)), dict(c=None, s=None)):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):   # a proper call, of CPU tensors
        call()


def test_the_library_refuses_what_it_cannot_read():
    L = _native.lib()
    x = torch.zeros(1, 1, 2, 16)
    a, keep = nr._arguments((x, x, x), (None,) * 3, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(2, 2, dtype=torch.int64), 1e-6, False, b"")
    for i in range(3):
        a.y[i] = a.x[i]
    good = dict(position_stride=2, count=2)
    for change in (dict(count=0), dict(count=5), dict(of=(2,) + (0,) * 31), dict(of=(0, 128) + (0,) * 30)):
        x = _native.Axes(**{**good, **{k: v for k, v in change.items() if k != "of"}}, of=(_native.C.c_ubyte * 32)(*change.get("of", (0,) * 32)))
        assert L.tritt_qk_norm_rotary_axes_fwd(a, x, None, None) == -13
    assert L.tritt_qk_norm_rotary_axes_fwd(a, None, None, None) == -13
    a.positions = None
    assert L.tritt_qk_norm_rotary_axes_fwd(a, _native.Axes(**good), None, None) == -13


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,T,D,dtype,weights,axes,inter,strided,pos", CASES)
@pytest.mark.parametrize("host", [True, False])
def test_forward_and_gradients(B, N, T, D, dtype, weights, axes, inter, strided, pos, host, monkeypatch):
    _native.lib()
    if not host:
        monkeypatch.setattr(_native, "host_norm_rotary", lambda *a: None)
        monkeypatch.setattr(_native, "host_norm_rotary_backward", lambda *a: None)
    xs, ws, cos, sin = _inputs(B, N, T, D, dtype, weights, 2 * len(axes), strided=strided)
    positions = _positions(pos, max(axes) + 1, B, T, 64)
    dys = [torch.randn(B, N, T, D, generator=torch.Generator().manual_seed(9 + i)).to(dtype) for i in range(3)]
    leaves = [x.to(DEV).requires_grad_(True) for x in xs]
    wl = [None if w is None else w.to(DEV).requires_grad_(True) for w in ws]
    out = ft.qk_norm_rotary(*leaves, *wl, _dev(cos), _dev(sin), _dev(positions), interleaved=inter, axes=axes)
    grads = torch.autograd.grad(out, leaves + [w for w in wl if w is not None], [d.to(DEV) for d in dys])
    for i in range(3):
        x = xs[i].double().requires_grad_(True)
        w = None if ws[i] is None else ws[i].double().requires_grad_(True)
        ref = orc.norm_rotary(x, w, cos, sin, positions, interleaved=inter, axes=axes)
        want = torch.autograd.grad(ref, [x] + ([w] if w is not None else []), dys[i].double())
        # (the bounds of the rotation with one axis: the arithmetic is the same)
        _close(out[i], ref.detach(), _bound(dtype, ref.detach(), ref.detach().abs().amax(-1, keepdim=True)))
        r = (x.detach().pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
        g = dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * (1 if w is None else float(w.detach().abs().max()))
        h = (x.detach() * r).abs().amax(-1, keepdim=True)
        _close(grads[i], want[0], _bound(dtype, want[0], r * g * (1 + h * h)))
        if w is not None:
            size = (dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * h).expand(B, N, T, D).sum((0, 2) if w.dim() == 2 else (0, 1, 2))
            _close(grads[3 + i], want[1], HALF_STEP[ws[i].dtype] * want[1].abs() + 64 * 2.0 ** -24 * size + 1e-30)
    ft.check_status(DEV)


@pytest.mark.gpu
def test_gradient_against_differences():
    axes, positions = ft.rotary_axes((3, 5), mixed=True), torch.tensor([[5, 9, 60], [0, 33, 2]])
    xs, ws, cos, sin = _inputs(1, 2, 3, 16, torch.float32, "heads", 16)
    leaves = [t.to(DEV).requires_grad_(True) for t in xs + ws]
    out = ft.qk_norm_rotary(*leaves, cos.to(DEV), sin.to(DEV), positions.to(DEV), axes=axes)
    dys = [torch.randn(o.shape, generator=torch.Generator().manual_seed(i)).to(DEV) for i, o in enumerate(out)]
    grads = torch.autograd.grad(out, leaves, dys)
    for k, leaf in enumerate(leaves):
        step = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(50 + k))
        moved = [t.detach().double().cpu() for t in leaves]
        f = lambda e: sum((orc.norm_rotary(moved[i] + (e * step.double() if k == i else 0), moved[3 + i] + (e * step.double() if k == 3 + i else 0),  # noqa: E731
                                           cos, sin, positions, axes=axes) * dys[i].double().cpu()).sum() for i in range(3))
        slope = float((f(1e-4) - f(-1e-4)) / 2e-4)
        assert abs(slope - float((grads[k].double().cpu() * step.double()).sum())) < 1e-4 * (1 + float((grads[k].double().cpu() * step.double()).abs().sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
def test_equal_axes_are_one_axis(inter):
    """All axes at the same position, in any order of pairs, give what one axis gives, bit for bit."""
    xs, ws, cos, sin = _inputs(2, 3, 50, 64, torch.bfloat16, "shared", 64, strided=True)
    args = [_dev(t) for t in (*xs, *ws, cos, sin)]
    p = torch.randint(0, 64, (2, 50), device=DEV)
    want = ft.qk_norm_rotary(*args, p, interleaved=inter)
    for axes in (ft.rotary_axes((16, 8, 8)), ft.rotary_axes((11, 11, 10), mixed=True)):
        got = ft.qk_norm_rotary(*args, p.expand(3, 2, 50), interleaved=inter, axes=axes)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_positions_that_the_tables_do_not_have():
    xs, ws, cos, sin = _inputs(1, 2, 4, 64, torch.float32, "none", 64)
    axes = ft.rotary_axes((16, 16), mixed=True)
    p = torch.tensor([[0, 1, 2, 64], [-1, 3, 0, 0]])
    got = ft.qk_norm_rotary(*[_dev(x) for x in xs], None, None, None, _dev(cos), _dev(sin), _dev(p), axes=axes)
    with pytest.raises(_native.TrittError):
        ft.check_status(DEV)
    ref = orc.norm_rotary(xs[0].double(), None, cos, sin, p, axes=axes)   # (the nearest rows of the tables)
    _close(got[0], ref, _bound(torch.float32, ref, ref.abs().amax(-1, keepdim=True)))
    # an axis that no pair has is not read
    ft.qk_norm_rotary(*[_dev(x) for x in xs], None, None, None, _dev(cos), _dev(sin), _dev(torch.stack((p[0] * 0, p[0] + 1000))), axes=(0,) * 32)
    ft.check_status(DEV)


@pytest.mark.gpu
def test_compiled_captured_and_on_another_stream():
    xs, ws, cos, sin = _inputs(2, 3, 20, 64, torch.bfloat16, "shared", 32)
    axes = ft.rotary_axes((4, 6, 6))
    args = [_dev(t) for t in (*xs, *ws, cos, sin)]
    p = _dev(_positions("batch", 3, 2, 20, 64))
    want = ft.qk_norm_rotary(*args, p, axes=axes)
    f = torch.compile(lambda *a: ft.qk_norm_rotary(*a, axes=axes), fullgraph=True, backend="aot_eager")
    leaves = [t.clone().requires_grad_(True) for t in args[:6]]
    dys = [torch.randn_like(w) for w in want]
    eager = [t.clone().requires_grad_(True) for t in args[:6]]
    y, z = f(*leaves, *args[6:], p), ft.qk_norm_rotary(*eager, *args[6:], p, axes=axes)
    assert all(torch.equal(a, b) for a, b in zip(want, y))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dys), torch.autograd.grad(z, eager, dys)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ft.qk_norm_rotary(*args, p, axes=axes)
    p.neg_().add_(63)   # (the positions are read on the device)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ft.qk_norm_rotary(*args, p, axes=axes)))
    torch.library.opcheck(torch.ops.flash_trittention.norm_rotary.default, (*[t.clone().requires_grad_(True) for t in args[:6]], *args[6:], p, 1e-6, False, list(axes)),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    with pytest.raises(NotImplementedError):
        ops.norm_rotary(*xs, *ws, cos, sin, p.cpu(), 1e-6, False, list(axes))
