"""Norms with rotation over more tokens than the grids hold at once: every block takes several, across the batch's borders, by copies that run
ahead; and heads in several groups.  Against the 64-bit formula, on the GPU."""
import pytest
import torch

import flash_trittention as ft
from oracle import serving_oracle as orc
from test_norm_rotary import DEV, HALF_STEP, _bound, _close

SMS, THREADS, HEADS = 148, 256, 4   # of the kernels' grids


def _grid(B, N, T, D, dtype, weights):
    """Steps of a block of the backward's grid, blocks of the forward's, groups of a token's heads, and the additions in the longest line of a
    sum over rows."""
    chunks, slots = -(-N // HEADS), THREADS // (D // 8)
    here = min(chunks, slots)
    groups, at_once = -(-chunks // here), slots // here
    blocks = min(-(-B * T // at_once), max(1, (3 if weights == "shared" and dtype != torch.float32 else 2) * SMS // (3 * groups)))
    steps = -(-B * T // (blocks * at_once))
    return steps, -(-B * T * chunks // slots), groups, steps * HEADS + slots + blocks * groups // 32 + 1 + 32


CASES = [  # B N T D dtype weights rot interleaved positions strided
    (3, 8, 3201, 64, torch.bfloat16, "shared", 64, False, True, True),
    (3, 8, 3201, 64, torch.float16, "heads", 32, True, True, False),
    (5, 16, 501, 128, torch.bfloat16, "shared", 128, False, True, True),
    (1201, 16, 7, 128, torch.float16, "shared", 64, True, False, True),     # a step is 84 sequences and 4 tokens
    (901, 13, 11, 128, torch.bfloat16, "heads", 128, False, True, False),
    (3, 37, 67, 256, torch.bfloat16, "heads", 256, False, True, True),      # two groups of a token's heads, the last of five
    (3, 37, 133, 256, torch.float16, "shared", 128, True, True, True),
    (7, 3, 5501, 32, torch.bfloat16, "shared", 32, False, False, False),
    (3, 13, 1601, 128, torch.float16, "shared", 0, False, False, True),
    (5, 6, 5303, 16, torch.float32, "heads", 16, False, True, False),
    (3, 37, 133, 256, torch.float32, "shared", 64, True, True, True),
    (3, 5, 4001, 64, torch.float32, "shared", 64, False, True, True),
]


@pytest.mark.parametrize("case", CASES)
def test_the_cases_are_what_they_are_for(case):
    B, N, T, D, dtype, weights = case[:6]
    assert _grid(B, N, T, D, dtype, weights)[0] >= 4 and T % 2
    assert any(_grid(*c[:6])[1] >= 8 * SMS for c in CASES) and sum(_grid(*c[:6])[2] > 1 for c in CASES) >= 2


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,T,D,dtype,weights,rot,inter,with_positions,strided", CASES)
def test_many_tokens(B, N, T, D, dtype, weights, rot, inter, with_positions, strided):
    g = torch.Generator(device=DEV).manual_seed(B * T)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    new = (lambda: randn(B, T, 5, N, D)[:, :, 2].transpose(1, 2)) if strided else (lambda: randn(B, N, T, D))
    xs, dys = [new() for _ in range(3)], [new() for _ in range(3)]
    ws = [(1 + 0.3 * torch.randn((N, D) if weights == "heads" else (D,), generator=g, device=DEV)).to(dtype) for _ in range(3)]
    cos, sin = ft.rotary_tables(8192, rot, device=DEV) if rot else (None, None)
    positions = torch.randint(0, 8192, (B, T), generator=g, device=DEV) if rot and with_positions else None
    leaves = [t.detach().requires_grad_(True) for t in xs + ws]
    out = ft.qk_norm_rotary(*leaves, cos, sin, positions, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, dys)
    ft.check_status(DEV)
    line = _grid(B, N, T, D, dtype, weights)[3]
    for i in range(3):
        # a weight for each row: its gradient's terms
        x = xs[i].double().requires_grad_(True)
        w = (ws[i].double()[None, :, None] if weights == "heads" else ws[i].double()).expand(B, N, T, D).clone().requires_grad_(True)
        ref = orc.norm_rotary(x, None, None, None, None) * w
        if rot:
            ref = _turned(ref, cos, sin, positions, inter)
        dx, terms = torch.autograd.grad(ref, [x, w], dys[i].double())
        ref = ref.detach().cpu()
        _close(out[i], ref, _bound(dtype, ref, ref.abs().amax(-1, keepdim=True)))
        # dx = r (g - h mean(g h)), as in the tests of few tokens
        r = (x.detach().pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
        size = dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * float(w.detach().abs().max())
        h = (x.detach() * r).abs().amax(-1, keepdim=True)
        assert grads[i].shape == xs[i].shape
        _close(grads[i], dx.cpu(), _bound(dtype, dx, r * size * (1 + h * h)).cpu())
        # a sum over rows in fp32: 2^-24 of the absolute sum for each addition in a line, and of each term what leads to it (its own
        # size and the largest of its row's: a rotated pair's other half)
        over = (0, 2) if weights == "heads" else (0, 1, 2)
        want, mass = terms.sum(over), (terms.abs().sum(over), (dys[i].double().abs().amax(-1, keepdim=True) * 1.5 * h).expand(B, N, T, D).sum(over))
        _close(grads[3 + i], want.cpu(), (HALF_STEP[dtype] * want.abs() + 2.0 ** -24 * (line * mass[0] + 64 * mass[1]) + 1e-30).cpu())


def _turned(u, cos, sin, positions, interleaved):
    """The rotation alone, of 64-bit rows."""
    B, N, T, D = u.shape
    at = torch.arange(T, device=u.device).expand(B, T) if positions is None else positions
    c, s, half = cos.double()[at][:, None], sin.double()[at][:, None], cos.shape[1]
    head = u[..., : 2 * half]
    a, b = (head[..., ::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2) if interleaved else torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, u[..., 2 * half:]), -1)
