"""Rotary positions on the GPU against the rotation in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# The angle is exact; the sine unit's result is off by less than 2^-18, so a rotated value by gain
# 2^-18 (|a| + |b|) and three fp32 roundings of its products, 2^-22 of them, before its one rounding to bf16 (2^-8).
SINE = 2.0 ** -18 + 2.0 ** -22


def _want(rotary, positions, x, inverse=False):
    """The rotation in 64 bits, and the bound of its error."""
    r = rotary.rotary_dim
    freq = torch.tensor(rotary.frequencies, dtype=torch.float64)
    pos = positions.cpu()
    if pos.dim() == 2:
        pos = pos[rotary._axes.long()].T
    else:
        pos = pos[:, None]
    # positions by frequencies exactly: the whole turns taken off in integers
    turns = [[(int(p) * int(t)) % 2 ** 64 for p, t in zip(row.expand(r // 2).tolist(), [int(f / (2 * math.pi) * 2 ** 64)
                                                                                    for f in freq.tolist()])]
             for row in pos]
    angle = torch.tensor([[2 * math.pi * (t / 2 ** 64) for t in row] for row in turns], dtype=torch.float64).view(-1, r // 2)
    gain = 1 / rotary.gain if inverse else rotary.gain
    c, s = (angle.cos() * gain)[:, None], (angle.sin() * gain * (-1 if inverse else 1))[:, None]
    y = x.double().cpu().clone()
    tol = torch.zeros_like(y)
    first = torch.arange(0, r, 2) if rotary.interleaved else torch.arange(r // 2)
    second = first + (1 if rotary.interleaved else r // 2)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    reach = SINE * gain * (a.abs() + b.abs())
    tol[..., first], tol[..., second] = reach, reach
    tol[..., :r] += 2.0 ** -8 * y[..., :r].abs()
    return y, tol


def _close(got, want, tol):
    over = (got.double().cpu() - want).abs() - tol
    assert over.numel() == 0 or float(over.max()) <= 0, f"{int((over > 0).sum())} values past the bound, by {float(over.max()):.3g}"


def _rows(t, heads, d, seed, pad=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(t, heads, d + pad, generator=gen).bfloat16().cuda()[..., :d]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(256, 64), (128, 128), (256, 256), (128, 66), (256, 6), (96, 2), (80, 80), (64, 30), (512, 512)])
@pytest.mark.parametrize("t,hq,hkv", [(1, 16, 4), (7, 5, 1), (130, 8, 2)])
def test_matches_the_rotation(d, r, t, hq, hkv, interleaved):
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(d, rotary_dim=r, base=1e6, interleaved=interleaved)
    q, k = _rows(t, hq, d, 1), _rows(t, hkv, d, 2)
    pos = torch.arange(t, device="cuda") * 977 + 100003
    got_q, got_k = rotary(pos, q, k)
    for got, x in ((got_q, q), (got_k, k)):
        _close(got, *_want(rotary, pos, x))
        assert torch.equal(got[..., r:], x[..., r:])


def test_rotates_in_place_in_one_buffer_of_queries_and_keys():
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(128, rotary_dim=64)
    both = _rows(40, 6, 128, 3).reshape(40, -1).contiguous()
    q, k = both[:, :512].view(40, 4, 128), both[:, 512:].view(40, 2, 128)
    pos = torch.arange(40, device="cuda") + 70
    want = rotary(pos, q, k)
    rotary(pos, q, k, out_q=q, out_k=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("first", [0, -5000, 2 ** 20 - 3, 2 ** 31 - 2, 2 ** 40 + 12345])
@pytest.mark.parametrize("scaling", [None, dict(kind="linear", factor=4.0), dict(kind="ntk", factor=8.0),
                                     dict(kind="yarn", factor=4.0, original_length=32768),
                                     dict(kind="banded", factor=8.0, original_length=8192)])
def test_far_positions_and_scalings(first, scaling):
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(128, base=10000.0, scaling=scaling)
    q = _rows(5, 2, 128, 3)
    pos = torch.arange(first, first + 5, device="cuda")
    _close(rotary(pos, q), *_want(rotary, pos, q))
    if first + 5 < 2 ** 31:
        assert torch.equal(rotary(pos.int(), q), rotary(pos, q))


@pytest.mark.parametrize("dealt", [False, True])
def test_positions_on_three_axes(dealt):
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(256, rotary_dim=64, base=1e7, sections=(11, 11, 10), sections_interleaved=dealt)
    q, k = _rows(33, 4, 256, 4), _rows(33, 1, 256, 5)
    grid = torch.stack([torch.arange(33) + 70000, torch.arange(33) // 8 + 70000, torch.arange(33) % 8 + 70000]).cuda()
    for pos in (grid, grid.T.contiguous().T, grid.int()):
        got_q, got_k = rotary(pos, q, k)
        _close(got_q, *_want(rotary, grid, q))
        _close(got_k, *_want(rotary, grid, k))


def test_strides_in_place_and_back():
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(128, rotary_dim=64, scaling=dict(kind="yarn", factor=4.0, original_length=4096))
    fused = _rows(50, 1, 12 * 128, 6).view(50, 12 * 128)
    q, k = fused[:, :8 * 128].view(50, 8, 128), fused[:, 8 * 128:10 * 128].view(50, 2, 128)
    pos = torch.randint(0, 100000, (100,), generator=torch.Generator().manual_seed(1)).cuda()[::2]
    want = [t.clone() for t in rotary(pos, q.contiguous(), k.contiguous())]
    got = rotary(pos, q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = _rows(50, 8, 128, 0, pad=3)                   # rows off any 16-byte piece
    odd.copy_(q)
    assert torch.equal(rotary(pos, odd), want[0])
    turned = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(rotary(pos, turned), want[0])
    before = fused.clone()
    rotary(pos, q, k, out_q=q, out_k=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(fused[:, 10 * 128:], before[:, 10 * 128:])
    # back: two roundings of bf16, the first of them turned
    back = rotary(pos, q, inverse=True).double()
    x = before[:, :8 * 128].view(50, 8, 128).double()
    pair = torch.cat([x[..., 32:64].abs(), x[..., :32].abs()], -1)
    tol = 2.0 ** -8 * back[..., :64].abs() + (2.0 ** -8 + 4 * SINE) * (x[..., :64].abs() + pair) * 1.001
    assert bool(((back - x)[..., :64].abs() <= tol).all())
    assert torch.equal(back[..., 64:], x[..., 64:])


def test_no_tokens_and_not_finite_values():
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(64)
    q = _rows(0, 3, 64, 0)
    assert rotary(torch.zeros(0, dtype=torch.int64, device="cuda"), q).shape == (0, 3, 64)
    q = _rows(2, 1, 64, 1)
    q[0, 0, 3] = float("nan")
    got = rotary(torch.tensor([9, 9], device="cuda"), q)
    assert got[0, 0].isnan().nonzero().flatten().tolist() == [3, 35]
    assert torch.isfinite(got[1]).all()


def test_captured_and_on_another_stream():
    from semblo_amd.rotary import RotaryEmbedding
    rotary = RotaryEmbedding(128, rotary_dim=64)
    q, k = _rows(3, 4, 128, 8), _rows(3, 2, 128, 9)
    pos = torch.tensor([5, 6, 7], device="cuda")
    want = rotary(pos, q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary(pos, q, k)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary(pos, q, k)
    for step in range(3):
        pos.add_(1)
        q.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        want = rotary(pos, q, k)
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
