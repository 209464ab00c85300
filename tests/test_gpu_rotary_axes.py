"""Rotary positions on several axes against the rotation in 64 bits (tolerances as in test_gpu_rotary.py): each pair by its own axis's position."""
import pytest
import torch

from conftest import seeded_bf16
from plain_operators import host  # noqa: F401
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu


def angles(cos, sin, positions, axes):
    """cos, sin [B,S,1,pairs] of positions [A,B,S] on the CPU."""
    at = positions.long()[torch.tensor(axes)].permute(1, 2, 0)
    i = torch.arange(len(axes))
    return cos[at, i][:, :, None], sin[at, i][:, :, None]


def axes_by_hand(sections, order):
    if order == "sections":
        return sum(([a] * n for a, n in enumerate(sections)), [])
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


CASES = [(128, (24, 20, 20)), (128, (16, 24, 24)), (72, (18, 18)), (64, (5, 3, 7, 1)), (80, (0, 8, 24)), (34, (1, 2)), (256, (64, 32, 32)), (512, (256,)), (512, (64, 64, 64, 64)), (2, (1,)),
         (96, (3, 13))]


@pytest.mark.parametrize("D, sections", CASES)
@pytest.mark.parametrize("order", ["sections", "rounds"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rotation_and_gradients(D, sections, order, layout, dtype, host):
    """q and k are column slices of one product, gradients come with heads in front of tokens."""
    from lingua_amd import rope
    B, S, H, K, P = 2, 9, 3, 2, 500
    half, axes = layout == "half", axes_by_hand(sections, order)
    assert rope.pair_axes(sections, order) == axes
    cos, sin = rope.rotary_tables(2 * len(axes), P)
    y = seeded_bf16((B * S, (H + 2 * K) * D), seed=1).cuda()
    q = y[:, :H * D].view(B, S, H, D).detach().requires_grad_()
    k = y[:, H * D:(H + K) * D].view(B, S, K, D).detach().requires_grad_()
    pos = torch.randint(0, P, (len(sections), B, S), generator=torch.Generator().manual_seed(2)).to(dtype)
    pos[:, 0, 0], pos[:, 1, 1] = 0, P - 1
    oq, ok = rope.rotary_axes(q, k, cos.cuda(), sin.cuda(), pos.cuda(), sections, order=order, layout=layout)
    c, s = angles(cos, sin, pos, axes)
    check(oq.detach(), q.detach().cpu(), c, s, half)
    check(ok.detach(), k.detach().cpu(), c, s, half)
    gq, gk = seeded_bf16((B, H, S, D), seed=3).transpose(1, 2), seeded_bf16((B, S, K, D), seed=4)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq.cuda(), gk.cuda()))
    check(dq, gq, c, -s, half)
    check(dk, gk, c, -s, half)


def test_equal_positions_are_one_axis():
    """Tokens of text, whose positions are equal on every axis, turn as `rotary` turns them, bit for bit."""
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(128, 1000))
    q, k = seeded_bf16((3, 7, 4, 128), seed=1).cuda(), seeded_bf16((3, 7, 2, 128), seed=2).cuda()
    pos = torch.randint(0, 1000, (3, 7), device="cuda")
    for layout in rope.LAYOUTS:
        want = rope.rotary(q, k, cos, sin, positions=pos, layout=layout)
        for order in rope.ORDERS:
            got = rope.rotary_axes(q, k, cos, sin, pos, (24, 20, 20), order=order, layout=layout)   # (broadcast over the axes)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_positions_of_any_strides(host):
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(64, 100))
    q, k = seeded_bf16((2, 6, 2, 64), seed=1).cuda(), seeded_bf16((2, 6, 1, 64), seed=2).cuda()
    pos = torch.randint(0, 100, (3, 2, 6), device="cuda")
    want = rope.rotary_axes(q, k, cos, sin, pos, (10, 11, 11))
    last = pos.permute(1, 2, 0).contiguous().permute(2, 0, 1)     # as (batch, token, axis)
    wide = torch.full((3, 4, 12), -1, device="cuda")
    wide[:, ::2, ::2] = pos
    for p in (last, wide[:, ::2, ::2], pos.int()):
        got = rope.rotary_axes(q, k, cos, sin, p, (10, 11, 11))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = rope.rotary_axes(q, k, cos, sin, pos[:, :1], (10, 11, 11))
    assert torch.equal(one[0], rope.rotary_axes(q, k, cos, sin, pos[:, :1].repeat(1, 2, 1), (10, 11, 11))[0])
    # tables in another layout
    turned = rope.rotary_axes(q, k, cos.t().contiguous().t(), sin, pos, (10, 11, 11))
    assert torch.equal(turned[0], want[0])


def test_positions_outside_the_tables():
    """NaN for a token with any position outside, on any axis, and nothing else."""
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(32, 10))
    q, k = seeded_bf16((1, 6, 2, 48), seed=1).cuda(), seeded_bf16((1, 6, 1, 48), seed=2).cuda()
    pos = torch.zeros((3, 1, 6), dtype=torch.int64, device="cuda")
    want = rope.rotary_axes(q, k, cos, sin, pos, (4, 6, 6))
    pos[0, 0, 1], pos[1, 0, 2], pos[2, 0, 4], pos[2, 0, 5] = 10, -1, 2 ** 40, -2 ** 40
    for p in (pos, pos[:, :, :4].int()):
        n = p.shape[2]
        got = rope.rotary_axes(q[:, :n], k[:, :n], cos, sin, p, (4, 6, 6))
        for g, w in zip(got, want):
            bad = [i for i in (1, 2, 4, 5) if i < n]
            good = [i for i in (0, 3) if i < n]
            assert bool(g[:, bad].isnan().all()) and torch.equal(g[:, good], w[:, good])


def test_tables_of_axes():
    from lingua_amd import rope
    for order in rope.ORDERS:
        cos, sin = rope.axes_tables((6, 0, 4), 50, theta=100.0, order=order)
        assert cos.shape == (50, 10)
        seen = [0, 0, 0]
        for i, a in enumerate(axes_by_hand((6, 0, 4), order)):
            angle = torch.arange(50, dtype=torch.float64) * 100.0 ** (-seen[a] / (6, 0, 4)[a])
            seen[a] += 1
            assert torch.equal(cos[:, i], angle.cos().float()) and torch.equal(sin[:, i], angle.sin().float())


def test_captured_call_replays_with_new_positions():
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(128, 1000))
    q, k = seeded_bf16((4, 1, 8, 128), seed=1).cuda(), seeded_bf16((4, 1, 2, 128), seed=2).cuda()
    pos = torch.arange(12, device="cuda").view(3, 4, 1)
    call = lambda: rope.rotary_axes(q, k, cos, sin, pos, (16, 24, 24), layout="half")  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        pos.add_(71)
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
