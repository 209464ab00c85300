"""Rotary positions against the rotation in 64 bits: fp32 products and sums are off by at most three roundings of the terms'
magnitudes, bf16 by half a step.  Both layouts, parts of the head, strides, positions, gradients."""
import pytest
import torch

import plain_operators as plain
from conftest import seeded_bf16
from plain_operators import host  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, x, cos, sin, in_halves):
    """cos, sin: [B or 1, S, 1, rot / 2]"""
    want = plain.rotate(x, cos, sin, in_halves)
    size = plain.rotate(x.abs().float(), cos.abs(), -sin.abs(), in_halves).abs() + plain.rotate(x.abs().float(), cos.abs(), sin.abs(), in_halves).abs()
    assert got.shape == x.shape and got.dtype == torch.bfloat16 and got.is_contiguous()
    assert plain.within(got, want, size * 3 * plain.FP32)
    rot = 2 * cos.shape[-1]
    assert torch.equal(got[..., rot:].cpu().view(torch.int16), x[..., rot:].cpu().contiguous().view(torch.int16))


# head size, turned columns: whole heads, parts, widths that allow vectors of 8, 4 and 1 pairs
HEADS = [(2, 2), (64, 64), (128, 64), (96, 40), (128, 128), (34, 6), (80, 16), (256, 128), (512, 512), (64, 2), (36, 24)]


@pytest.mark.parametrize("D,rot", HEADS)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,S,H,K", [(1, 1, 1, 1), (2, 5, 3, 1), (1, 33, 8, 2)])
def test_rotation(D, rot, layout, B, S, H, K):
    from lingua_amd import rope
    cos, sin = rope.rotary_tables(rot, 40)
    q, k = seeded_bf16((B, S, H, D), seed=D), seeded_bf16((B, S, K, D), seed=rot)
    gq, gk = rope.rotary(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), layout=layout)
    c, s = cos[None, :S, None], sin[None, :S, None]
    check(gq, q, c, s, layout == "half")
    check(gk, k, c, s, layout == "half")


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_strides_and_gradients(layout, dtype, host):
    """q and k are column slices of one product, gradients come with heads in front of tokens; positions far and in any order."""
    from lingua_amd import rope
    B, S, H, K, D, rot = 3, 17, 6, 2, 64, 48
    half = layout == "half"
    cos, sin = rope.rotary_tables(rot, 100000, scaling="yarn", factor=8, trained_length=4096)
    y = seeded_bf16((B * S, (H + 2 * K) * D), seed=1).cuda()
    q = y[:, :H * D].view(B, S, H, D).detach().requires_grad_()
    k = y[:, H * D:(H + K) * D].view(B, S, K, D).detach().requires_grad_()
    pos = torch.randint(0, 100000, (B, S), generator=torch.Generator().manual_seed(2)).to(dtype)
    pos[0, 0], pos[1, 1] = 0, 99999
    oq, ok = rope.rotary(q, k, cos.cuda(), sin.cuda(), positions=pos.cuda(), layout=layout)
    c, s = cos[pos.long()][:, :, None], sin[pos.long()][:, :, None]
    check(oq.detach(), q.detach().cpu(), c, s, half)
    check(ok.detach(), k.detach().cpu(), c, s, half)
    gq, gk = seeded_bf16((B, H, S, D), seed=3).transpose(1, 2), seeded_bf16((B, S, K, D), seed=4)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq.cuda(), gk.cuda()))
    check(dq, gq, c, -s, half)
    check(dk, gk, c, -s, half)
    # one of the two alone, and none
    oq, ok = rope.rotary(q, k.detach(), cos.cuda(), sin.cuda(), positions=pos.cuda(), layout=layout)
    (dq2,) = torch.autograd.grad(oq, q, gq.cuda())
    assert torch.equal(dq2, dq)
    # positions that broadcast over the batch
    oq, _ = rope.rotary(q, k, cos.cuda(), sin.cuda(), positions=pos[1].cuda(), layout=layout)
    check(oq.detach(), q.detach().cpu(), cos[pos[1].long()][None, :, None], sin[pos[1].long()][None, :, None], half)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,S,H", [(2, 5, 3), (1, 7, 1), (4, 1, 2)])
def test_heads_at_odd_elements(layout, B, S, H, host):
    """Operands and gradients that start at an odd element and whose rows are an odd number of elements apart."""
    from lingua_amd import rope
    D, rot = 32, 16
    cos, sin = rope.rotary_tables(rot, S)
    odd = [seeded_bf16((B * S, H * D + 5), seed=i).cuda()[:, 3:3 + H * D].unflatten(1, (H, D)).unflatten(0, (B, S)) for i in range(3)]
    q, k = odd[0].detach().requires_grad_(), odd[1].detach()
    oq, ok = rope.rotary(q, k, cos.cuda(), sin.cuda(), layout=layout)
    (dq,) = torch.autograd.grad(oq, q, odd[2])
    for got, x, s in ((oq.detach(), odd[0], sin), (ok, odd[1], sin), (dq, odd[2], -sin)):
        check(got, x.cpu(), cos[None, :, None], s[None, :, None], layout == "half")


def test_it_is_the_eager_chain_bit_for_bit():
    """The chain that the benchmark's model runs between its projections and its attention."""
    from bench_workloads import apply_rope, rope_tables
    from lingua_amd import rope
    cos, sin = rope_tables(64, 50, 10000.0, "cuda")
    q, k = seeded_bf16((2, 50, 4, 64), seed=1).cuda(), seeded_bf16((2, 50, 2, 64), seed=2).cuda()
    gq, gk = rope.rotary(q, k, cos, sin)
    assert torch.equal(gq, apply_rope(q, cos, sin)) and torch.equal(gk, apply_rope(k, cos, sin))
    # the same table as rotation matrices, and heads in front of tokens
    freqs = torch.stack((cos, -sin, sin, cos), -1).unflatten(-1, (2, 2))
    eq, ek = rope.apply_rotary_emb(q, k, 1, freqs)
    assert torch.equal(eq, gq) and torch.equal(ek, gk)
    tq, tk = rope.apply_rotary_emb(q.transpose(1, 2), k.transpose(1, 2), 2, freqs)
    assert torch.equal(tq.transpose(1, 2), gq) and torch.equal(tk.transpose(1, 2), gk)


def test_strange_values_and_positions():
    from lingua_amd import ops
    cos, sin = torch.ones(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    x = seeded_bf16((1, 6, 2, 24), seed=1).cuda()
    x[0, 1, 0, 0], x[0, 1, 1, 20] = float("nan"), float("inf")
    pos = torch.tensor([0, 3, -1, 4, 2 ** 40, 2], device="cuda")
    (y, none) = ops.rotary(x, None, cos, sin, positions=pos)
    assert none is None
    known = torch.tensor([True, True, False, False, False, True])
    assert bool(torch.isnan(y[0, ~known, :, :16]).all())
    assert torch.equal(torch.isnan(y[0, known, :, :16]).sum(), torch.tensor(2, device="cuda")) and float(y[0, 1, 1, 20]) == float("inf")
    assert torch.equal(y[0, 5], x[0, 5])


@pytest.mark.parametrize("shape", [(0, 3, 2, 16), (2, 0, 2, 16), (2, 3, 0, 16)])
def test_empty(shape):
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(16, 8))
    q = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    oq, ok = rope.rotary(q, q, cos, sin)
    assert oq.shape == ok.shape == shape


def test_captured_rotary_replays():
    from lingua_amd import rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(64, 4096))
    q, k = seeded_bf16((8, 1, 8, 64), seed=1).cuda(), seeded_bf16((8, 1, 2, 64), seed=2).cuda()
    pos = torch.arange(8, device="cuda")[:, None].contiguous()
    rope.rotary(q, k, cos, sin, positions=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oq, ok = rope.rotary(q, k, cos, sin, positions=pos, layout="half")
    for i in range(3):
        pos.add_(1000)
        q.copy_(seeded_bf16((8, 1, 8, 64), seed=10 + i))
        wq, wk = rope.rotary(q, k, cos, sin, positions=pos, layout="half")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oq, wq) and torch.equal(ok, wk)


def test_refusals():
    from lingua_amd import ops, rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(16, 8))
    q = seeded_bf16((2, 3, 4, 16), seed=1).cuda()
    bad = [lambda: rope.rotary(q, q, cos, sin, layout="other"), lambda: rope.rotary(q.float(), q, cos, sin), lambda: rope.rotary(q, q[:1], cos, sin),
           lambda: rope.rotary(q[..., :8], q[..., :8], cos, sin), lambda: rope.rotary(q, q, cos, sin[:4]), lambda: rope.rotary(q, q, cos.double(), sin.double()),
           lambda: rope.rotary(q, q, cos[:2], sin[:2]), lambda: rope.rotary(q, q, cos, sin, positions=torch.zeros(5, dtype=torch.int64, device="cuda")),
           lambda: rope.rotary(q, q, cos, sin, positions=torch.zeros(3, device="cuda")), lambda: rope.rotary(q, q, cos, sin, positions=torch.zeros(3, dtype=torch.int64)),
           lambda: rope.rotary(q.cpu(), q, cos, sin), lambda: rope.apply_rotary_emb(q, q, 1, cos), lambda: ops.rotary(None, None, cos, sin),
           lambda: rope.rotary(q[0], q[0], cos, sin), lambda: rope.rotary(seeded_bf16((1, 1, 1, 514)).cuda(), seeded_bf16((1, 1, 1, 514)).cuda(), cos, sin)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
