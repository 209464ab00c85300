"""The norm of a residual sum, forward and backward.

The sum is PyTorch's bit for bit, and everything behind it is what ``rmsnorm_cast_rowwise`` leaves for that sum, bit for bit, which has
tests of its own; beside that the whole is held against 64 bits.  Rounding of r: a lane adds at most 32 squares in a row, 64 lanes and
16 waves are added in trees and rows, a division and a root follow: fewer than 128 roundings of 2^-24."""
import pytest
import torch

import plain_operators as plain
from conftest import seeded_bf16
from plain_operators import host  # noqa: F401

pytestmark = pytest.mark.gpu

EPS = 1e-5
SHAPES = [(1, 8), (1, 2048), (5, 264), (33, 2048), (600, 1000), (1027, 2048), (17, 4096), (520, 4104), (9, 8192)]


def inputs(shape, w_dtype):
    R, C = shape
    x, res = seeded_bf16(shape, std=2.0, seed=R + C), seeded_bf16(shape, std=3.0, seed=R * 3 + C)
    w = (1.0 + 0.1 * torch.randn(C, generator=torch.Generator().manual_seed(C))).to(w_dtype)
    return x, res, w


def bits(t):
    return t.cpu().contiguous().view({2: torch.int16, 4: torch.int32, 1: torch.uint8}[t.element_size()])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_col", [False, True])
def test_forward(shape, w_dtype, with_col):
    from lingua_amd import ops
    x, res, w = (t.cuda() for t in inputs(shape, w_dtype))
    if shape[0] > 4:
        res[2] = -x[2]                    # a row of zeros
    cols = [torch.zeros(shape[1], device="cuda") if with_col else None for _ in range(2)]
    h, y, q, s, rstd = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS, col_amax=cols[0])
    assert torch.equal(bits(h), bits(x + res))
    y0, q0, s0, rstd0 = ops.rmsnorm_cast_rowwise(h, w, EPS, col_amax=cols[1])
    for a, b in ((y, y0), (q, q0), (s, s0), (rstd, rstd0)) + (((cols[0], cols[1]),) if with_col else ()):
        assert torch.equal(bits(a), bits(b))
    _, _, y64 = plain.add_rmsnorm(x.cpu(), res.cpu(), w.cpu(), EPS)
    assert plain.within(y, y64, y64.abs() * 128 * plain.FP32)
    h2, y2, q2, s2, r2 = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS, want_q=False, want_rstd=False)
    assert q2 is None and s2 is None and r2 is None and torch.equal(bits(h2), bits(h)) and torch.equal(bits(y2), bits(y))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32])
def test_backward(shape, w_dtype, host):
    """gx: the terms' magnitudes times the roundings of r (128), of the row's mean (128) and a few products.  gw: 512 workgroups add up
    their rows one by one, then eight sums of 64 and those eight."""
    from lingua_amd import norm
    x, res, w = inputs(shape, w_dtype)
    gy, gh = seeded_bf16(shape, std=0.05, seed=1), seeded_bf16(shape, std=0.05, seed=2)
    leaves = [t.cuda().requires_grad_() for t in (x, res, w)]
    h, y = norm.add_rmsnorm(*leaves, EPS)
    gx, gres, gw = torch.autograd.grad((h, y), leaves, (gh.cuda(), gy.cuda()))
    assert torch.equal(bits(gx), bits(gres)) and gw.dtype == w_dtype
    h64, r64, _ = plain.add_rmsnorm(x, res, w, EPS)
    g64, gw64, size, gw_size = plain.add_rmsnorm_gradients(h64, r64, w.double(), gy.double(), gh.double())
    assert plain.within(gx, g64, size * 512 * plain.FP32)
    gw_bound = gw_size * (shape[0] / 512 + 64 + 8 + 128 + 4) * plain.FP32
    if w_dtype == torch.bfloat16:
        assert plain.within(gw, gw64, gw_bound)
    else:
        assert bool(((gw.cpu().double() - gw64).abs() <= gw_bound).all())


def test_gradients_of_the_formula_against_differences():
    """What the kernels are held against, by autograd's own differences in 64 bits."""
    g = torch.Generator().manual_seed(0)
    h, w = torch.randn(3, 8, generator=g, dtype=torch.float64), torch.randn(8, generator=g, dtype=torch.float64)
    gy, gh = torch.randn(3, 8, generator=g, dtype=torch.float64), torch.randn(3, 8, generator=g, dtype=torch.float64)

    def loss(h, w):
        return (gh * h).sum() + (gy * h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w).sum()

    r = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    g64, gw64, _, _ = plain.add_rmsnorm_gradients(h, r, w, gy, gh)
    step = 1e-6
    for t, want in ((h, g64), (w, gw64)):
        for i in range(t.numel()):
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += step
            down.view(-1)[i] -= step
            other = (lambda v: loss(v, w)) if t is h else (lambda v: loss(h, v))
            assert abs(float((other(up) - other(down)) / (2 * step)) - float(want.view(-1)[i])) < 1e-6


@pytest.mark.parametrize("used", ["both", "sum", "norm"])
def test_either_output_alone(used, host):
    from lingua_amd import norm, ops
    x, res, w = (t.cuda() for t in inputs((70, 520), torch.float32))
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]
    h, y = norm.add_rmsnorm(*leaves, EPS)
    gy, gh = seeded_bf16((70, 520), std=0.05, seed=1).cuda(), seeded_bf16((70, 520), std=0.05, seed=2).cuda()
    outs, gs = {"both": ((h, y), (gh, gy)), "sum": ((h,), (gh,)), "norm": ((y,), (gy,))}[used]
    gx, gres, gw = torch.autograd.grad(outs, leaves, gs, allow_unused=True)
    if used == "sum":
        assert torch.equal(gx, gh) and torch.equal(gres, gh) and gw is None
        return
    _, _, _, _, rstd = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
    want = ops.rmsnorm_bwd(gy, h.detach(), w, rstd) if used == "norm" else ops.add_rmsnorm_bwd(gy, gh, h.detach(), w, rstd)
    assert torch.equal(bits(gx), bits(want[0])) and torch.equal(bits(gw), bits(want[1]))


def test_rows_apart_one_tensor_twice_leading_dimensions_and_no_rows():
    from lingua_amd import norm, ops
    x, res, w = (t.cuda() for t in inputs((40, 512), torch.bfloat16))
    wide = torch.zeros(40, 1024, dtype=torch.bfloat16, device="cuda")
    wide[:, 256:768] = x
    want = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
    for a, b in zip(ops.add_rmsnorm_cast_rowwise(wide[:, 256:768], res, w, EPS), want):
        assert torch.equal(bits(a), bits(b))
    h, y = norm.add_rmsnorm(x.view(2, 20, 512), x.view(2, 20, 512), w, EPS)
    assert h.shape == y.shape == (2, 20, 512) and torch.equal(bits(h.view(40, 512)), bits(x + x))
    xe = x[:0].requires_grad_()
    we = w.clone().requires_grad_()
    h, y = norm.add_rmsnorm(xe, res[:0], we, EPS)
    gx, gw = torch.autograd.grad(h.sum() + y.sum(), (xe, we))
    assert gx.shape == (0, 512) and bool((gw == 0).all())


def test_values_that_are_not_finite_stay_in_their_rows():
    from lingua_amd import ops
    x, res, w = (t.cuda() for t in inputs((6, 512), torch.bfloat16))
    x[1, 7], x[3, 9], res[3, 9] = float("nan"), float("inf"), -float("inf")
    x[4, 2] = float("inf")
    h, y, q, s, _ = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
    assert torch.equal(torch.isnan(h), torch.isnan(x + res))
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3]).all()) and bool(torch.isfinite(y[[0, 2, 5]]).all())
    q0, s0, _ = ops.cast_rowwise(y)
    assert torch.equal(bits(q0), bits(q)) and torch.equal(torch.isnan(s0), torch.isnan(s))


def test_linears_behind_it_find_their_input_quantised():
    from lingua_amd import float8 as f8, norm
    x, res, w = (t.cuda() for t in inputs((32, 256), torch.bfloat16))
    _, y = norm.add_rmsnorm(x, res, w, EPS)
    q, s, _ = f8._fwd_cast.get(y, "a linear")
    from lingua_amd import ops
    q0, s0, _ = ops.cast_rowwise(y)
    assert torch.equal(bits(q), bits(q0)) and torch.equal(bits(s), bits(s0))
    f8.clear_cast_memos()


def test_fused_blocks_of_a_model():
    """Forward, blocks with the residual norm fused give the bits of those without (the second norm reads the same sum); forward and
    backward, the bits of blocks that call ``add_rmsnorm`` themselves."""
    from bench_workloads import Llama, TransformerBlock
    from lingua_amd import convert_linears_to_fp8, norm

    class Block(TransformerBlock):
        def forward(self, x, cos, sin):
            h, y = norm.add_rmsnorm(x, self.attention(self.attention_norm(x), cos, sin), self.ffn_norm.weight, self.ffn_norm.eps)
            return h + self.feed_forward(y)

    outs = {}
    for kind in ("apart", "by hand", "fused"):
        model = Llama(n_layers=2, dim=256, n_heads=4, ffn_dim=512, vocab=64).to("cuda", torch.bfloat16)
        model.init_weights(seed=1)
        convert_linears_to_fp8(model, "rowwise", r"layers\.[0-9]+\.")
        keys = list(model.state_dict())
        norm.fuse_rmsnorm(model)
        if kind == "by hand":
            for layer in model.layers:
                layer.__class__ = Block
        if kind == "fused":
            norm.fuse_residual_norm(model)
            norm.fuse_residual_norm(model)    # once more changes nothing
        assert list(model.state_dict()) == keys
        tokens = torch.randint(0, 64, (2, 24), generator=torch.Generator().manual_seed(2)).cuda()
        logits = model(tokens)
        grads = torch.autograd.grad(logits.float().square().mean(), list(model.parameters()))
        outs[kind] = (logits.detach(), grads)
    assert torch.equal(outs["apart"][0], outs["fused"][0]) and torch.equal(outs["by hand"][0], outs["fused"][0])
    for name, a, b in zip(keys, outs["by hand"][1], outs["fused"][1]):
        assert name == "tok_embeddings.weight" or torch.equal(a, b), name    # (the embedding's gradient is added up by atomics)


def test_captured_norm_replays():
    from lingua_amd import ops
    x, res, w = (t.cuda() for t in inputs((3, 2048), torch.bfloat16))
    ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
    for i in range(3):
        x.copy_(seeded_bf16((3, 2048), seed=50 + i))
        want = ops.add_rmsnorm_cast_rowwise(x, res, w, EPS)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out, want))


def test_rows_off_their_lines(host):
    """Operands and gradients that start at odd elements, an odd number of elements apart: copied, with the results of dense ones."""
    from lingua_amd import norm
    R, C = 5, 72
    odd = [seeded_bf16((R, C + 3), seed=i).cuda()[:, 1:1 + C] for i in range(4)]
    w = seeded_bf16((C,), seed=9).cuda()

    def run(x, res, gh, gy):
        x, res = x.detach().requires_grad_(), res.detach().requires_grad_()
        h, y = norm.add_rmsnorm(x, res, w, EPS)
        return (h, y) + torch.autograd.grad((h, y), (x, res), (gh, gy))

    for got, want in zip(run(*odd), run(*(t.contiguous() for t in odd))):
        assert torch.equal(got, want)


def test_refusals():
    from lingua_amd import norm, ops
    x, res, w = (t.cuda() for t in inputs((4, 64), torch.bfloat16))
    big = torch.zeros(2, 8200, dtype=torch.bfloat16, device="cuda")
    rstd = torch.ones(4, 1, device="cuda")
    for call in (lambda: ops.add_rmsnorm_cast_rowwise(x, res[:3], w, EPS), lambda: ops.add_rmsnorm_cast_rowwise(x, res.float(), w, EPS),
                 lambda: ops.add_rmsnorm_cast_rowwise(x, res, w[:32], EPS), lambda: ops.add_rmsnorm_cast_rowwise(x.cpu(), res.cpu(), w.cpu(), EPS),
                 lambda: ops.add_rmsnorm_cast_rowwise(x[:, :20], res[:, :20], w[:20], EPS), lambda: ops.add_rmsnorm_cast_rowwise(big, big, big[0], EPS),
                 lambda: norm.add_rmsnorm(x, res[:, :32], w, EPS), lambda: norm.add_rmsnorm(x[0], res[0], w, EPS), lambda: norm.add_rmsnorm(x.half(), res, w, EPS),
                 lambda: ops.add_rmsnorm_bwd(x, x[:2], x, w, rstd), lambda: ops.add_rmsnorm_bwd(x, x, x, w, rstd[:2]),
                 lambda: ops.add_rmsnorm_bwd(x, x, x, w, rstd, gw_dtype=torch.float16),
                 lambda: norm.fuse_residual_norm(torch.nn.ModuleDict({"layers": torch.nn.ModuleList([torch.nn.Linear(2, 2)])}))):
        with pytest.raises(RuntimeError):
            call()
