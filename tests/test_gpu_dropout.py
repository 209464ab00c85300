"""Dropout whose mask is never stored: its bits against the generator in whole numbers, alone, into a sum and inside the residual norms."""
import pytest
import torch

import plain_more as plain
import plain_operators
from conftest import seeded_bf16
from plain_operators import host, within  # noqa: F401

pytestmark = pytest.mark.gpu

EPS = 1e-5


def numbers(seed=0x0123456789abcdef, step=5):
    from lingua_amd import dropout
    n = dropout.numbers(seed)
    n[1] = step
    return n


def test_generator_is_the_published_one():
    """The known answers that the generator's authors publish with it (counter and key zero, and all ones)."""
    assert plain.philox((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = 0xffffffff
    assert plain.philox((ones,) * 4, (ones, ones)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (333, 2064), (3, 5, 11), (4096,)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("added", [False, True])
def test_bits(shape, p, added, host):
    from lingua_amd import dropout
    n = numbers(seed=-3, step=2 ** 40 + 7)
    drop = dropout.Drop(p, n, site=9 if p == 0.1 else 2 ** 32 - 1)
    x, res, g = (seeded_bf16(shape, seed=i).cuda() for i in range(3))
    x.requires_grad_(), res.requires_grad_()
    keep = plain.keeps(n, drop.site, p, x.numel())
    want = plain.dropped(x.detach(), keep, p)
    if added:
        y = dropout.dropout_add(x, res, drop)
        gx, gres = torch.autograd.grad(y, (x, res), g)
        want = res.detach().float() + want
        assert torch.equal(gres, g)
    else:
        y = dropout.dropout(x, drop)
        gx, = torch.autograd.grad(y, x, g)
    assert torch.equal(y, want.to(torch.bfloat16)) and torch.equal(gx, plain.dropped(g, keep, p).to(torch.bfloat16))


def test_share_and_independence():
    """Of 2^20 elements the share that is dropped is p within five deviations, and another seed, step or site drops others."""
    from lingua_amd import dropout
    x = torch.ones(1 << 20, dtype=torch.bfloat16, device="cuda")
    base = dropout.Drop(0.25, numbers(), 1)
    masks = [dropout.dropout(x, d) == 0 for d in (base, base._replace(site=2), base._replace(numbers=numbers(step=6)), base._replace(numbers=numbers(seed=1)))]
    deviation = (0.25 * 0.75 / x.numel()) ** 0.5
    for m in masks:
        assert abs(float(m.double().mean()) - 0.25) < 5 * deviation
    for i in range(1, 4):   # together: p^2
        assert abs(float((masks[0] & masks[i]).double().mean()) - 0.0625) < 5 * (0.0625 * 0.9375 / x.numel()) ** 0.5
    # neighbours at distances within and across groups and words
    for d in (1, 2, 7, 8, 4096):
        assert abs(float((masks[0][:-d] & masks[0][d:]).double().mean()) - 0.0625) < 5 * (0.0625 * 0.9375 / x.numel()) ** 0.5


def test_what_is_dropped_is_gone(host):
    from lingua_amd import dropout
    n = numbers()
    x = torch.full((4096,), float("nan"), dtype=torch.bfloat16, device="cuda")
    x[::2] = float("inf")
    keep = plain.keeps(n, 0, 0.5, 4096).cuda()
    y = dropout.dropout(x, dropout.Drop(0.5, n))
    assert bool((y[~keep] == 0).all()) and not bool(y[keep].isfinite().any())
    assert not bool(dropout.dropout(x, dropout.Drop(1.0, n)).any())


def test_elements_off_lines(host):
    from lingua_amd import dropout
    x = seeded_bf16((1001,), seed=1).cuda()
    drop = dropout.Drop(0.3, numbers())
    for i in range(1, 9):
        assert torch.equal(dropout.dropout(x[i:], drop), dropout.dropout(x[i:].clone(), drop))
    wide = seeded_bf16((40, 30), seed=2).cuda()
    assert torch.equal(dropout.dropout(wide[:, 1:20], drop), dropout.dropout(wide[:, 1:20].contiguous(), drop))
    assert torch.equal(dropout.dropout(wide.t(), drop), dropout.dropout(wide.t().contiguous(), drop))
    assert dropout.dropout(wide[:0], drop).shape == (0, 30)


NORM_SIZES = [(1, 8), (3, 1152), (5, 2056), (2, 4104), (4, 6152), (3, 8192), (1040, 256)]


@pytest.mark.parametrize("R, C", NORM_SIZES)
@pytest.mark.parametrize("centred", [True, False])
def test_inside_the_norms(R, C, centred, host):
    """The sum is dropout_add's bit for bit; y, the copy, its scales and the column amaxes are those of the norm of that sum; gradients are
    within their rounding of 64 bits and dropped where forward dropped."""
    from lingua_amd import dropout, norm, ops
    n = numbers()
    drop = dropout.Drop(0.2, n, site=3)
    x, res, gy, gh = (seeded_bf16((R, C), std=s, seed=i).cuda() for i, s in enumerate((1.0, 2.0, 0.1, 0.1)))
    w = (1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(1))).cuda().requires_grad_()
    b = (0.2 * torch.randn(C, generator=torch.Generator().manual_seed(2))).to(torch.bfloat16).cuda().requires_grad_() if centred else None
    want_h = dropout.dropout_add(x, res, drop)
    col, col1 = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    h, y, q, scale, stats = ops.layernorm_cast_rowwise(x, w.detach(), None if b is None else b.detach(), EPS, res, drop, centred, col_amax=col)
    assert torch.equal(h, want_h)
    if centred:
        alone = ops.layernorm_cast_rowwise(h, w.detach(), b.detach(), EPS, col_amax=col1)[1:4]
    else:
        alone = ops.rmsnorm_cast_rowwise(h, w.detach(), EPS, col_amax=col1)[:3]
    for a, c in zip((y, q, scale, col), (*alone, col1)):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))

    x.requires_grad_(), res.requires_grad_()
    if centred:
        h2, y2 = norm.add_layernorm(x, res, w, b, EPS, drop)
        gx, gres, gw, gb = torch.autograd.grad((h2, y2), (x, res, w, b), (gh, gy))
    else:
        h2, y2 = norm.add_rmsnorm(x, res, w, EPS, drop)
        gx, gres, gw = torch.autograd.grad((h2, y2), (x, res, w), (gh, gy))
    assert torch.equal(h2, h) and torch.equal(y2, y)
    keep = plain.keeps(n, 3, 0.2, R * C)
    w64 = w.detach().double()
    if centred:
        hat, r, _ = plain.layernorm(h, w64, b.detach().double(), EPS)
        (g, want_w, want_b), (err, err_w, err_b) = plain.layernorm_grads(h, hat, r, w64, gy, gh.double())
        assert plain.grad_within(gb, want_b, err_b)
    else:
        r = 1 / (h.double().square().mean(1, keepdim=True) + EPS).sqrt()
        g, want_w, size, size_w = plain_operators.add_rmsnorm_gradients(h.double(), r, w64, gy.double(), gh.double())
        # sums of up to 8192 columns and R rows, each addition and product off by half a step
        err, err_w = size * 100 * plain.FP32, size_w * (R + 110) * plain.FP32
    assert within(gres, g, err) and plain.grad_within(gw, want_w, err_w)
    factor = 65536 / (65536 - round(65536 * 0.2))
    keep = keep.view(R, C).cuda()
    assert within(gx, torch.where(keep, g * factor, torch.zeros_like(g)), torch.where(keep, err * factor + g.abs() * factor * plain.FP32, torch.zeros_like(g)))
    assert bool((gx[~keep] == 0).all())
    # the sum's gradient alone
    h3 = (norm.add_layernorm(x, res, w, b, EPS, drop) if centred else norm.add_rmsnorm(x, res, w, EPS, drop))[0]
    gx, gres = torch.autograd.grad(h3, (x, res), gh)
    assert torch.equal(gres, gh) and torch.equal(gx, dropout.dropout(gh, drop))


def test_far_elements():
    """Elements beyond 2^31."""
    from lingua_amd import dropout
    n = numbers()
    count = (1 << 31) + 64
    x = torch.ones(count, dtype=torch.bfloat16, device="cuda")
    y = dropout.dropout(x, dropout.Drop(0.5, n))
    first = count - 128
    keep = plain.keeps(n, 0, 0.5, 128, first=first)
    assert torch.equal((y[first:] != 0).cpu(), keep)


def test_numbers_changed_between_the_passes_are_an_error(host):
    from lingua_amd import dropout, norm
    n = numbers()
    x, res = (seeded_bf16((16, 64), seed=i).cuda().requires_grad_() for i in range(2))
    for make in (lambda d: dropout.dropout(x, d), lambda d: dropout.dropout_add(x, res, d), lambda d: norm.add_layernorm(x, res, dropout=d)[1]):
        y = make(dropout.Drop(0.5, n))
        n[1] += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_modules():
    from lingua_amd import dropout
    n = numbers()
    shared = torch.nn.Dropout(0.3)
    model = torch.nn.ModuleDict({"a": torch.nn.Dropout(0.1), "b": torch.nn.Sequential(shared, torch.nn.Identity(), shared), "c": torch.nn.Dropout(0.2)})
    dropout.convert_dropouts(model, n, "a|b")
    assert type(model["c"]) is torch.nn.Dropout
    assert (model["a"].p, model["a"].site, model["b"][0].site, model["b"][2].site) == (0.1, 0, 1, 2)
    dropout.convert_dropouts(model, n)
    assert model["c"].site == 3
    x = seeded_bf16((64, 64), seed=1).cuda()
    assert torch.equal(model["a"](x), dropout.dropout(x, dropout.Drop(0.1, n, 0)))
    model.eval()
    assert model["a"](x) is x and model["a"].drop() is None


def test_replayed_steps_drop_other_elements():
    """A captured step that counts itself: every replay equals the eager step of its number."""
    from lingua_amd import dropout, norm
    n = numbers(step=0)
    side = torch.cuda.Stream()
    x, res = (seeded_bf16((64, 256), seed=i).cuda().requires_grad_() for i in range(2))
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    g = seeded_bf16((64, 256), std=0.1, seed=3).cuda()

    def step(n):
        h, y = norm.add_layernorm(dropout.dropout(x, dropout.Drop(0.1, n, 1)), res, w, dropout=dropout.Drop(0.1, n, 2))
        grads = torch.autograd.grad((h, y), (x, res, w), (g, g))
        return (h.detach(), y.detach(), *grads)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(n)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(n)
        n[1] += 1
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        seen.append([t.clone() for t in out])
        assert int(n[1]) == i + 1
    for i, got in enumerate(seen):
        x2, res2, w2 = (t.detach().clone().requires_grad_() for t in (x, res, w))
        m = numbers(step=i)
        h, y = norm.add_layernorm(dropout.dropout(x2, dropout.Drop(0.1, m, 1)), res2, w2, dropout=dropout.Drop(0.1, m, 2))
        want = (h, y, *torch.autograd.grad((h, y), (x2, res2, w2), (g, g)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.equal(seen[0][0], seen[1][0])


@pytest.mark.parametrize("count", [4096, 1001])
@pytest.mark.parametrize("off", [0, 1])
def test_in_place(count, off):
    """The library's entry with the output over either operand."""
    from lingua_amd import _lib, dropout
    n, lib, stream = numbers(), _lib.load(), torch.cuda.current_stream().cuda_stream
    x, res = (seeded_bf16((count + off,), seed=i).cuda()[off:] for i in range(2))
    drop = dropout.Drop(0.3, n, 7)
    for residual, into in ((None, "x"), (res, "x"), (res, "residual")):
        want = dropout.dropout(x, drop) if residual is None else dropout.dropout_add(x, residual, drop)
        ops = {"x": x, "residual": residual}
        room = torch.full((count + off + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
        y = room[off:off + count].copy_(ops[into])
        ops[into] = y
        assert lib.l8_dropout(ops["x"].data_ptr(), None if residual is None else ops["residual"].data_ptr(), y.data_ptr(), count, n.data_ptr(), 7, round(65536 * 0.3), stream) == 0
        assert torch.equal(y, want) and bool((room[off + count:] == 7).all())
