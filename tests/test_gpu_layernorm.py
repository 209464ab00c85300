"""Layer norm, its residual sum and its fp8 copy against 64 bits, both host paths; the modules."""
import pytest
import torch

import oracle
import plain_more as plain
from conftest import seeded_bf16
from plain_operators import host, within  # noqa: F401

pytestmark = pytest.mark.gpu

EPS = 1e-5


def param(C, dtype, seed, mean):
    return (mean + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def operands(R, C, seed=0, offset=0.0):
    x, res = (seeded_bf16((R, C), std=s, seed=seed + i) for i, s in enumerate((1.0, 2.0)))
    if offset:
        x = (x.float() + offset).to(torch.bfloat16)
    return x.cuda(), res.cuda()


def check(h, y, q, scale, stats, w, b, col=None):
    w64, b64 = (torch.full((h.shape[1],), v, dtype=torch.float64, device="cuda") if t is None else t.double() for t, v in ((w, 1.0), (b, 0.0)))
    hat, r, want = plain.layernorm(h, w64, b64, EPS)
    assert within(y, want, plain.y_error(h, hat, r, w64, b64))
    if stats is not None:
        mean = h.double().mean(1)
        assert bool(((stats[0].double() - mean).abs() <= 46 * plain.FP32 * h.double().abs().mean(1) + 1e-37).all())
    if q is not None:
        qo, so, _ = oracle.cast_rowwise(y.cpu())
        assert torch.equal(q.cpu().view(torch.uint8), qo) and torch.equal(scale.cpu().flatten(), so)
    if col is not None:
        assert torch.equal(col, y.float().abs().amax(0))


SIZES = [(1, 8), (1, 2048), (3, 1152), (7, 2056), (2, 4104), (5, 6152), (4, 8192), (521, 512), (1030, 1000), (2100, 2048), (600, 4096), (1100, 72), (513, 8184)]


@pytest.mark.parametrize("R, C", SIZES)
@pytest.mark.parametrize("added", [False, True])
def test_forward(R, C, added, host):
    from lingua_amd import ops
    x, res = operands(R, C, seed=R + C)
    for i, (w, b) in enumerate([(param(C, torch.bfloat16, 1, 1.0), param(C, torch.float32, 2, 0.0)), (param(C, torch.float32, 1, 1.0), None), (None, None)]):
        col = torch.empty(C, device="cuda") if i == 1 else None
        h, y, q, scale, stats = ops.layernorm_cast_rowwise(x, w, b, EPS, residual=res if added else None, want_q=i < 2, col_amax=col, on_lines=i == 0)
        if added:
            assert torch.equal(h, x + res)
        else:
            assert h is None
        assert (q is None) == (i == 2)
        check(x + res if added else x, y, q, scale, stats, w, b, col)


def test_one_result_for_any_number_of_rows():
    """A row's result is that of the row alone, in both layouts."""
    from lingua_amd import ops
    for C in (1152, 2048):
        x, res = operands(2000, C)
        w, b = param(C, torch.bfloat16, 1, 1.0), param(C, torch.bfloat16, 2, 0.0)
        many = ops.layernorm_cast_rowwise(x, w, b, EPS, residual=res)
        few = ops.layernorm_cast_rowwise(x[700:703], w, b, EPS, residual=res[700:703])
        for a, c in zip(many[:4], few[:4]):
            assert torch.equal(a[700:703].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(many[4][:, 700:703], few[4])


@pytest.mark.parametrize("C", [1000, 4096])
def test_mean_far_from_zero(C):
    """No digits are lost where the mean is hundreds of deviations away."""
    from lingua_amd import ops
    x, _ = operands(9, C, offset=300.0)
    _, y, _, _, stats = ops.layernorm_cast_rowwise(x, None, None, EPS, want_q=False)
    check(x, y, None, None, stats, None, None)


def test_rows_of_one_value_and_not_finite():
    """A constant row is its bias, exactly where the mean is; a row that holds an infinity or NaN is NaN and leaves the others alone."""
    from lingua_amd import ops
    R, C = 6, 1160
    x, _ = operands(R, C)
    x[0], x[1] = 0, 3.0
    x[2, 5], x[3, 1159] = float("inf"), float("nan")
    x[4, 7] = torch.finfo(torch.bfloat16).min
    w, b = param(C, torch.float32, 1, 1.0), param(C, torch.float32, 2, 0.0)
    _, y, q, scale, _ = ops.layernorm_cast_rowwise(x, w, b, EPS)
    assert torch.equal(y[0], b.to(torch.bfloat16)) and torch.equal(y[1], b.to(torch.bfloat16))
    assert bool(y[2:4].isnan().all()) and bool(q[2:4].float().isnan().all()) and bool(scale[2:4].isnan().all())
    good = [0, 1, 5]
    _, alone, q1, s1, _ = ops.layernorm_cast_rowwise(x[good], w, b, EPS)
    assert torch.equal(y[good], alone) and torch.equal(q[good].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(scale[good], s1)
    # a value whose square passes fp32's range: 1 / deviation is zero
    assert torch.equal(y[4], b.to(torch.bfloat16))


@pytest.mark.parametrize("R, C", [(1, 64), (3, 1152), (521, 2048), (40, 2056), (13, 4104), (9, 6152), (700, 8192), (1100, 520), (2, 8)])
@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(R, C, added, dtype, host):
    from lingua_amd import norm
    x, res = operands(R, C, seed=R)
    w, b = param(C, dtype, 1, 1.0), param(C, torch.float32, 2, 0.0)
    leaves = [t.requires_grad_() for t in (x, res, w, b)]
    gy, gh = seeded_bf16((R, C), std=0.1, seed=5).cuda(), seeded_bf16((R, C), std=0.1, seed=6).cuda()
    if added:
        h, y = norm.add_layernorm(x, res, w, b, EPS)
        gx, gres, gw, gb = torch.autograd.grad((h, y), leaves, (gh, gy))
        assert torch.equal(gx, gres) and gx.data_ptr() != 0
    else:
        h, y = x, norm.layernorm(x, w, b, EPS)
        gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
        gh = None
    h = h.detach()
    hat, r, _ = plain.layernorm(h, w.detach().double(), b.detach().double(), EPS)
    want, err = plain.layernorm_grads(h, hat, r, w.detach().double(), gy, None if gh is None else gh.double())
    assert within(gx, want[0], err[0])
    assert gw.dtype == dtype and gb.dtype == torch.float32
    assert plain.grad_within(gw, want[1], err[1]) and plain.grad_within(gb, want[2], err[2])


@pytest.mark.parametrize("R", [513, 1027, 3001])
@pytest.mark.parametrize("C", [8, 504, 512, 520, 1024, 1032, 1152, 1536, 1544, 2048])
def test_gradients_of_many_short_rows(R, C):
    """Rows of one to four chunks of 512 columns, more of them than workgroups: the gradients against 64 bits, and those of x what they are
    for a few of the rows alone, with and without a gradient of the sum and a dropped operand."""
    from lingua_amd import dropout, ops
    x, res = operands(R, C, seed=C)
    gy, gh = seeded_bf16((R, C), std=0.1, seed=5).cuda(), seeded_bf16((R, C), std=0.1, seed=6).cuda()
    w, b = param(C, torch.float32, 1, 1.0), param(C, torch.bfloat16, 2, 0.0)
    drop = dropout.Drop(0.3, dropout.numbers(8), 2)
    for centred, d, gsum in ((True, None, None), (True, None, gh), (True, drop, gh), (False, drop, gh), (False, drop, None)):
        h, _, _, _, stats = ops.layernorm_cast_rowwise(x, w, b if centred else None, EPS, res, d, centred, want_q=False)
        gx, gres, gw, gb = ops.layernorm_bwd(gy, gsum, h, w, stats, d, centred, torch.float32, torch.float32 if centred else None)
        whole = gx if gres is None else gres
        if centred:
            hat, r, _ = plain.layernorm(h, w.double(), b.double(), EPS)
            want, err = plain.layernorm_grads(h, hat, r, w.double(), gy, None if gsum is None else gsum.double())
            assert within(whole, want[0], err[0])
            assert plain.grad_within(gw, want[1], err[1]) and plain.grad_within(gb, want[2], err[2])
        few = ops.layernorm_bwd(gy[:5], None if gsum is None else gsum[:5], h[:5], w, stats[:, :5], d, centred)
        assert torch.equal(gx[:5], few[0]) and (gres is None or torch.equal(gres[:5], few[1]))


def test_gradients_against_differences():
    """The gradient of a weighted sum of outputs against central differences of the 64-bit form along random directions."""
    from lingua_amd import norm
    R, C = 4, 96
    x, _ = operands(R, C)
    w, b = param(C, torch.float32, 1, 1.0), param(C, torch.float32, 2, 0.0)
    gy = seeded_bf16((R, C), seed=3).cuda()
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(norm.layernorm(x, w, b, EPS), leaves, gy)

    def f(x, w, b):
        return float((plain.layernorm(x, w, b, EPS)[2] * gy.double()).sum())

    at = [t.detach().double() for t in leaves]
    for i in range(3):
        d = torch.randn(at[i].shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        step = 1e-4
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step * d, at[i] - step * d
        slope = (f(*up) - f(*down)) / (2 * step)
        got = float((grads[i].double() * d).sum())
        # each entry of gx is off by its rounding; differences of a smooth function by the square of the step
        off = float((grads[i].double().abs() * d.abs()).sum()) * (2.0 ** -8 if i == 0 else 1e-5) + 1e-4 * float((grads[i].double() * d).abs().sum())
        assert abs(got - slope) <= off


@pytest.mark.parametrize("which", ["x", "w", "b", "none", "h only", "y only"])
def test_parts_of_the_gradient(which, host):
    from lingua_amd import norm
    R, C = 37, 264
    x, res = operands(R, C)
    w, b = param(C, torch.bfloat16, 1, 1.0), param(C, torch.bfloat16, 2, 0.0)
    gy, gh = seeded_bf16((R, C), std=0.1, seed=5).cuda(), seeded_bf16((R, C), std=0.1, seed=6).cuda()
    full = [t.detach().clone().requires_grad_() for t in (x, res, w, b)]
    h, y = norm.add_layernorm(*full, EPS)
    if which == "h only":
        gx, gres = torch.autograd.grad(h, full[:2], gh)
        assert torch.equal(gx, gh) and torch.equal(gres, gh)
        return
    if which == "y only":
        a = torch.autograd.grad(y, full, gy, retain_graph=True)
        c = torch.autograd.grad((h, y), full, (torch.zeros_like(gh), gy))
        assert all(torch.equal(u, v) for u, v in zip(a, c))
        return
    want = dict(zip("xrwb", torch.autograd.grad((h, y), full, (gh, gy))))
    some = [t.detach().clone().requires_grad_(n == which) for t, n in zip((x, res, w, b), "xrwb")]
    h, y = norm.add_layernorm(*some, EPS)
    assert y.requires_grad == (which != "none")
    if which != "none":
        # (a sum that does not learn passes no gradient)
        outs = [(h, gh), (y, gy)] if h.requires_grad else [(y, gy)]
        got, = torch.autograd.grad([o for o, _ in outs], [t for t in some if t.requires_grad], [g for _, g in outs])
        assert torch.equal(got, want[which])


def test_strides_and_empty_rows(host):
    from lingua_amd import norm, ops
    wide = seeded_bf16((50, 600), seed=1).cuda()
    x, odd = wide[:, 8:272], wide[:, 3:267]
    w = param(264, torch.bfloat16, 1, 1.0)
    for t in (x, odd, wide.t()[:264].t(), wide[::3, :264]):
        assert torch.equal(norm.layernorm(t, w), norm.layernorm(t.contiguous(), w))
    g = torch.autograd.grad(norm.layernorm(x.requires_grad_(), w), x, wide[:, 8:272].t().contiguous().t())[0]
    assert torch.equal(g, torch.autograd.grad(norm.layernorm(x, w), x, wide[:, 8:272].contiguous())[0])
    assert torch.equal(norm.layernorm(x.view(5, 10, 264) if x.is_contiguous() else x.reshape(5, 10, 264), w).view(50, 264), norm.layernorm(x, w))
    # (1 to 7 elements off a 16-byte line: the weight is read where it lies)
    odd_w = torch.zeros(265, dtype=torch.bfloat16, device="cuda")[1:].copy_(w)
    assert torch.equal(norm.layernorm(x, odd_w), norm.layernorm(x, w))
    none = torch.empty((0, 264), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = norm.layernorm(none, w.requires_grad_())
    gx, gw = torch.autograd.grad(y, (none, w), y.detach())
    assert y.shape == gx.shape == (0, 264) and not gw.any()
    col = torch.ones(264, device="cuda")
    ops.layernorm_cast_rowwise(none.detach(), None, None, EPS, col_amax=col)
    assert not col.any()


def test_module_in_front_of_fp8_linears():
    """The linears behind an Fp8LayerNorm take its copy: the bits of linears behind nn.LayerNorm's place taken by the unfused norm."""
    from lingua_amd import convert_linears_to_fp8, norm, ops
    model = torch.nn.ModuleDict({"attention_norm": torch.nn.LayerNorm(256), "a": torch.nn.Linear(256, 128, bias=False), "b": torch.nn.Linear(256, 64)}).to("cuda", torch.bfloat16)
    with torch.no_grad():
        model["attention_norm"].weight.copy_(param(256, torch.bfloat16, 1, 1.0))
        model["attention_norm"].bias.copy_(param(256, torch.bfloat16, 2, 0.0))
    keys = list(model.state_dict())
    convert_linears_to_fp8(model, "rowwise", "^[ab]$")
    norm.fuse_layernorm(model)
    assert type(model["attention_norm"]) is norm.Fp8LayerNorm and list(model.state_dict()) == keys
    x = seeded_bf16((48, 256), seed=3).cuda().requires_grad_()
    g = seeded_bf16((48, 192), std=0.1, seed=4).cuda()
    names, timer = [], []
    ops.kernel_timer = timer
    try:
        y = model["attention_norm"](x)
        out = torch.cat((model["a"](y), model["b"](y)), 1)
        names = [n for n, *_ in timer]
    finally:
        ops.kernel_timer = None
    assert "layernorm_cast_rowwise" in names and names.count("cast_rowwise") + names.count("cast_rowwise_many") <= 2   # the weights alone
    grads = torch.autograd.grad(out, [x, *model.parameters()], g)
    ln = model["attention_norm"]
    y2 = norm.layernorm(x, ln.weight, ln.bias, ln.eps)     # files nothing
    out2 = torch.cat((model["a"](y2), model["b"](y2)), 1)
    assert torch.equal(out, out2)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(out2, [x, *model.parameters()], g)))
    with pytest.raises(RuntimeError, match="not a LayerNorm"):
        norm.fuse_layernorm(torch.nn.ModuleDict({"ffn_norm": torch.nn.Linear(8, 8)}))
