"""Low-rank adapters of many requests against 64 bits: every rank the kernels know, ragged sizes, tokens in any order, none, strangers."""
import pytest
import torch

import plain_more as plain
from conftest import seeded_bf16
from plain_operators import host, within  # noqa: F401

pytestmark = pytest.mark.gpu


def bank(n, r, K, N, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (seeded_bf16((n, r, K), std=K ** -0.5, seed=seed).cuda(), seeded_bf16((n, r, N), std=0.3, seed=seed + 1).cuda(), (0.5 + torch.rand(n, generator=g)).cuda())


def tokens_of(T, n, how, seed=0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    if how == "one":
        index = torch.full((T,), n - 1)
    elif how == "none":
        index = torch.full((T,), -1)
    elif how == "mixed":       # any order, a tenth without one
        index = torch.randint(-1, n, (T,), generator=g)
        index[torch.rand(T, generator=g) < 0.1] = -1
    else:                      # requests one behind the other
        cuts = torch.randperm(T, generator=g)[:5].sort().values
        index = torch.randint(0, n, (6,), generator=g)[torch.searchsorted(cuts, torch.arange(T), right=True)]
    return index.to(dtype).cuda()


def run(T, n, r, K, N, how, seed=0, dtype=torch.int32, scaled=True):
    from lingua_amd import adapters
    a, b, scale = bank(n, r, K, N, seed)
    x, y, gy = seeded_bf16((T, K), seed=seed + 2).cuda(), seeded_bf16((T, N), seed=seed + 3).cuda(), seeded_bf16((T, N), std=0.1, seed=seed + 4).cuda()
    index = tokens_of(T, n, how, seed, dtype)
    scale = scale if scaled else None
    leaves = [t.requires_grad_() for t in (y, x, a, b)]
    out = adapters.add_lowrank(*leaves, index, scale)
    dy, gx, ga, gb = torch.autograd.grad(out, leaves, gy)
    want, size, _, _ = plain.lowrank(y, x, a, b, index, scale)
    assert within(out.detach(), want, size)
    none = index < 0
    assert torch.equal(out.detach()[none], y.detach()[none]) and not gx[none].any()
    assert torch.equal(dy, gy)
    wants, sizes = plain.lowrank_grads(x, a, b, index, scale, gy)
    for got, w, s in zip((gx, ga, gb), wants, sizes):
        assert within(got, w, s)


@pytest.mark.parametrize("T", [1, 2, 16, 17, 63, 100, 257, 700])
@pytest.mark.parametrize("n, how", [(1, "one"), (3, "mixed"), (5, "runs"), (70, "mixed"), (2, "none")])
def test_tokens(T, n, how, host):
    if how == "runs" and T < 6:
        how = "mixed"
    run(T, n, 16, 200, 328, how, seed=T + n)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 48, 56, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("T, n", [(37, 4), (330, 2)])
def test_ranks(r, T, n, host):
    run(T, n, r, 264, 520, "mixed", seed=r)


@pytest.mark.parametrize("K, N", [(8, 8), (8, 4104), (2064, 8), (56, 72), (64, 128), (136, 512), (1024, 1032), (4096, 40)])
@pytest.mark.parametrize("T", [5, 200])
def test_features(K, N, T, host):
    run(T, 2, 16, K, N, "mixed", seed=K + T, dtype=torch.int64, scaled=T == 5)


@pytest.mark.parametrize("T, n, how", [(3000, 2, "runs"), (2900, 1, "one"), (4200, 3, "mixed"), (1500, 9, "runs")])
def test_groups_of_several_tiles(T, n, how, host):
    """Factors' gradients whose sums meet over several workgroups, and small ones beside large ones."""
    run(T, n, 8, 72, 136, how, seed=T)
    run(T, n, 40, 520, 16, how, seed=T)


@pytest.mark.parametrize("T, n, how", [(300, 2, "mixed"), (1000, 1, "one"), (70, 5, "runs"), (2900, 3, "mixed"), (1, 1, "one"), (65, 2, "none")])
@pytest.mark.parametrize("r, D", [(8, 8), (16, 136), (8, 520), (16, 1160), (16, 512), (24, 136), (32, 520), (24, 1160), (32, 8), (32, 512)])
def test_gradient_and_product_from_one_reading(T, n, how, r, D):
    """The factor's gradient is `outer`'s, the product within its error of 64 bits, rows of no adapter aside; values that are not finite stay in
    their tokens."""
    from lingua_amd import ops
    _, b, scale = bank(n, r, 8, D, seed=T)
    z = seeded_bf16((T, D), seed=1).cuda()
    h = torch.randn((2, T, r), generator=torch.Generator().manual_seed(2)).cuda()
    index = tokens_of(T, n, how, seed=T)
    plan = ops.lowrank_route(index, n)
    z[T // 2, D - 1] = float("inf")
    grad, also = ops.lowrank_outer_shrink(h, z, b, scale, plan)
    want, = ops.lowrank_outer([(h, z)], scale, n, r, plan)
    # (tiles of other sizes: sums in another order)
    bad = ~want.isfinite()
    assert torch.equal(bad, ~grad.isfinite())
    plain_sum = torch.zeros(b.shape, dtype=torch.float64)
    size = plain_sum.clone()
    hd, zd = h.double().sum(0).cpu(), z.double().cpu()
    for i in range(n):
        at = (index == i).nonzero()[:, 0].cpu()
        plain_sum[i] = float(scale[i]) * (hd[at].t() @ zd[at])
        size[i] = float(scale[i]) * (plain.SPLIT + plain.FP32 * (2 * len(at) + 24)) * (hd[at].abs().t() @ zd[at].abs())
    assert within(grad[~bad], plain_sum[~bad.cpu()], size[~bad.cpu()])
    for i in range(n):
        at = (index == i).nonzero()[:, 0].cpu()
        got, x, f = also[0].double().cpu()[at], zd[at], b[i].double().cpu()
        want = x @ f.t()
        fine = x.isfinite().all(1)
        assert bool(((got - want).abs() <= plain.FP32 * (D + 16) * (x.abs() @ f.abs().t()))[fine].all()) and not bool(got[~fine].isfinite().any())


@pytest.mark.parametrize("T, n, r", [(2300, 2, 16), (5000, 7, 32), (2048, 1, 24)])
def test_large_backward(T, n, r, host):
    """A pass that reads the gradient once for both."""
    from lingua_amd import ops
    K, N = 72, 8200
    assert ops.lowrank_outer_shrink_pays(T, r, N) and not ops.lowrank_outer_shrink_pays(T, 40, N) and not ops.lowrank_outer_shrink_pays(T, r, 4096)
    run(T, n, r, K, N, "mixed", seed=T)


@pytest.mark.parametrize("T", [1, 5, 64, 1023, 1024, 1025, 5000])
@pytest.mark.parametrize("n", [1, 3, 64, 200])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_route(T, n, dtype):
    """A stable order: adapters, then tokens without one, then strangers."""
    from lingua_amd import ops
    g = torch.Generator().manual_seed(T)
    index = torch.randint(-3, n + 2, (T,), generator=g)
    if dtype == torch.int64:
        index[::7] += 1 << 32       # (no adapter's, though its lower half may be)
    group = torch.where(index == -1, n, torch.where((index >= 0) & (index < n), index, n + 1))
    order, starts = ops.lowrank_route(index.to(dtype).cuda(), n)
    assert torch.equal(order.cpu().long(), group.sort(stable=True).indices)
    want = torch.cat((torch.zeros(1, dtype=torch.long), torch.bincount(group, minlength=n + 2).cumsum(0)))
    assert torch.equal(starts.cpu().long(), want)


@pytest.mark.parametrize("T", [40, 400])
def test_strangers_and_values_that_are_not_finite(T, host):
    """An index of no adapter makes its token NaN, an infinite or NaN token itself, and neither anything else; factors' gradients leave
    strangers out."""
    from lingua_amd import adapters
    n, r, K, N = 3, 16, 72, 136
    a, b, scale = bank(n, r, K, N)
    x, y, gy = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((T, N), std=0.1, seed=4).cuda()
    index = tokens_of(T, n, "mixed", 1)
    index[3], index[20], index[21] = n, -2, 2 ** 31 - 1
    strange = [3, 20, 21]
    x[3] = float("nan")
    leaves = [t.requires_grad_() for t in (x, a, b)]
    out = adapters.add_lowrank(y, *leaves, index, scale)
    gx, ga, gb = torch.autograd.grad(out, leaves, gy)
    assert bool(out[strange].isnan().all()) and bool(gx[strange].isnan().all())
    keep = [t for t in range(T) if t not in strange]
    sub = [t.detach()[keep].clone() for t in (y, x)]
    want, size, _, _ = plain.lowrank(*sub, a, b, index[keep], scale)
    assert within(out.detach()[keep], want, size)
    wants, sizes = plain.lowrank_grads(sub[1], a, b, index[keep], scale, gy[keep])
    assert within(gx[keep], wants[0], sizes[0]) and within(ga, wants[1], sizes[1]) and within(gb, wants[2], sizes[2])
    # a NaN and an infinity in two tokens of adapter 1, and in a token without one: every other token keeps its bits
    index[:] = 1
    index[::5] = 0
    index[7] = -1
    clean = adapters.add_lowrank(y, x.detach().nan_to_num(), a, b, index, scale)
    bad = x.detach().nan_to_num()
    bad[11, 5], bad[12, 60], bad[7, 0] = float("nan"), float("inf"), float("nan")
    got = adapters.add_lowrank(y, bad, a, b, index, scale)
    others = [t for t in range(T) if t not in (11, 12)]
    assert torch.equal(got[others], clean[others]) and bool(got[11].isnan().all()) and not bool(got[12].isfinite().any())
    # the last tokens of an adapter whose rows stand in for those behind them
    last = int((index == 0).nonzero()[-1])
    bad = x.detach().nan_to_num().requires_grad_()
    inf = gy.clone()
    inf[last, 3] = float("inf")
    ga2, gb2 = torch.autograd.grad(adapters.add_lowrank(y, bad, a, b, index, scale), (a, b), inf)
    ga1, gb1 = torch.autograd.grad(adapters.add_lowrank(y, bad, a, b, index, scale), (a, b), gy)
    assert torch.equal(ga2[1], ga1[1]) and torch.equal(gb2[1], gb1[1]) and torch.equal(gb2[0][:, 4:], gb1[0][:, 4:])
    # (infinite or NaN: h enters as two numbers, whose products with an infinity may be of different signs)
    assert not bool(gb2[0][:, 3].isfinite().any())


def test_strides_shapes_and_plans(host):
    from lingua_amd import adapters, ops
    n, r, K, N, T = 3, 16, 72, 136, 60
    a, b, scale = bank(n, r, K, N)
    wide = seeded_bf16((T, 400), seed=5).cuda()
    x, y = wide[:, 8:8 + K], wide[:, 96:96 + N]
    index = tokens_of(T, n, "mixed")
    want = adapters.add_lowrank(y.clone(), x.clone(), a, b, index, scale)
    assert torch.equal(adapters.add_lowrank(y, x, a, b, index, scale), want)
    odd = torch.zeros((T, 401), dtype=torch.bfloat16, device="cuda")[:, 1:]
    odd.copy_(wide)
    assert torch.equal(adapters.add_lowrank(odd[:, 96:96 + N], odd[:, 8:8 + K], a, b, index, scale), want)
    assert torch.equal(adapters.add_lowrank(y.t().contiguous().t(), x.t().contiguous().t(), a, b, index.repeat_interleave(2)[::2], scale), want)
    turned = a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(adapters.add_lowrank(y, x, *turned, index, scale), want)
    off = torch.empty(a.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(a.shape).copy_(a)
    assert torch.equal(adapters.add_lowrank(y, x, off, b, index, torch.stack((scale, scale), 1)[:, 0]), want)
    # leading dimensions, a plan for several calls, one token
    shaped = adapters.add_lowrank(y.reshape(3, 20, N), x.reshape(3, 20, K), a, b, index.view(3, 20), scale)
    assert shaped.shape == (3, 20, N) and torch.equal(shaped.view(T, N), want)
    plan = adapters.route(index.view(3, 20), n)
    for _ in range(2):
        assert torch.equal(adapters.add_lowrank(y.reshape(3, 20, N), x.reshape(3, 20, K), a, b, plan, scale).view(T, N), want)
    one = adapters.add_lowrank(y[4], x[4], a, b, index[4], scale)
    assert one.shape == (N,) and torch.equal(one, want[4])
    # in place, and beside rows that are another's
    h = ops.lowrank_shrink(x, a, (plan.order, plan.starts))
    big = torch.full((T + 2, N + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[:T, :N]
    assert ops.lowrank_expand(y, h, b, scale, (plan.order, plan.starts), out=out) is out and torch.equal(out, want)
    assert bool((big[T:] == 7).all()) and bool((big[:, N:] == 7).all())
    out.copy_(y)
    version = out._version
    ops.lowrank_expand(out, h, b, scale, (plan.order, plan.starts), out=out)
    assert torch.equal(out, want) and out._version > version
    with pytest.raises(RuntimeError, match="overlap"):
        ops.lowrank_expand(big[1:T + 1, :N], h, b, scale, (plan.order, plan.starts), out=out)


def test_no_tokens_and_repeated_runs(host):
    from lingua_amd import adapters
    n, r, K, N = 4, 16, 264, 520
    a, b, scale = (t.requires_grad_(t.dtype == torch.bfloat16) for t in bank(n, r, K, N))
    x = torch.empty((0, K), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = torch.empty((0, N), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = adapters.add_lowrank(y, x, a, b, torch.empty(0, dtype=torch.int32, device="cuda"), scale)
    grads = torch.autograd.grad(out, (x, y, a, b), out.detach())
    assert out.shape == (0, N) and not grads[2].any() and not grads[3].any()
    # the same bits every time
    T = 3000
    x, y, gy = seeded_bf16((T, K), seed=2).cuda().requires_grad_(), seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((T, N), std=0.1, seed=4).cuda()
    index = tokens_of(T, n, "mixed")
    first = None
    for _ in range(3):
        out = adapters.add_lowrank(y, x, a, b, index, scale)
        got = (out.detach(), *torch.autograd.grad(out, (x, a, b), gy))
        first = first or got
        assert all(torch.equal(u, v) for u, v in zip(got, first))


@pytest.mark.parametrize("which", ["y", "x", "a", "b", "xa", "ab", "none"])
def test_parts_of_the_gradient(which, host):
    from lingua_amd import adapters
    T, n, r, K, N = 70, 2, 24, 72, 136
    a, b, scale = bank(n, r, K, N)
    x, y, gy = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((T, N), std=0.1, seed=4).cuda()
    index = tokens_of(T, n, "mixed")
    full = {k: t.clone().requires_grad_() for k, t in zip("yxab", (y, x, a, b))}
    out = adapters.add_lowrank(*full.values(), index, scale)
    want = dict(zip("yxab", torch.autograd.grad(out, list(full.values()), gy)))
    some = {k: t.clone().requires_grad_(k in which and which != "none") for k, t in zip("yxab", (y, x, a, b))}
    got = adapters.add_lowrank(*some.values(), index, scale)
    assert torch.equal(got, out) and got.requires_grad == (which != "none")
    if which != "none":
        for k, g in zip(which, torch.autograd.grad(got, [some[k] for k in which], gy)):
            assert torch.equal(g, want[k])


def test_gradients_against_differences():
    """Central differences of the 64-bit form along random directions."""
    from lingua_amd import adapters
    T, n, r, K, N = 20, 2, 8, 24, 32
    a, b, scale = bank(n, r, K, N)
    x, y, gy = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((T, N), seed=4).cuda()
    index = tokens_of(T, n, "mixed")
    leaves = [t.requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(adapters.add_lowrank(y, *leaves, index, scale), leaves, gy)
    at = [t.detach().double() for t in leaves]
    for i in range(3):
        d = torch.randn(at[i].shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        ends = []
        for sign in (1, -1):
            moved = list(at)
            moved[i] = at[i] + sign * 1e-3 * d
            ends.append(float((plain.lowrank(y, *moved, index, scale)[0] * gy.double().cpu()).sum()))
        slope = (ends[0] - ends[1]) / 2e-3      # exact: the form is linear in each
        # a gradient's entries are off by half a bf16 step and by their sums' errors, which are far below that
        assert abs(float((grads[i].double() * d).sum()) - slope) <= 2.0 ** -7.9 * float((grads[i].double() * d).abs().sum()) + 1e-6 * abs(slope) + 1e-9


@pytest.mark.parametrize("T", [12, 300])
def test_captured_calls(T):
    """A serving call and a training step replayed with another index and other inputs equal the eager ones."""
    from lingua_amd import adapters
    n, r, K, N = 3, 16, 264, 136
    make = lambda: [t.requires_grad_(t.dtype == torch.bfloat16) for t in (seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((T, K), seed=2).cuda(), *bank(n, r, K, N))]  # noqa: E731
    gy = seeded_bf16((T, N), std=0.1, seed=4).cuda()
    index = tokens_of(T, n, "mixed")

    def step(y, x, a, b, scale):
        out = adapters.add_lowrank(y, x, a, b, index, scale)
        return (out.detach(), *torch.autograd.grad(out, (x, a, b), gy))

    leaves = make()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*leaves)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves)
    for i in range(3):
        index.copy_(tokens_of(T, n, "mixed", seed=50 + i))
        with torch.no_grad():
            leaves[1].copy_(seeded_bf16((T, K), seed=60 + i))
        eager = make()
        with torch.no_grad():
            eager[1].copy_(leaves[1])
        want = step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("kind", ["fp8", "mxfp4", "plain"])
def test_modules(kind):
    """Banks beside a model's linears: nothing changes while they are fresh or no request has one; a loaded adapter is the merged weight's
    low-rank part; the linears' parameters keep learning or stay frozen as they were."""
    from bench_workloads import FeedForward
    from lingua_amd import adapters, convert_linears_to_fp8, mxfp4
    model = torch.nn.ModuleDict({"mlp": FeedForward(128, 352)}).to("cuda", torch.bfloat16)
    if kind == "fp8":
        convert_linears_to_fp8(model, "rowwise", "w[123]")
    elif kind == "mxfp4":
        mxfp4.convert_linears_to_mxfp4(model, "w[123]")
    model.requires_grad_(False)
    x = seeded_bf16((2, 24, 128), seed=1).cuda()
    want = model["mlp"](x)
    requests = adapters.Requests(3)
    adapters.add_adapters(model, requests, 16, r"w[12]$", alpha=32)
    adapters.add_adapters(model, requests, 16, r"w[12]")      # (the linears inside are not adapted twice)
    assert type(model["mlp"].w1) is type(model["mlp"].w2) is adapters.AdaptedLinear and type(model["mlp"].w3) is not adapters.AdaptedLinear
    assert type(model["mlp"].w1.linear) is not adapters.AdaptedLinear and float(model["mlp"].w1.scale[0]) == 2
    index = torch.tensor([0, 2], device="cuda")[:, None].expand(2, 24)
    assert torch.equal(model["mlp"](x), want)
    requests.set(index)
    assert torch.equal(model["mlp"](x), want)
    down, up = seeded_bf16((8, 128), std=0.1, seed=5).cuda(), seeded_bf16((352, 8), std=0.1, seed=6).cuda()
    model["mlp"].w1.load(2, down, up, scale=0.5)
    w1 = model["mlp"].w1
    y, base = w1(x), w1.linear(x)
    assert torch.equal(y[0], base[0])
    a, b = down[None], up.t()[None].contiguous()
    ref, size, _, _ = plain.lowrank(base[1], x[1], a, b, torch.zeros(24, dtype=torch.long), torch.tensor([0.5]))
    # (the bank's rank is 16: eight ranks of zeros more)
    assert within(y[1], ref, 2 * size)
    requests.set(None)
    assert torch.equal(model["mlp"](x), want)
    requests.set(index)
    grads = torch.autograd.grad(model["mlp"](x).float().square().sum(), [p for p in model.parameters() if p.requires_grad])
    assert len(grads) == 4 and all(bool(g.isfinite().all()) for g in grads)
    assert not grads[0][1].any() and grads[0][2].any()      # adapter 1 has no request; the first's b is zero, and its a learns nothing yet
    with pytest.raises(RuntimeError, match="do not fit"):
        w1.load(3, down, up)


def test_requests_of_a_captured_model():
    """A captured forward pass of an adapted linear sees the requests that are set between its replays; another batch size in between leaves it
    alone; setting requests between a forward and its backward pass is an error; a model that was rounded to bf16 as a whole still runs."""
    from lingua_amd import adapters
    requests = adapters.Requests(3)
    lin = adapters.AdaptedLinear(torch.nn.Linear(64, 128, bias=False, dtype=torch.bfloat16, device="cuda"), requests, 8)
    with torch.no_grad():
        lin.b.copy_(seeded_bf16((3, 8, 128), std=0.3, seed=1))
    lin.to(torch.bfloat16)
    assert lin.scale.dtype == torch.bfloat16
    x = seeded_bf16((40, 64), seed=2).cuda()
    first = torch.arange(40, device="cuda") % 4 - 1
    requests.set(first)
    with torch.no_grad():
        lin(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(x)
        for i in range(3):
            requests.set(torch.zeros(7 + i, dtype=torch.int32, device="cuda"))
            lin(x[:7 + i])
            index = first.roll(i)
            requests.set(index)
            want = adapters.add_lowrank(lin.linear(x), x, lin.a, lin.b, index, lin.scale.float())
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lin(x), want)
    y = lin(x)
    requests.set(first)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inference_mode():
    """Tensors without version counters go through every operator."""
    from lingua_amd import adapters, dropout, norm, rope
    n, r, K, N, T = 3, 16, 64, 128, 100
    a, b, scale = bank(n, r, K, N)
    x, y, w = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda(), seeded_bf16((K,), seed=4).cuda()
    index, drop = tokens_of(T, n, "mixed"), dropout.Drop(0.2, dropout.numbers(1))
    cos, sin = (t.cuda() for t in rope.rotary_tables(32, 200))
    pos = torch.arange(2 * T, device="cuda").view(2, 1, T)

    def run():
        requests = adapters.Requests(n)
        requests.set(index)
        requests.set(index)
        return (adapters.add_lowrank(y, x, a, b, index, scale), adapters.add_lowrank(y, x, a, b, requests.plan, scale), norm.layernorm(x, w, w, quantise=True),
                *norm.add_layernorm(x, x, w, dropout=drop), *norm.add_rmsnorm(x, x, w, 1e-5, drop), dropout.dropout(x, drop),
                *rope.rotary_axes(x.view(1, T, 2, 32), x.view(1, T, 2, 32), cos, sin, pos, (8, 8)))

    want = run()
    with torch.inference_mode():
        x, y = x.clone(), y.clone()
        assert all(torch.equal(u, v) for u, v in zip(run(), want))


def test_requests_first_set_in_inference_mode():
    """A batch shape that an evaluation in inference mode had first is trained on afterwards, and the other way round."""
    from lingua_amd import adapters
    n, r, K, N, T = 3, 16, 64, 128, 100
    a, b, scale = bank(n, r, K, N)
    x, y, index = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda(), tokens_of(T, n, "mixed")
    want = adapters.add_lowrank(y, x, a, b, index, scale)
    requests = adapters.Requests(n)
    with torch.inference_mode():
        requests.set(index.clone())
        assert torch.equal(adapters.add_lowrank(y, x, a, b, requests.plan, scale), want)
    for k in range(2):
        requests.set(index.roll(k))
        leaf = a.clone().requires_grad_()
        got = adapters.add_lowrank(y, x, leaf, b, requests.plan, scale)
        assert torch.equal(got, adapters.add_lowrank(y, x, a, b, index.roll(k), scale))
        got.float().sum().backward()
        assert leaf.grad.isfinite().all()
        with torch.inference_mode():
            requests.set(index)
            assert torch.equal(adapters.add_lowrank(y, x, a, b, requests.plan, scale), want)


@pytest.mark.parametrize("r", [16, 32, 64])
@pytest.mark.parametrize("T, n", [(40, 3), (300, 2), (1000, 70)])
def test_an_order_that_route_did_not_make(T, n, r):
    """Contents of an order that has not been written yet: results are whatever they are, and what lies around the outputs stays as it was."""
    from lingua_amd import ops
    K, N, guard = 72, 136, 64
    a, b, scale = bank(n, r, K, N)
    x, y = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda()
    g = torch.Generator().manual_seed(T + r)
    for k in range(4):
        low, high = [(-2 ** 31, 2 ** 31), (-5, T + 5), (0, 1), (T, T + 1)][k]
        plan = tuple(torch.randint(low, high, (m,), generator=g).int().cuda() for m in (T, n + 3))
        h = ops.lowrank_shrink(x, a, plan)
        out = torch.full((T + 2 * guard, N), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.lowrank_expand(y, torch.zeros_like(h), b, scale, plan, out[guard:guard + T])
        grads = ops.lowrank_outer([(h, x), (h, y)], scale, n, r, plan)
        if r <= 32:
            ops.lowrank_outer_shrink(h, y, b, scale, plan)
        torch.cuda.synchronize()
        assert (out[:guard] == 7).all() and (out[guard + T:] == 7).all() and [t.shape for t in grads] == [a.shape, b.shape]


def test_requests_of_many_shapes():
    """Batches of ever other sizes do not pile up memory; the shape that a captured pass reads stays."""
    from lingua_amd import adapters
    requests = adapters.Requests(3)
    lin = adapters.AdaptedLinear(torch.nn.Linear(64, 128, bias=False, dtype=torch.bfloat16, device="cuda"), requests, 8)
    x = seeded_bf16((300, 64), seed=2).cuda()
    with torch.no_grad():
        lin.b.copy_(seeded_bf16((3, 8, 128), std=0.3, seed=1))
        index = torch.arange(40, device="cuda") % 4 - 1
        requests.set(index)
        lin(x[:40])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(x[:40])
        for T in range(1, 300):
            requests.set(torch.full((T,), T % 3, dtype=torch.int32, device="cuda"))
            if T % 50 == 0:
                want = adapters.add_lowrank(lin.linear(x[:T]), x[:T], lin.a, lin.b, torch.full((T,), T % 3, device="cuda"), lin.scale)
                assert torch.equal(lin(x[:T]), want)
        assert len(requests._plans) <= 66
        with pytest.raises(RuntimeError, match="int32 or int64"):
            requests.set(index.float())     # (and what the graph reads is still there)
        assert (40,) in [k[0] for k in requests._plans]
        for i in range(2):
            requests.set(index.roll(i))
            want = adapters.add_lowrank(lin.linear(x[:40]), x[:40], lin.a, lin.b, index.roll(i), lin.scale)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_compiled_module():
    from lingua_amd import adapters
    requests = adapters.Requests(3)
    lin = adapters.AdaptedLinear(torch.nn.Linear(64, 128, bias=False, dtype=torch.bfloat16, device="cuda"), requests, 8)
    with torch.no_grad():
        lin.b.copy_(seeded_bf16((3, 8, 128), std=0.3, seed=1))
    x = seeded_bf16((40, 64), seed=2).cuda()
    compiled = torch.compile(lin, backend="eager")
    for i in range(2):
        requests.set((torch.arange(40, device="cuda") + i) % 4 - 1)
        want, got = lin(x), compiled(x)
        assert torch.equal(got, want)
        for u, v in zip(torch.autograd.grad(got.float().sum(), (lin.a, lin.b)), torch.autograd.grad(want.float().sum(), (lin.a, lin.b))):
            assert torch.equal(u, v)
