"""A run of layer norm, dropout, rotary positions on several axes and low-rank adapters, as a model uses them: in training inside a block for
text and patches, in generation as one captured step; and what every operator owes its callers -- captures, compilers, threads, hooks,
second derivatives."""
import pytest
import torch
import torch.nn.functional as F

import plain_more as plain
from bench_workloads import FeedForward
from conftest import seeded_bf16
from plain_operators import host, within  # noqa: F401

pytestmark = pytest.mark.gpu

SECTIONS = (4, 6, 6)


class Attention(torch.nn.Module):
    def __init__(self, dim, heads):
        super().__init__()
        self.heads = heads
        self.wq, self.wk, self.wv, self.wo = (torch.nn.Linear(dim, dim, bias=False) for _ in range(4))

    def forward(self, x, cos, sin, positions):
        from lingua_amd import rope
        B, S, D = x.shape
        q, k, v = (w(x).view(B, S, self.heads, -1) for w in (self.wq, self.wk, self.wv))
        q, k = rope.rotary_axes(q, k, cos, sin, positions, SECTIONS, order="rounds", layout="half")
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        return self.wo(o.transpose(1, 2).reshape(B, S, D))


class Block(torch.nn.Module):
    def __init__(self, dim, heads, hidden):
        super().__init__()
        self.attention, self.feed_forward = Attention(dim, heads), FeedForward(dim, hidden)
        self.attention_norm, self.ffn_norm = torch.nn.LayerNorm(dim), torch.nn.LayerNorm(dim)
        self.drop, self.drop2 = torch.nn.Dropout(0.1), torch.nn.Dropout(0.2)

    def forward(self, x, fused, *where):
        from lingua_amd import dropout
        a = self.attention(self.attention_norm(x), *where)
        if fused:
            h, y = self.ffn_norm.add(a, x, self.drop.drop())
        else:
            h = dropout.dropout_add(a, x, self.drop.drop()) if self.training else a + x
            y = self.ffn_norm(h)
        return h + self.drop2(self.feed_forward(y))


def model_of(numbers):
    """Two blocks: frozen fp8 attention and MXFP4 MLP, adapters beside some of their linears, layer norms that learn."""
    from lingua_amd import adapters, convert_linears_to_fp8, dropout, mxfp4, norm
    model = torch.nn.ModuleDict({"layers": torch.nn.ModuleList([Block(128, 4, 368) for _ in range(2)])}).to("cuda", torch.bfloat16)
    with torch.no_grad():
        for i, p in enumerate(model.parameters()):
            p.copy_(seeded_bf16(tuple(p.shape), std=0.08, seed=i) + (p.dim() == 1))
    convert_linears_to_fp8(model, "rowwise", "attention")
    mxfp4.convert_linears_to_mxfp4(model, "feed_forward")
    for name, p in model.named_parameters():
        p.requires_grad_("norm" in name)
    norm.fuse_layernorm(model)
    dropout.convert_dropouts(model, numbers)
    requests = adapters.Requests(3)
    adapters.add_adapters(model, requests, 8, r"w[qv]$|w2$")
    with torch.no_grad():
        for i, m in enumerate(m for m in model.modules() if isinstance(m, adapters.AdaptedLinear)):
            m.a.copy_(seeded_bf16(tuple(m.a.shape), std=0.1, seed=100 + i))
            m.b.copy_(seeded_bf16(tuple(m.b.shape), std=0.1, seed=200 + i))
    return model, requests


def places(B, S):
    at = torch.arange(S, device="cuda")
    steps = torch.stack((at // 16, at // 4 % 4, at % 4))[:, None]
    return torch.where(at < 6, at, 6 + steps).expand(3, B, S).contiguous()


def test_training_steps():
    """The fused sums give the bits of the sums and norms one by one; a step repeated gives its bits again, the next step others; an adapter
    that no request has learns nothing; without gradients the same logits; in evaluation nothing is dropped."""
    from lingua_amd import dropout, rope
    n = dropout.numbers(11)
    model, requests = model_of(n)
    B, S = 3, 29
    x = seeded_bf16((B, S, 128), seed=1).cuda().requires_grad_()
    g = seeded_bf16((B, S, 128), std=0.1, seed=2).cuda()
    where = (*(t.cuda() for t in rope.rotary_tables(2 * sum(SECTIONS), 64)), places(B, S))
    index = torch.tensor([0, -1, 2], device="cuda")[:, None].expand(B, S)
    learning = [p for p in model.parameters() if p.requires_grad]

    def forward(fused=True):
        y = x
        for layer in model["layers"]:
            y = layer(y, fused, *where)
        return y

    def step():
        requests.set(index)
        y = forward()
        return (y.detach(), *torch.autograd.grad(y, (x, *learning), g))

    first = step()
    assert all(bool(t.isfinite().all()) for t in first)
    assert torch.equal(first[0], forward(fused=False))
    with torch.no_grad():
        assert torch.equal(first[0], forward())
    assert all(torch.equal(a, b) for a, b in zip(step(), first))
    banks = [t for t, p in zip(first[2:], learning) if p.dim() == 3]
    assert len(banks) == 12 and all(not b[1].any() and b[0].any() and b[2].any() for b in banks)
    n[1] += 1
    assert not torch.equal(step()[0], first[0])
    model.eval()
    with torch.no_grad():
        assert torch.equal(forward(), forward(fused=False))


def test_generation_step_in_a_graph():
    """Residual layer norm, a packed projection and its adapters, rotary positions: one captured step for several sequences, replayed with new
    tokens, positions and adapters and with eager work in between, equals the eager step."""
    from lingua_amd import adapters, mxfp4, norm, rope
    B, dim, H, D = 5, 256, 4, 64
    packed = mxfp4.pack(seeded_bf16((2 * H * D, dim), std=0.05, seed=1).cuda())
    a, b = seeded_bf16((4, 16, dim), std=0.06, seed=2).cuda(), seeded_bf16((4, 16, 2 * H * D), std=0.1, seed=3).cuda()
    w, bias = seeded_bf16((dim,), seed=4).cuda(), seeded_bf16((dim,), seed=5).cuda()
    cos, sin = (t.cuda() for t in rope.axes_tables((8, 12, 12), 5000))
    x, res = seeded_bf16((B, dim), seed=6).cuda(), seeded_bf16((B, dim), seed=7).cuda()
    pos, index = torch.arange(3 * B, device="cuda").view(3, B, 1), torch.tensor([0, 3, -1, 3, 1], device="cuda")

    def step():
        h, y = norm.add_layernorm(x, res, w, bias)
        qk = adapters.add_lowrank(mxfp4.linear_packed(y, *packed), y, a, b, index).view(B, 1, 2 * H, D)
        return (h, *rope.rotary_axes(qk[:, :, :H], qk[:, :, H:], cos, sin, pos, (8, 12, 12)))

    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(3):
            x.copy_(seeded_bf16((B, dim), seed=20 + i))
            pos.add_(131)
            index.copy_(index.roll(1))
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want))


NAMES = ["layernorm", "add_layernorm", "add_rmsnorm", "dropout", "dropout_add", "rotary_axes", "add_lowrank"]


def make(name, seed=0):
    """An operator's call on leaves of its own -> (call, leaves that its gradient asks for)."""
    from lingua_amd import adapters, dropout, norm, rope
    x, res, w, b = (seeded_bf16(s, std=0.5, seed=seed + i).cuda().requires_grad_() for i, s in enumerate(((16, 64), (16, 64), (64,), (64,))))
    a, c = (seeded_bf16((3, 8, 64), std=0.3, seed=seed + 5 + i).cuda().requires_grad_() for i in range(2))
    cos, sin = (t.cuda() for t in rope.rotary_tables(32, 50))
    drop = dropout.Drop(0.3, dropout.numbers(seed))
    index = torch.tensor([0, 2, -1, 1] * 4, device="cuda")
    pos = torch.arange(48, device="cuda").view(3, 1, 16)
    rows = lambda t: t.view(1, 16, 2, 32)  # noqa: E731
    return {"layernorm": (lambda: norm.layernorm(x, w, b), (x, w, b)),
            "add_layernorm": (lambda: norm.add_layernorm(x, res, w, b, dropout=drop)[1], (x, res, w, b)),
            "add_rmsnorm": (lambda: norm.add_rmsnorm(x, res, w, 1e-5, drop)[1], (x, res, w)),
            "dropout": (lambda: dropout.dropout(x, drop), (x,)),
            "dropout_add": (lambda: dropout.dropout_add(x, res, drop), (x, res)),
            "rotary_axes": (lambda: rope.rotary_axes(rows(x), rows(res), cos, sin, pos, (4, 6, 6))[0].view(16, 64), (x,)),
            "add_lowrank": (lambda: adapters.add_lowrank(res, x, a, c, index, torch.ones(3, device="cuda")), (res, x, a, c))}[name]


GY = dict(std=0.1, seed=9)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", [n for n in NAMES if n != "rotary_axes"])     # (whose leaf is behind a view here)
def test_capture_is_refused_while_a_graph_of_the_leaves_lives(name, native, monkeypatch):
    from lingua_amd import float8
    if not native:
        monkeypatch.setattr(float8, "_plain_call", lambda: False)
    call, _ = make(name)
    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match=f"{name}: captured while .* same leaf"):
            call()
        with torch.no_grad():
            out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.detach())


@pytest.mark.parametrize("name", NAMES)
def test_compiled_calls_equal_eager_ones(name):
    call, leaves = make(name)
    torch._dynamo.reset()
    want, got = call() * 2.0, torch.compile(lambda: call() * 2.0, backend="eager")()
    torch._dynamo.reset()
    gy = seeded_bf16((16, 64), **GY).cuda()
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, gy), torch.autograd.grad(want, leaves, gy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name, host):
    """A gradient that was made for differentiation has the bits of an ordinary one, and whoever asks for its derivative gets an error, or,
    where it varies with nothing but the incoming gradient and that is a constant, a constant."""
    call, leaves = make(name)
    said = {"dropout_add": "dropout", "rotary_axes": "rotary"}.get(name, name)
    ordinary = torch.autograd.grad(call().float().square().sum(), leaves)
    loss = call().float().square().sum()
    grads = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(g, o) for g, o in zip(grads, ordinary))
    passed_on = {"dropout_add": (1,), "add_lowrank": (0,)}.get(name, ())     # the residual's and the projection's: the incoming gradient itself
    for i, g in enumerate(grads):
        if i not in passed_on:
            with pytest.raises(RuntimeError, match=f"{said} is not differentiable twice"):
                (loss + g.float().square().sum()).backward(retain_graph=True)
    constant = torch.autograd.grad(call(), leaves, torch.ones((16, 64), dtype=torch.bfloat16, device="cuda"), create_graph=True)
    linear = {"dropout": (0,), "dropout_add": (0, 1), "rotary_axes": (0,), "add_lowrank": (0,), "layernorm": (2,), "add_layernorm": (3,)}.get(name, ())
    for i, g in enumerate(constant):
        assert g.requires_grad == (i not in linear)


@pytest.mark.parametrize("name", NAMES)
def test_kept_operands_in_other_layouts(name, host):
    """Hooks on saved tensors hand every second operand back with its elements apart: the gradients are the same."""
    call, leaves = make(name)
    gy = seeded_bf16((16, 64), **GY).cuda()
    want = torch.autograd.grad(call(), leaves, gy)
    for parity in (0, 1):
        kept = []

        def pack(t):
            kept.append(t)
            return torch.stack((t, torch.full_like(t, 7)), -1)[..., 0] if len(kept) % 2 == parity else t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = call()
        assert kept
        for got, w in zip(torch.autograd.grad(y, leaves, gy), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("name", NAMES)
def test_gradients_of_any_layout(name, host):
    """Incoming gradients that are broadcast, transposed or off their lines."""
    call, leaves = make(name)
    dense = seeded_bf16((16, 64), **GY).cuda()
    one = torch.tensor(0.5, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros((16, 67), dtype=torch.bfloat16, device="cuda")[:, 3:]
    off.copy_(dense)
    for gy in (one.expand(16, 64), dense.t().contiguous().t(), off, dense[:1].expand(16, 64)):
        for got, w in zip(torch.autograd.grad(call(), leaves, gy), torch.autograd.grad(call(), leaves, gy.contiguous().clone())):
            assert torch.equal(got, w)


@pytest.mark.parametrize("name", NAMES)
def test_results_may_be_written_in_place(name, host):
    call, leaves = make(name)
    gy = seeded_bf16((16, 64), **GY).cuda()
    want = torch.autograd.grad(call() * 2.0, leaves, gy)
    y = call()
    y.mul_(2.0)
    for got, w in zip(torch.autograd.grad(y, leaves, gy), want):
        assert torch.equal(got, w)


def test_operands_do_not_share_a_gradient(host):
    from lingua_amd import dropout, norm
    x, res, w = (seeded_bf16(s, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (8, 64), (64,))))
    for drop in (None, dropout.Drop(0.5, dropout.numbers(1))):
        for t in (x, res, w):
            t.grad = None
        for _ in range(2):
            h, y = norm.add_layernorm(x, res, w, dropout=drop)
            (h.sum() + y.sum()).backward()
        assert x.grad.data_ptr() != res.grad.data_ptr()
        assert drop is not None or torch.equal(x.grad, res.grad)


def test_threads_at_once():
    """Four threads, each on a stream of its own, through every operator forward and backward: the results of one after the other."""
    import threading
    gy = seeded_bf16((16, 64), **GY).cuda()
    sets = [[make(name, seed=10 * i) for name in NAMES] for i in range(4)]

    def step(calls):
        out = []
        for call, leaves in calls:
            y = call()
            out += [y.detach(), *torch.autograd.grad(y, leaves, gy)]
        return out

    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = step(sets[i])
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(u, v) for u, v in zip(a, b))


def test_two_graphs_at_once():
    """Two captured steps replayed side by side on two streams share no workspace."""
    from lingua_amd import adapters, norm
    T, n, r, K, N = 400, 3, 16, 264, 520
    a, b = seeded_bf16((n, r, K), std=0.06, seed=1).cuda(), seeded_bf16((n, r, N), std=0.3, seed=2).cuda()
    w = torch.ones(K, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    index = (torch.arange(T, device="cuda") % 4 - 1).int()
    ins = [(seeded_bf16((T, K), seed=10 + i).cuda(), seeded_bf16((T, N), seed=20 + i).cuda()) for i in range(2)]
    g = seeded_bf16((T, K), std=0.1, seed=5).cuda()

    def step(x, y):
        z = norm.layernorm(x, w)
        gw, = torch.autograd.grad(z, w, g)
        with torch.no_grad():
            return z.detach(), gw, adapters.add_lowrank(y, z, a, b, index)

    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)], []
    for s, i in zip(streams, ins):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*i)
    torch.cuda.synchronize()
    for s, gr, i in zip(streams, graphs, ins):
        with torch.cuda.graph(gr, stream=s):
            outs.append(step(*i))
    for k in range(3):
        for i in ins:
            i[0].copy_(seeded_bf16((T, K), seed=50 + k))
            i[0].mul_(1 + k)
        torch.cuda.synchronize()
        for _ in range(5):
            for s, gr in zip(streams, graphs):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        w.requires_grad_()
        with torch.cuda.stream(streams[0]):
            want = [step(*i) for i in ins]
        torch.cuda.synchronize()
        for out, t in zip(outs, want):
            assert all(torch.equal(u, v) for u, v in zip(out, t))


def test_wide_projections_of_many_tokens():
    """Workgroups that go on over several stretches of columns, the last of them beyond the last column."""
    from lingua_amd import adapters
    T, n, K, N = 8200, 3, 72, 2056
    index = torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(1)).cuda()
    index[17] = 7
    x, y = seeded_bf16((T, K), seed=2).cuda(), seeded_bf16((T, N), seed=3).cuda()
    for r in (24, 40, 128):
        a, b = seeded_bf16((n, r, K), std=0.1, seed=4).cuda(), seeded_bf16((n, r, N), std=0.1, seed=5).cuda()
        out = adapters.add_lowrank(y, x, a, b, index)
        keep = torch.arange(T, device="cuda") != 17
        want, size, _, _ = plain.lowrank(y[keep], x[keep], a, b, index[keep], None)
        assert bool(out[17].isnan().all()) and within(out[keep], want, size)
        assert torch.equal(out[index < 0], y[index < 0])


def test_more_than_two_to_the_31st():
    """Operands of more than 2^31 elements: what the operators make of the last rows is what they make of those rows alone."""
    from lingua_amd import dropout, ops
    R, C, tail = 540672, 4096, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    for i in range(0, R, 1 << 16):
        x[i:i + (1 << 16)] = torch.randn(x[i:i + (1 << 16)].shape, generator=g, device="cuda")
    w = x[0].clone()
    h, y, q, scale, stats = ops.layernorm_cast_rowwise(x, w, None, 1e-5, residual=x)
    want = ops.layernorm_cast_rowwise(x[-tail:], w, None, 1e-5, residual=x[-tail:])
    for a, b in zip((h, y, q, scale), want):
        assert torch.equal(a[-tail:].view(torch.uint8), b.view(torch.uint8))
    del h, q, scale, want
    gx, _, gw, gb = ops.layernorm_bwd(x, None, x, w, stats, gw_dtype=torch.float32, gb_dtype=torch.float32)
    want = ops.layernorm_bwd(x[-tail:], None, x[-tail:], w, stats[:, -tail:])[0]
    assert torch.equal(gx[-tail:], want) and bool(gw.isfinite().all()) and bool(gb.isfinite().all())
    del gx, gw, gb, stats
    drop = dropout.Drop(0.5, dropout.numbers(3))
    hd = ops.layernorm_cast_rowwise(x, w, None, 1e-5, residual=y, drop=drop, want_q=False)[0]
    assert torch.equal(hd, ops.dropout(x, drop, residual=y))
    del hd, y
    # tokens whose rows lie beyond 2^31 elements, in a bank of one
    index = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    index[-tail:] = 0
    a, b = seeded_bf16((1, 8, C), std=0.02, seed=1).cuda(), seeded_bf16((1, 8, C), std=0.3, seed=2).cuda()
    out = ops.lowrank_add(x, x, a, b, index)
    # (few tokens alone share K out differently: the sums' last bits may differ)
    want, size, _, _ = plain.lowrank(x[-tail:], x[-tail:], a, b, index[-tail:], None)
    assert within(out[-tail:], want, size) and torch.equal(out[:-tail], x[:-tail])


def test_broadcast_and_transposed_operands(host):
    """Operands whose rows are one row, and whose rows lie apart: results those of dense copies, gradients summed over what was broadcast."""
    from lingua_amd import adapters, dropout, norm, rope
    R, C = 24, 64
    drop = dropout.Drop(0.3, dropout.numbers(4))
    a, b = (seeded_bf16((3, 8, C), std=0.3, seed=5 + i).cuda() for i in range(2))
    w, gy = seeded_bf16((C,), seed=8).cuda(), seeded_bf16((R, C), **GY).cuda()
    index = torch.tensor([1], device="cuda").expand(R)
    cos, sin = (t.cuda() for t in rope.rotary_tables(32, 50))
    pos = torch.tensor([3], device="cuda").expand(2, 1, R)
    heads = lambda t: t.view(1, R, 2, 32) if t.stride(0) else t.unflatten(1, (2, 32))[None]  # noqa: E731
    calls = {"layernorm": lambda x, r: norm.layernorm(x, w, w), "add_layernorm": lambda x, r: norm.add_layernorm(x, r, w, dropout=drop)[1],
             "add_rmsnorm": lambda x, r: norm.add_rmsnorm(x, r, w, 1e-5, drop)[1], "dropout": lambda x, r: dropout.dropout(x, drop),
             "dropout_add": lambda x, r: dropout.dropout_add(x, r, drop), "add_lowrank": lambda x, r: adapters.add_lowrank(r, x, a, b, index),
             "rotary_axes": lambda x, r: rope.rotary_axes(heads(x), heads(r), cos, sin, pos, (8, 8))[0].reshape(R, C)}
    leaf, wide = seeded_bf16((1, C), seed=1).cuda().requires_grad_(), seeded_bf16((C, R), seed=2).cuda().requires_grad_()
    for name, call in calls.items():
        for x, r in ((leaf.expand(R, C), wide.t()), (wide.t(), leaf.expand(R, C))):
            dense = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (x, r)]
            y, want = call(x if name != "rotary_axes" else x.contiguous(), r if name != "rotary_axes" else r.contiguous()), call(*dense)
            assert torch.equal(y, want), name
            got = torch.autograd.grad(y, (leaf, wide), gy, allow_unused=True)
            ref = torch.autograd.grad(want, dense, gy, allow_unused=True)
            ref = ref if x.shape == (R, C) and x.stride(0) == 0 else ref[::-1]
            for g, d, t in zip(got, ref, (leaf, wide)):
                if d is None:
                    assert g is None or not g.any()
                elif t is wide:
                    assert torch.equal(g, d.t()), name
                else:   # 24 rows added up in torch's order, rounded once
                    total = d.double().sum(0, keepdim=True)
                    assert bool(((g.double() - total).abs() <= 2.0 ** -8 * total.abs() + 25 * 2.0 ** -8 * 2.0 ** -8 * d.double().abs().sum(0)).all()), name


def test_copied_models():
    """A deep copy has its own numbers and requests, and computes what the model does."""
    import copy
    from lingua_amd import adapters, dropout
    numbers, requests = dropout.numbers(3), adapters.Requests(2)
    model = torch.nn.Sequential(torch.nn.Linear(64, 64, bias=False, dtype=torch.bfloat16, device="cuda"), torch.nn.Dropout(0.5))
    adapters.add_adapters(model, requests, 8, "0")
    dropout.convert_dropouts(model, numbers)
    with torch.no_grad():
        model[0].b.copy_(seeded_bf16((2, 8, 64), seed=1))
    x = seeded_bf16((10, 64), seed=2).cuda()
    index = torch.arange(10, device="cuda") % 3 - 1
    requests.set(index)
    other = copy.deepcopy(model)
    want = model(x)
    assert torch.equal(other(x), want)
    requests.set(None)
    numbers[1] += 1
    assert torch.equal(other(x), want) and not torch.equal(model(x), want)
    other[0].requests.set(index.roll(1))
    requests.set(index)
    numbers[1] -= 1
    assert torch.equal(model(x), want)
