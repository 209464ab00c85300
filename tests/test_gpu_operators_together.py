"""A run of the residual norm, the rotary positions and MXFP4 linears, as a model uses them: in training inside the stand-in model of the
benchmark, and in generation as one captured step."""
import pytest
import torch
import torch.nn.functional as F

import plain_operators as plain
from bench_workloads import Attention, Llama
from conftest import seeded_bf16
from plain_operators import host  # noqa: F401

pytestmark = pytest.mark.gpu


class RotaryAttention(Attention):
    """The stand-in attention with its rotary positions by the kernel."""

    def forward(self, x, cos, sin):
        from lingua_amd import rope
        B, S, _ = x.shape
        q, k, v = (lin(x).view(B, S, self.n_heads, self.head_dim) for lin in (self.wq, self.wk, self.wv))
        q, k = rope.rotary(q, k, cos, sin)
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        return self.wo(o.transpose(1, 2).reshape(B, S, -1))


def model_of(new):
    """fp8 attention, MXFP4 MLP; `new`: with the residual norm and the rotary kernel in place of the eager chains."""
    from lingua_amd import convert_linears_to_fp8, mxfp4, norm
    from lingua_amd.qkv import fuse_qkv
    model = Llama(n_layers=2, dim=256, n_heads=4, ffn_dim=720, vocab=64).to("cuda", torch.bfloat16)
    model.init_weights(seed=1)
    convert_linears_to_fp8(model, "rowwise", r"layers\.[0-9]+\.attention\.")
    mxfp4.convert_linears_to_mxfp4(model, r"layers\.[0-9]+\.feed_forward\.")
    norm.fuse_rmsnorm(model)
    fuse_qkv(model)
    if new:
        norm.fuse_residual_norm(model)
        for layer in model.layers:
            layer.attention.__class__ = RotaryAttention
    return model


def sum_error(a, b, K):
    return (a.abs() @ b.abs().t()) * (K * plain.FP32)


def test_training_step():
    """Logits are those of the model without the two fusions, bit for bit; every MXFP4 linear's output and gradients are what the format
    makes of its own input, weight and output gradient; a second step gives the same bits."""
    from lingua_amd import mxfp4
    tokens = torch.randint(0, 64, (3, 37), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        plain_logits = model_of(False)(tokens)
    model = model_of(True)
    seen = []

    def keep(module, args, out):
        entry = {"module": module, "x": args[0].detach().flatten(end_dim=-2), "y": out.detach().flatten(end_dim=-2)}
        args[0].register_hook(lambda g: entry.update(gx_sum=g.detach()))
        out.register_hook(lambda g: entry.update(gy=g.detach().flatten(end_dim=-2)))
        seen.append(entry)

    handles = [m.register_forward_hook(keep) for m in model.modules() if type(m) is mxfp4.Mxfp4Linear]
    logits = model(tokens)
    assert torch.equal(logits, plain_logits)
    F.cross_entropy(logits.flatten(0, 1).float(), tokens.flatten()).backward()
    for h in handles:
        h.remove()
    assert len(seen) == 6
    q = plain.mx_rounded
    for e in seen:
        x, w, gy = e["x"].cpu(), e["module"].weight.detach().cpu(), e["gy"].cpu()
        want = q(x) @ q(w).t()
        assert plain.within(e["y"], want, sum_error(q(x), q(w), x.shape[1]))
        gt, xt = q(gy.t().contiguous()), q(x.t().contiguous())
        assert plain.within(e["module"].weight.grad, gt @ xt.t(), sum_error(gt, xt, x.shape[0]))
        if e["module"] in [layer.feed_forward.w2 for layer in model.layers]:   # (w1 and w3 share an input: autograd adds two gradients)
            gn, wn = q(gy), q(w.t().contiguous())
            assert plain.within(e["gx_sum"].flatten(end_dim=-2), gn @ wn.t(), sum_error(gn, wn, gy.shape[1]))
    grads = [p.grad.clone() for p in model.parameters()]
    assert all(bool(torch.isfinite(g).all()) for g in grads)
    model.zero_grad()
    F.cross_entropy(model(tokens).flatten(0, 1).float(), tokens.flatten()).backward()
    for (name, p), g in zip(model.named_parameters(), grads):
        assert name == "tok_embeddings.weight" or torch.equal(p.grad, g), name     # (an embedding's gradient is added up by atomics)


def test_generation_step_in_a_graph():
    """Residual norm, packed projections, rotary positions, packed output: one captured step for several sequences, replayed with new
    tokens and positions and with eager work in between, equals the eager step."""
    from lingua_amd import mxfp4, norm, rope
    B, dim, H, D = 5, 256, 4, 64
    wq, wo = (mxfp4.pack(seeded_bf16((n, k), std=0.05, seed=n).cuda()) for n, k in ((2 * H * D, dim), (dim, H * D)))
    gain = seeded_bf16((dim,), seed=7).cuda()
    cos, sin = (t.cuda() for t in rope.rotary_tables(D, 10000, scaling="linear", factor=4))
    x, res, pos = seeded_bf16((B, dim), seed=8).cuda(), seeded_bf16((B, dim), seed=9).cuda(), torch.arange(B, device="cuda")[:, None]

    def step():
        h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
        qk = mxfp4.linear_packed(y, *wq).view(B, 1, 2 * H, D)
        q, k = rope.rotary(qk[:, :, :H], qk[:, :, H:], cos, sin, positions=pos, layout="half")
        return h, k, mxfp4.linear_packed(q.reshape(B, H * D), *wo)

    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(3):
            x.copy_(seeded_bf16((B, dim), seed=20 + i))
            pos.add_(997)
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_backward_in_a_graph():
    """A training step of the three operators captured whole, leaves of its own: replays equal the eager step."""
    from lingua_amd import mxfp4, norm, rope
    B, S, H, D = 2, 24, 4, 32
    make = lambda: [seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((B * S, H * D), (B * S, H * D), (H * D,), (H * D, H * D)))]  # noqa: E731
    cos, sin = (t.cuda() for t in rope.rotary_tables(D, S))
    gy = seeded_bf16((B, S, H, D), std=0.01, seed=9).cuda()

    def step(x, res, gain, w):
        h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
        q = mxfp4.mxfp4_linear(y, w).view(B, S, H, D)
        q, _ = rope.rotary(q, h.view(B, S, H, D), cos, sin)
        return torch.autograd.grad(q, (x, res, gain, w), gy)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    captured = make()
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(*captured)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*captured)
    for i in range(3):
        with torch.no_grad():
            captured[0].copy_(seeded_bf16((B * S, H * D), seed=30 + i))
        eager = make()
        with torch.no_grad():
            eager[0].copy_(captured[0])
        want = step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def calls(x, w, gain, cos, sin):
    """Each operator's differentiable call on the leaves x [8,64], w [64,64] and gain [64]."""
    from lingua_amd import mxfp4, norm, rope
    return {"add_rmsnorm": lambda: norm.add_rmsnorm(x, x.detach(), gain, 1e-5)[1],
            "rotary": lambda: rope.rotary(x.view(1, 8, 2, 32), x.view(1, 8, 2, 32).detach(), cos, sin)[0],
            "mxfp4_linear": lambda: mxfp4.mxfp4_linear(x, w)}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["add_rmsnorm", "mxfp4_linear"])
def test_capture_is_refused_while_a_graph_of_the_leaves_lives(name, native, monkeypatch):
    from lingua_amd import float8, rope
    if not native:
        monkeypatch.setattr(float8, "_plain_call", lambda: False)
    x, w, gain = (seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (64, 64), (64,))))
    call = calls(x, w, gain, *(t.cuda() for t in rope.rotary_tables(32, 8)))[name]
    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="same leaf"):
            call()
        with torch.no_grad():
            out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.detach())


def test_operands_do_not_share_a_gradient():
    """Both operands of the residual sum have the same gradient, each in memory of its own."""
    from lingua_amd import norm
    x, res, gain = (seeded_bf16(s, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (8, 64), (64,))))
    for _ in range(2):
        h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
        (h.sum() + y.sum()).backward()
        assert x.grad.data_ptr() != res.grad.data_ptr() and torch.equal(x.grad, res.grad)


@pytest.mark.parametrize("name", ["add_rmsnorm", "rotary", "mxfp4_linear"])
def test_compiled_calls_equal_eager_ones(name):
    """A compiler's tracer does not see into the calls: they stay whole, and so do their gradients."""
    from lingua_amd import rope
    leaves = [seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (64, 64), (64,)))]
    tables = [t.cuda() for t in rope.rotary_tables(32, 8)]

    def run(x, w, gain):
        return calls(x, w, gain, *tables)[name]() * 2.0

    torch._dynamo.reset()
    want, got = run(*leaves), torch.compile(run, backend="eager")(*leaves)
    torch._dynamo.reset()
    gy = seeded_bf16(tuple(want.shape), std=0.01, seed=5).cuda()
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, gy, allow_unused=True), torch.autograd.grad(want, leaves, gy, allow_unused=True)):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_threads_at_once():
    """Four threads, each on a stream of its own, through every operator forward and backward: the results of one after the other."""
    import threading
    from lingua_amd import mxfp4, norm, rope
    cos, sin = (t.cuda() for t in rope.rotary_tables(32, 16))

    def operands(i):
        leaves = [seeded_bf16(s, std=0.1, seed=10 * i + j).cuda().requires_grad_() for j, s in enumerate(((16, 128), (16, 128), (128,), (128, 128)))]
        return leaves, seeded_bf16((1, 16, 4, 32), std=0.01, seed=i).cuda(), mxfp4.pack(leaves[3])

    def step(leaves, gy, packed):
        x, res, gain, w = leaves
        h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
        q, _ = rope.rotary(mxfp4.mxfp4_linear(y, w).view(1, 16, 4, 32), h.view(1, 16, 4, 32), cos, sin)
        return (q.detach(), mxfp4.linear_packed(y, *packed)) + torch.autograd.grad(q, leaves, gy)

    sets = [operands(i) for i in range(4)]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i] = step(*sets[i])
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(u, v) for u, v in zip(a, b))


def twice(name, x, w, gain, tables):
    """An operator's output on x [8,64] and the leaves whose gradients a further pass may run into."""
    from lingua_amd import mxfp4, norm, rope
    if name == "add_rmsnorm":
        return norm.add_rmsnorm(x, x.detach(), gain, 1e-5)[1], (x, gain)
    if name == "rotary":
        return rope.rotary(x.view(1, 8, 2, 32), x.view(1, 8, 2, 32), *tables)[0].view(8, 64), (x,)
    return mxfp4.mxfp4_linear(x, w, gain), (x, w, gain)


@pytest.mark.parametrize("name", ["add_rmsnorm", "rotary", "mxfp4_linear"])
def test_second_derivatives_are_refused(name, host):
    """A gradient that was itself made for differentiation has the bits of an ordinary one, and whoever asks for its derivative gets an
    error, not the derivative of everything but this operator."""
    from lingua_amd import rope
    leaves = [seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (64, 64), (64,)))]
    tables = [t.cuda() for t in rope.rotary_tables(32, 8)]
    y, of = twice(name, *leaves, tables)
    ordinary = torch.autograd.grad(y.float().square().sum(), of)
    for i, leaf in enumerate(of):
        y, _ = twice(name, *leaves, tables)
        loss = y.float().square().sum()
        grads = torch.autograd.grad(loss, of, create_graph=True)
        assert all(torch.equal(g, o) for g, o in zip(grads, ordinary))
        with pytest.raises(RuntimeError, match=f"{name} is not differentiable twice"):
            (loss + grads[i].float().square().sum()).backward()
        # the same where only this leaf's gradient was asked for
        y, _ = twice(name, *leaves, tables)
        loss = y.float().square().sum()
        g, = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match=f"{name} is not differentiable twice"):
            (loss + g.float().square().sum()).backward()
    # a pass that does not run into them goes through
    y, _ = twice(name, *leaves, tables)
    loss = y.float().square().sum()
    torch.autograd.grad(loss, of, create_graph=True)
    for leaf in leaves:
        leaf.grad = None
    loss.backward()
    assert all(torch.equal(leaf.grad, o) for leaf, o in zip(of, ordinary))


def test_second_derivatives_of_a_linear_loss(host):
    """The gradient that arrives is a constant: what an operator makes of it varies where the operator is not linear in its inputs, and
    only there."""
    from lingua_amd import mxfp4, norm, rope
    x, w, gain = (seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (64, 64), (64,))))
    tables = [t.cuda() for t in rope.rotary_tables(32, 8)]

    def grads(y, of):
        return torch.autograd.grad(y, of, torch.ones_like(y), create_graph=True)

    for g in grads(norm.add_rmsnorm(x, x.detach(), gain, 1e-5)[1], (x, gain)) + grads(mxfp4.mxfp4_linear(x, w), (x, w)):
        with pytest.raises(RuntimeError, match="is not differentiable twice"):
            g.float().sum().backward()
    for y, of in ((mxfp4.mxfp4_linear(x, w.detach(), gain), (x, gain)), (mxfp4.mxfp4_linear(x.detach(), w), (w,)),
                  (rope.rotary(x.view(1, 8, 2, 32), x.view(1, 8, 2, 32).detach(), *tables)[0], (x,)),
                  (norm.add_rmsnorm(x.detach(), x.detach(), gain, 1e-5)[1], (gain,))):
        assert not any(g.requires_grad for g in grads(y, of))
    # the sum alone passes its gradient through, and the derivative of that
    h, _ = norm.add_rmsnorm(x, x.detach(), gain, 1e-5)
    scale = torch.tensor(3.0, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((h * scale).sum(), x, create_graph=True)
    g.sum().backward()
    assert float(scale.grad) == x.numel()


@pytest.mark.parametrize("kind", ["mxfp4", "fp8"])
def test_captured_linears_share_no_kept_weight(kind, monkeypatch):
    """With copies of the weights kept between calls: a warm-up and two captures on one stream.  A weight that has changed since, the second
    graph replayed without the first, and an eager call on that stream give what a call without kept copies gives."""
    import lingua_amd
    from lingua_amd import Fp8Linear, mxfp4
    monkeypatch.setattr(lingua_amd.config, "cache_weight_casts", True)
    lin = (mxfp4.Mxfp4Linear if kind == "mxfp4" else Fp8Linear)(256, 128, bias=False, dtype=torch.bfloat16, device="cuda")
    xs = [seeded_bf16((m, 256), seed=m).cuda() for m in (3, 40)]
    stream, graphs, ys = torch.cuda.Stream(), [torch.cuda.CUDAGraph() for _ in xs], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(stream):
            for x in xs:
                lin(x)
        torch.cuda.synchronize()
        for x, graph in zip(xs, graphs):
            with torch.cuda.graph(graph, stream=stream):
                ys.append(lin(x))
        with torch.cuda.stream(stream):
            eager = lin(xs[1])
        lin.weight.mul_(-2.0)
        torch.cuda.synchronize()
        lingua_amd.clear_cast_memos()
        want = [lin(x) for x in xs]
        assert torch.equal(eager * -2.0, want[1])
        for i in (1, 1, 0):
            ys[i].zero_()
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(ys[i], want[i])
    lingua_amd.clear_cast_memos()


def test_column_amaxes_elsewhere_are_refused():
    """A kernel writes (or reads) them through their address: on the host it would be no address of the GPU's."""
    from lingua_amd import ops
    x, w, col = seeded_bf16((16, 64), seed=1).cuda(), seeded_bf16((64,), seed=2).cuda(), torch.zeros(64)
    for call in (lambda c: ops.add_rmsnorm_cast_rowwise(x, x, w, 1e-5, col_amax=c), lambda c: ops.rmsnorm_cast_rowwise(x, w, 1e-5, col_amax=c),
                 lambda c: ops.cast_rowwise(x, col_amax=c), lambda c: ops.cast_colwise_transposed(x, c), lambda c: ops.swiglu_cast_rowwise(x, x, col_amax=c),
                 lambda c: ops.swiglu_bwd_cast_rowwise(x, x, x, c, c), lambda c: ops.swiglu_bwd_cast_transposed(x, x, x, c, c, c)):
        call(col.cuda())
        with pytest.raises(RuntimeError, match="same device"):
            call(col)


@pytest.mark.parametrize("shape", [(24, 64), (2, 12, 64)])
def test_outputs_may_be_written_in_place(shape, host):
    """As any operator's: the norm and what it is multiplied by in place have the gradients of the product, and a sum that was written
    over before the backward pass that needs it is an error."""
    from lingua_amd import norm
    x, res, gain = (seeded_bf16(s, seed=i).cuda().requires_grad_() for i, s in enumerate((shape, shape, (64,))))
    h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
    want = torch.autograd.grad((y * 2.0).sum() + h.sum(), (x, res, gain))
    h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
    y.mul_(2.0)
    for got, w in zip(torch.autograd.grad(y.sum() + h.sum(), (x, res, gain)), want):
        assert torch.equal(got, w)
    h, y = norm.add_rmsnorm(x, res, gain, 1e-5)
    h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("name", ["add_rmsnorm", "rotary"])
def test_kept_operands_in_other_layouts(name, host):
    """Hooks on saved tensors hand every second operand back with its elements apart: the gradients are the same."""
    from lingua_amd import rope
    leaves = [seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((8, 64), (64, 64), (64,)))]
    tables = [t.cuda() for t in rope.rotary_tables(32, 8)]

    def run():
        y, of = twice(name, *leaves, tables)
        return lambda: torch.autograd.grad(y, of, gy)

    def apart(t):
        return torch.stack((t, torch.full_like(t, 7.0)), -1)[..., 0]

    gy = seeded_bf16((8, 64), std=0.01, seed=5).cuda()
    want = run()()
    for parity in (0, 1):
        calls_made = []

        def pack(t):
            calls_made.append(t)
            return apart(t) if len(calls_made) % 2 == parity else t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            later = run()
        assert calls_made
        for got, w in zip(later(), want):
            assert torch.equal(got, w)


class Gate(torch.autograd.Function):
    """silu, whose backward takes the same steps in a pass that is itself differentiated (PyTorch's rounds more often there)."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return F.silu(x)

    @staticmethod
    def backward(ctx, g):
        with torch.no_grad():
            return torch.ops.aten.silu_backward(g, ctx.saved_tensors[0])


def test_a_model_whose_gradients_are_made_for_differentiation(monkeypatch):
    """The refusal waits until somebody differentiates: a pass with create_graph through every operator and the fp8 ones beside them has the
    bits of an ordinary one."""
    model = model_of(True)
    for layer in model.layers:
        mlp = layer.feed_forward
        monkeypatch.setattr(mlp, "forward", lambda x, m=mlp: m.w2(Gate.apply(m.w1(x)) * m.w3(x)))
    tokens = torch.randint(0, 64, (2, 37), generator=torch.Generator().manual_seed(2)).cuda()
    names, of = zip(*[(n, p) for n, p in model.named_parameters() if n != "tok_embeddings.weight"])   # (that gradient is added up by atomics)

    def grads(**kwargs):
        return torch.autograd.grad(F.cross_entropy(model(tokens).flatten(0, 1).float(), tokens.flatten()), of, **kwargs)

    want = grads()
    for name, got, w in zip(names, grads(create_graph=True), want):
        assert torch.equal(got, w), name
