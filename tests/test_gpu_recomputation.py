"""Dropout and adapters under activation checkpointing, which computes a forward pass again in the backward pass: gradients of the same elements
and the same adapters, or an error where the seed and step or the requests have changed in between."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from conftest import seeded_bf16
from plain_operators import host  # noqa: F401

pytestmark = pytest.mark.gpu

NAMES = ["dropout", "dropout_add", "add_layernorm", "add_rmsnorm", "adapters"]


def make(name):
    """(a call of one tensor, what changes before its next batch)."""
    from lingua_amd import adapters, dropout, norm
    n, w = dropout.numbers(3), seeded_bf16((64,), seed=4).cuda()
    res = seeded_bf16((48, 64), seed=5).cuda()
    requests = adapters.Requests(3)
    a, b = (seeded_bf16((3, 8, 64), std=0.3, seed=6 + i).cuda() for i in range(2))
    index = torch.arange(48, device="cuda") % 4 - 1
    requests.set(index)
    drop = dropout.Drop(0.5, n, 2)
    call = {"dropout": lambda x: dropout.dropout(x, drop), "dropout_add": lambda x: dropout.dropout_add(x, res, drop),
            "add_layernorm": lambda x: norm.add_layernorm(x, res, w, w, dropout=drop)[1], "add_rmsnorm": lambda x: norm.add_rmsnorm(x, res, w, 1e-5, drop)[1],
            "adapters": lambda x: adapters.add_lowrank(res, x, a, b, requests.plan)}[name]

    def advance():
        if name == "adapters":
            requests.set(index.roll(1))
        else:
            n[1] += 1
    return (lambda x: call(x) * 2.0), advance


@pytest.mark.parametrize("name", NAMES)
def test_recomputed_passes(name, host):
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 64), std=0.1, seed=2).cuda()
    call, advance = make(name)
    want, = torch.autograd.grad(call(x), x, g)
    for reentrant in (False, True):
        x.grad = None
        checkpoint(call, x, use_reentrant=reentrant).backward(g)
        assert torch.equal(x.grad, want)


@pytest.mark.parametrize("name", NAMES)
def test_changes_before_a_recomputation_are_an_error(name, host):
    """Also of a batch whose successor has gone through both passes already."""
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 64), std=0.1, seed=2).cuda()
    call, advance = make(name)
    first = checkpoint(call, x, use_reentrant=False)
    advance()
    second = checkpoint(call, x, use_reentrant=False)
    want, = torch.autograd.grad(call(x), x, g)
    got, = torch.autograd.grad(second, x, g)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation between the forward pass and its recomputation"):
        first.backward(g)


@pytest.mark.parametrize("name", NAMES)
def test_copies_kept_on_the_host(name, host):
    """Saved tensors that a hook copies are those of the forward pass, whatever changes afterwards."""
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 64), std=0.1, seed=2).cuda()
    call, advance = make(name)
    want, = torch.autograd.grad(call(x), x, g)
    with torch.autograd.graph.save_on_cpu():
        y = call(x)
    advance()
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want)


@pytest.mark.parametrize("reentrant", [False, True])
def test_modules_of_requests(reentrant, host):
    """Of an adapted linear under either kind of checkpointing: the plain gradients, and an error where other requests, or none, were set before
    the backward pass.  (A recomputation that is stopped when all saved tensors are there again does not ask for requests that the forward pass
    did not have: its gradients are right.)"""
    from lingua_amd import adapters
    requests = adapters.Requests(3)
    lin = adapters.AdaptedLinear(torch.nn.Linear(64, 128, bias=False, dtype=torch.bfloat16, device="cuda"), requests, 8)
    torch.nn.init.normal_(lin.b, std=0.3)
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 128), std=0.1, seed=2).cuda()
    index = torch.arange(48, device="cuda") % 4 - 1
    call = lambda t: lin(t) * 2.0  # noqa: E731
    for i in (index, index.roll(1), None):
        requests.set(i)
        want = torch.autograd.grad(call(x), x, g)[0]
        x.grad = None
        checkpoint(call, x, use_reentrant=reentrant).backward(g)
        assert torch.equal(x.grad, want)
    for first, second in ((index, index.roll(1)), (index, None), (None, index), (index, index[:8])):
        requests.set(first)
        want = torch.autograd.grad(call(x), x, g)[0]
        y = checkpoint(call, x, use_reentrant=reentrant)
        requests.set(second)
        if first is None and not reentrant:
            assert torch.equal(torch.autograd.grad(y, x, g)[0], want)
            continue
        with pytest.raises(RuntimeError, match="Requests: set between a forward pass and its recomputation"):
            y.backward(g)


class Twice(torch.nn.Module):
    def __init__(self, both):
        super().__init__()
        self.drop, self.both = torch.nn.Dropout(0.5), both

    def forward(self, x, reentrant=None):
        def part(t):
            t = self.drop(t)
            return self.drop(t * 1.5) if self.both else t * 1.5
        return part(x) if reentrant is None else checkpoint(part, x, use_reentrant=reentrant)


def test_a_module_that_is_called_twice(host):
    """Its two calls drop independently, forward and backward alike, and the pass repeated drops the same again."""
    from lingua_amd import dropout
    model = dropout.convert_dropouts(Twice(True), dropout.numbers(3))
    x = torch.ones(1 << 20, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = model(x)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    stays = float((y != 0).double().mean())    # of two independent draws of a half: a quarter
    assert abs(stays - 0.25) < 5 * (0.25 * 0.75 / x.numel()) ** 0.5
    assert torch.equal(gx, y.detach()) and torch.equal(model(x), y)


@pytest.mark.parametrize("reentrant", [False, True])
def test_modules_of_dropout(reentrant, host):
    """Under either kind of checkpointing: the plain gradients of a module that is called once, an error for one that is called twice and for a
    step that was advanced before the backward pass."""
    from lingua_amd import dropout
    n = dropout.numbers(3)
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 64), std=0.1, seed=2).cuda()
    model = dropout.convert_dropouts(Twice(False), n)
    for _ in range(2):
        want, = torch.autograd.grad(model(x), x, g)
        x.grad = None
        model(x, reentrant).backward(g)
        assert torch.equal(x.grad, want)
        n[1] += 1
    y = model(x, reentrant)
    n[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation between the forward pass and its recomputation"):
        y.backward(g)
    y = model(x, reentrant)
    model.drop.numbers = n.clone()
    with pytest.raises(RuntimeError, match="exchanged"):
        y.backward(g)
    model = dropout.convert_dropouts(Twice(True), n)
    y = model(x, reentrant)
    model.eval()
    model(x)
    model.train()
    with pytest.raises(RuntimeError, match="several times in a forward pass"):
        y.backward(g)


def test_compiled_model():
    from lingua_amd import dropout
    n = dropout.numbers(3)
    x, g = seeded_bf16((48, 64), seed=1).cuda().requires_grad_(), seeded_bf16((48, 64), std=0.1, seed=2).cuda()
    model = dropout.convert_dropouts(Twice(True), n)
    torch._dynamo.reset()
    compiled = torch.compile(model, backend="eager")
    for _ in range(3):
        want, got = model(x), compiled(x)
        assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, x, g)[0], torch.autograd.grad(want, x, g)[0])
        n[1] += 1
    torch._dynamo.reset()
