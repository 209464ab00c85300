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
