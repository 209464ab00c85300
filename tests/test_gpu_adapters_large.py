"""Low-rank adapters at the sizes of served banks, prompts and training steps, against 64 bits."""
import pytest
import torch

import plain_more as plain
from conftest import seeded_bf16
from plain_operators import host, within  # noqa: F401

pytestmark = pytest.mark.gpu


def normal(*shape, std=1.0, seed=0):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda", dtype=torch.bfloat16) * std


def test_backward_of_a_bank_of_thousands(host):
    """A call that the forward pass takes has a backward pass: 16384 adapters, of which a batch uses three, beside the one reading of a large
    gradient."""
    from lingua_amd import adapters, ops
    n, r, K, N, T = 16384, 8, 8, 8192, 131072
    assert ops.lowrank_outer_shrink_pays(T, r, N)
    a, b = normal(n, r, K, std=K ** -0.5, seed=1), normal(n, r, N, std=0.3, seed=2)
    used = torch.tensor([0, 7, n - 1], device="cuda")
    index = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    index[100:5100], index[70000:70040], index[T - 300:] = 0, 7, n - 1
    at = (index >= 0).nonzero()[:, 0]
    x, y, gy = normal(T, K, seed=3), normal(T, N, seed=4), normal(T, N, std=0.1, seed=5)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    out = adapters.add_lowrank(y, *leaves, index)
    gx, ga, gb = torch.autograd.grad(out, leaves, gy)
    few = torch.searchsorted(used, index[at].long())
    want, size, _, _ = plain.lowrank(y[at], x[at], a[used], b[used], few, None)
    assert within(out.detach()[at], want, size)
    wants, sizes = plain.lowrank_grads(x[at], a[used], b[used], few, None, gy[at])
    assert within(gx[at], wants[0], sizes[0]) and within(ga[used], wants[1], sizes[1]) and within(gb[used], wants[2], sizes[2])
    for g in (ga, gb):
        g[used] = 0
        assert not g.any()
    gx[at] = 0
    assert not gx.any()
