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


def requests_of(T, used, seed=0):
    """Tokens of requests one behind the other, each with an adapter of ``used`` or, a tenth of the tokens, none."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randperm(T - 1, generator=g)[:2 * len(used)].add(1).sort().values
    which = torch.tensor(used)[torch.randint(0, len(used), (2 * len(used) + 1,), generator=g)]
    which[:len(used)] = torch.tensor(used)
    index = which[torch.searchsorted(cuts, torch.arange(T), right=True)]
    index[torch.rand(T, generator=g) < 0.1] = -1
    return index.int().cuda()


def against_64_bits(T, n, r, K, N, index, train, seed=0):
    """add_lowrank of a bank of n, and with ``train`` its gradients; adapters that no token has get gradients of zero."""
    from lingua_amd import adapters
    a, b = normal(n, r, K, std=K ** -0.5, seed=seed + 1), normal(n, r, N, std=0.3, seed=seed + 2)
    scale = 0.5 + torch.rand(n, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
    x, y = normal(T, K, seed=seed + 3), normal(T, N, seed=seed + 4)
    used = index[index >= 0].unique().long()
    few = torch.where(index < 0, -1, torch.searchsorted(used, index.long()))
    with torch.no_grad():
        served = adapters.add_lowrank(y, x, a, b, index, scale)
    want, size, _, _ = plain.lowrank(y, x, a[used], b[used], few, scale[used])
    assert within(served, want, size) and torch.equal(served[index < 0], y[index < 0])
    if not train:
        return
    gy = normal(T, N, std=0.1, seed=seed + 5)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    out = adapters.add_lowrank(y, *leaves, index, scale)
    gx, ga, gb = torch.autograd.grad(out, leaves, gy)
    assert within(out.detach(), want, size)
    wants, sizes = plain.lowrank_grads(x, a[used], b[used], few, scale[used], gy)
    assert within(gx, wants[0], sizes[0]) and within(ga[used], wants[1], sizes[1]) and within(gb[used], wants[2], sizes[2])
    for g in (ga, gb):
        g[used] = 0
        assert not g.any()


@pytest.mark.parametrize("r, K, N", [(24, 4104, 11000), (40, 4096, 8200), (64, 4096, 9224), (64, 9000, 12296), (72, 4104, 8200), (128, 4096, 11000)])
def test_prompts(r, K, N):
    """Five requests' prompts beside a wide projection: h in several parts, and workgroups of the sum that go on over an even or odd number of
    stretches of columns, the last of them beyond the last column."""
    from lingua_amd import _lib
    T, n = 2055, 12
    assert _lib.load().l8_lowrank_splits(T, n, r, K) > 1
    against_64_bits(T, n, r, K, N, requests_of(T, [1, 4, 5, 9, 11], seed=r), False, seed=r)


@pytest.mark.parametrize("r, K, N", [(24, 1032, 1160), (40, 1096, 520), (64, 1160, 1032), (96, 1032, 264), (128, 2056, 1096)])
@pytest.mark.parametrize("T", [4100, 8300])
def test_training_steps_of_high_rank(T, r, K, N, host):
    """Many tokens in tiles of 32 and of 64, waves of several steps with a remainder, factors' gradients that meet over several workgroups."""
    against_64_bits(T, 3, r, K, N, requests_of(T, [0, 2], seed=T + r), True, seed=r)


@pytest.mark.parametrize("n", [13, 256, 1024])
@pytest.mark.parametrize("T, r", [(40, 16), (100, 8), (257, 64), (1021, 16), (2055, 16), (2055, 64), (2055, 128)])
def test_large_banks_of_which_few_are_used(n, T, r, host):
    against_64_bits(T, n, r, 264, 520, requests_of(T, [0, 3, 7, n - 2, n - 1], seed=n + T), True, seed=n)


@pytest.mark.parametrize("T, n", [(66, 70), (256, 256), (300, 1000)])
def test_generation_with_an_adapter_a_token(T, n, host):
    index = torch.randperm(n, generator=torch.Generator().manual_seed(T)).repeat(2)[:T].int().cuda()
    index[5] = -1
    for r in (8, 64):
        against_64_bits(T, n, r, 520, 264, index, False, seed=T)


def test_a_scale_that_asks_for_a_gradient_is_refused(host):
    from lingua_amd import adapters
    x, a, b = normal(40, 64), normal(2, 8, 64), normal(2, 8, 64)
    index, scale = torch.zeros(40, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda", requires_grad=True)
    for i in (index, adapters.route(index, 2)):
        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="scale asks for a gradient"):
                adapters.add_lowrank(leaf, leaf, a, b, i, scale)
            with torch.no_grad():
                assert torch.equal(adapters.add_lowrank(leaf, leaf, a, b, i, scale), adapters.add_lowrank(leaf, leaf, a, b, i))
