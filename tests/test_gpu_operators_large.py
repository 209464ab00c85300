"""The residual norm, rotary positions and MXFP4 operators on operands of more than 2^31 elements: what they make of the last rows is
what they make of those rows alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TAIL = 64


def big(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 1 << 16):     # (a piece at a time: the generator's own temporaries)
        x[i:i + (1 << 16)] = torch.randn(x[i:i + (1 << 16)].shape, generator=g, device="cuda")
    return x


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_residual_norm():
    from lingua_amd import ops
    R, C = 540672, 4096
    x, res, w = big(R, C, 1), big(R, C, 2), big(1, C, 3)[0]
    assert x.numel() > 2 ** 31
    h, y, q, scale, rstd = ops.add_rmsnorm_cast_rowwise(x, res, w, 1e-5)
    for got, want in zip((h, y, q, scale, rstd), ops.add_rmsnorm_cast_rowwise(x[-TAIL:], res[-TAIL:], w, 1e-5)):
        assert same(got[-TAIL:], want)
    gx, gw = ops.add_rmsnorm_bwd(y, x, h, w, rstd)
    want, _ = ops.add_rmsnorm_bwd(y[-TAIL:], x[-TAIL:], h[-TAIL:], w, rstd[-TAIL:])
    assert same(gx[-TAIL:], want) and bool(torch.isfinite(gw).all())


def test_rotary():
    from lingua_amd import ops, rope
    S, H, D = 70016, 256, 128
    x = big(S * H, D, 1).view(1, S, H, D)
    assert x.numel() > 2 ** 31
    cos, sin = rope.rotary_tables(D, S, device="cuda")
    got, _ = ops.rotary(x, None, cos, sin)
    assert same(got[:, -TAIL:], ops.rotary(x[:, -TAIL:], None, cos[-TAIL:], sin[-TAIL:])[0])
    heads_first = x.view(1, H, S, D).transpose(1, 2)     # tokens 128 elements apart, heads 2^23 and more
    got, _ = ops.rotary(heads_first, None, cos, sin, in_halves=True)
    assert same(got[:, -TAIL:], ops.rotary(heads_first[:, -TAIL:], None, cos[-TAIL:], sin[-TAIL:], in_halves=True)[0])


def test_mxfp4_casts():
    from lingua_amd import ops
    R, C = 66048, 33024
    x = big(R, C, 1)
    assert x.numel() > 2 ** 31
    (q, s), (qt, st) = ops.cast_mxfp4(x, transposed=True)
    (wq, ws), (wqt, wst) = ops.cast_mxfp4(x[-TAIL:], transposed=True)     # a whole number of blocks of rows
    assert same(q[-TAIL:], wq) and same(s[-TAIL:], ws)
    assert same(qt[:, -TAIL // 2:], wqt) and same(st[:, -TAIL // 32:], wst)
    back = ops.mxfp4_to_bf16(q, s, C)
    assert same(back[-TAIL:], ops.mxfp4_to_bf16(wq, ws, C))


@pytest.mark.parametrize("blocks", [4, 9])
@pytest.mark.parametrize("odd", [0, 1])
def test_mxfp4_product(blocks, odd):
    """Both kernels, results stored as wide as they can be and column by column."""
    from lingua_amd import ops
    from test_gpu_mxfp4 import exact_product, operand
    M, N = 66000, 33024 + odd
    a, b = [[t.cuda() for t in operand(n, blocks, n)] for n in (M, N)]
    got = ops.gemm_mxfp4_nt(a[0], b[0], a[1], b[1])
    assert got.numel() > 2 ** 31
    for rows in (slice(0, 300), slice(M - 300, M)):
        want = exact_product([t[rows] for t in a], b).to(torch.bfloat16)
        assert torch.equal(got[rows], want)
