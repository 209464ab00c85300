"""MXFP4 casts, products and linears against the format's definition in 64 bits.

Casts are exact: codes and scales must be equal.  Products of codes and scales are exact in fp32 for the integer-like operands used
where equality is asked for; elsewhere a sum over K is off by at most K * 2^-24 of the sum of magnitudes, and bf16 by half a step."""
import pytest
import torch

import plain_operators as plain
from conftest import seeded_bf16
from plain_operators import host  # noqa: F401

pytestmark = pytest.mark.gpu


def spread(R, C, seed):
    """bf16 of every exponent: a level for each block, values down to 2^-9 of it, every mantissa, both signs."""
    g = torch.Generator().manual_seed(seed)
    level = torch.randint(0, 255, (R, (C + 31) // 32), generator=g).repeat_interleave(32, 1)[:, :C]
    exponent = (level - torch.randint(0, 10, (R, C), generator=g)).clamp(min=0)
    bits = torch.randint(0, 2, (R, C), generator=g) << 15 | exponent << 7 | torch.randint(0, 128, (R, C), generator=g)
    return (bits - (bits >= 1 << 15).long() * (1 << 16)).to(torch.int16).view(torch.bfloat16)


def check_cast(pair, x):
    code, byte = plain.mx_quantise(x)
    assert pair[0].dtype == torch.float4_e2m1fn_x2 and pair[1].dtype == torch.float8_e8m0fnu
    assert torch.equal(pair[1].view(torch.uint8).cpu(), byte.cpu())
    assert torch.equal(pair[0].view(torch.uint8).cpu(), plain.mx_pack(code).cpu())


@pytest.mark.parametrize("shape", [(1, 8), (1, 32), (3, 24), (33, 40), (31, 64), (256, 128), (257, 136), (300, 2064), (70, 4096), (2048, 1024)])
def test_casts_are_the_formats(shape):
    from lingua_amd import ops
    x = spread(*shape, seed=shape[0] + shape[1])
    rows, cols = ops.cast_mxfp4(x.cuda(), rowwise=True, transposed=True)
    check_cast(rows, x)
    check_cast(cols, x.t().contiguous())
    alone, none = ops.cast_mxfp4(x.cuda())
    assert none is None
    check_cast(alone, x)
    none, alone = ops.cast_mxfp4(x.cuda(), rowwise=False, transposed=True, on_lines=True)
    assert none is None
    check_cast(alone, x.t().contiguous())


# Shapes that give every unit a tile of 256 x 128: a last band of rows and last columns that are not full, 79, 130 and 2188 bands
@pytest.mark.parametrize("shape", [(2500, 4104), (4129, 2056), (70001, 64)])
def test_large_casts_are_the_formats(shape):
    from lingua_amd import ops
    R, C = shape
    assert (R + 255) // 256 * ((C + 127) // 128) >= torch.cuda.get_device_properties(0).multi_processor_count
    x = spread(R, C, seed=R + C)
    x[40:104, :] = 0.0
    x[41:104:2, :] = -0.0
    x[200:264, 8:16] = torch.tensor(2.0 ** -133).to(torch.bfloat16)
    x[300, :], x[301, 5] = 2.0 ** -133, 0.0
    x[777, 33], x[R - 1, C - 1], x[1500, 2], x[R - 40, 40] = float("nan"), float("inf"), -float("inf"), float("nan")
    x = x.cuda()
    rows, cols = ops.cast_mxfp4(x, rowwise=True, transposed=True)
    check_cast(rows, x)
    check_cast(cols, x.t().contiguous())
    none, alone = ops.cast_mxfp4(x, rowwise=False, transposed=True, on_lines=True)
    assert none is None
    check_cast(alone, x.t().contiguous())


def test_cast_of_blocks_that_are_zero_or_not_finite_and_of_rows_apart():
    from lingua_amd import ops
    wide = seeded_bf16((70, 256), seed=3)
    wide[2, :] = 0.0
    wide[3, :] = -0.0
    wide[5, 40], wide[6, 100], wide[7, 101] = float("nan"), float("inf"), -float("inf")
    wide[9, :] = torch.tensor(2.0 ** -133).to(torch.bfloat16)     # the smallest subnormal
    wide[10, ::2] = torch.finfo(torch.bfloat16).max
    x = wide[:, 32:232]
    rows, cols = ops.cast_mxfp4(wide.cuda()[:, 32:232], rowwise=True, transposed=True)
    check_cast(rows, x)
    check_cast(cols, x.t().contiguous())
    back = ops.mxfp4_to_bf16(*rows, 200)
    want = plain.mx_values(*plain.mx_quantise(x))[:, :200]
    assert torch.equal(torch.isnan(back.cpu()), torch.isnan(want)) and bool(torch.isnan(want).any())
    assert torch.equal(back.cpu().double().nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("R,C", [(0, 32), (4, 0), (0, 0)])
def test_empty_casts(R, C):
    from lingua_amd import ops
    rows, cols = ops.cast_mxfp4(torch.empty(R, C, dtype=torch.bfloat16, device="cuda"), transposed=True)
    assert rows[0].shape == (R, (C + 31) // 32 * 16) and cols[0].shape == (C, (R + 31) // 32 * 16)
    assert ops.mxfp4_to_bf16(*rows, C).shape == (R, C)


@pytest.mark.parametrize("R,blocks,cols", [(1, 1, 1), (5, 3, 70), (40, 7, 224), (3, 65, 2065)])
def test_back_to_bf16_of_any_bytes(R, blocks, cols):
    """Every code under every scale, dense rows of scales of odd length, as uint8; exact, with bf16's own overflow."""
    from lingua_amd import ops
    g = torch.Generator().manual_seed(blocks)
    q = torch.randint(0, 256, (R, blocks * 16), generator=g, dtype=torch.uint8)
    s = torch.randint(0, 256, (R, blocks), generator=g, dtype=torch.uint8)
    s.view(-1)[0] = 255
    s.view(-1)[-1] = 254 if s.numel() > 1 else 255
    back = ops.mxfp4_to_bf16(q.cuda(), s.cuda(), cols).cpu()
    want = plain.mx_values(plain.mx_unpack(q), s)[:, :cols].to(torch.bfloat16)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("shapes", [((333, 264), (64, 1040)), ((2500, 4096), (4100, 2056)), ((5, 8), (70000, 64)), ((0, 64), (32, 64))])
@pytest.mark.parametrize("wanted", [("rows columns", "rows columns"), ("columns", "columns"), ("rows", "rows columns"), ("rows", "rows")])
def test_two_casts_in_one_call(shapes, wanted):
    """The bytes of single casts, whichever copies are wanted; what lies between rows stays."""
    import struct
    from lingua_amd import _lib, ops
    pack, kept, pairs = [], [], []
    for i, ((R, C), want) in enumerate(zip(shapes, wanted)):
        x = seeded_bf16((R, C), seed=R + C).cuda()
        copies = []
        for name, (rows, cols) in (("rows", (R, C)), ("columns", (C, R))):
            blocks = (cols + 31) // 32
            q = torch.full((rows, blocks * 16 + 16), 0xA5, dtype=torch.uint8, device="cuda")
            s = torch.full((rows, (blocks + 7) // 4 * 4), 0xA5, dtype=torch.uint8, device="cuda")
            copies.append((q, s, blocks) if name in want else None)
        pack += [x.data_ptr(), R, C, C]
        for c in copies:
            pack += [0, 0, 0, 0] if c is None else [c[0].data_ptr(), c[0].stride(0), c[1].data_ptr(), c[1].stride(0)]
        kept.append(x)
        pairs.append(copies)
    _lib.check(_lib.load().l8_cast_mxfp4_two(struct.pack("24q", *pack), torch.cuda.current_stream().cuda_stream), "l8_cast_mxfp4_two")
    for x, copies in zip(kept, pairs):
        for c, single in zip(copies, ops.cast_mxfp4(x, transposed=True)):
            if c is not None:
                q, s, blocks = c
                assert torch.equal(q[:, :blocks * 16], single[0].view(torch.uint8)) and torch.equal(s[:, :blocks], single[1].view(torch.uint8))
                assert bool((q[:, blocks * 16:] == 0xA5).all()) and bool((s[:, blocks:] == 0xA5).all())


def operand(rows, blocks, seed, low=126, high=129):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (rows, blocks * 16), generator=g, dtype=torch.uint8),
            torch.randint(low, high, (rows, blocks), generator=g, dtype=torch.uint8))


def exact_product(a, b):
    return plain.mx_values(plain.mx_unpack(a[0]), a[1]) @ plain.mx_values(plain.mx_unpack(b[0]), b[1]).t()


# (rows of A, of B, blocks): each kernel -- few tiles to many --, partial tiles in both directions, K from one block on, one block to
# either side of a stage (8) and of a window of scales (16), columns that are no multiple of what a lane stores
PRODUCTS = [(1, 1, 1), (1, 16, 2), (5, 7, 3), (16, 16, 4), (17, 33, 7), (64, 64, 8), (65, 63, 9), (100, 130, 15), (130, 100, 16), (48, 272, 17), (200, 200, 33),
            (1021, 2064, 5), (2000, 1500, 24), (1100, 2056, 43), (4100, 2051, 9), (4096, 2304, 40), (3000, 4099, 17)]


@pytest.mark.parametrize("M,N,blocks", PRODUCTS)
@pytest.mark.parametrize("with_bias", [False, True])
def test_products_are_exact(M, N, blocks, with_bias):
    """Codes are multiples of 1/2 up to 6, scales 1/2, 1, 2: every partial sum is a multiple of 1/16 below 2^18 and exact in fp32."""
    from lingua_amd import ops
    a, b = operand(M, blocks, M + N), operand(N, blocks, N + blocks)
    bias = torch.randint(-64, 64, (N,), generator=torch.Generator().manual_seed(N)).to(torch.bfloat16) if with_bias else None
    got = ops.gemm_mxfp4_nt(*(t.cuda() for t in (a[0], b[0], a[1], b[1])), None if bias is None else bias.cuda())
    want = exact_product([t.cuda() for t in a], [t.cuda() for t in b])
    if bias is not None:
        want = want + bias.cuda().double()
    assert torch.equal(got, want.to(torch.bfloat16))


@pytest.mark.parametrize("M,N,blocks", [(3, 40, 11), (300, 520, 21), (2100, 2200, 13)])
def test_product_reads_no_scale_behind_a_row(M, N, blocks):
    """Rows of codes and scales further apart than they are long, with NaN scales and full codes in between; results into columns of a
    wider matrix, whose other columns stay."""
    from lingua_amd import ops
    a, b = operand(M, blocks, 1), operand(N, blocks, 2)

    def apart(q, s):
        wq = torch.full((q.shape[0], q.shape[1] + 48), 0x77, dtype=torch.uint8, device="cuda")
        ws = torch.full((s.shape[0], s.shape[1] + 32 + -s.shape[1] % 16), 255, dtype=torch.uint8, device="cuda")
        wq[:, :q.shape[1]], ws[:, :s.shape[1]] = q.cuda(), s.cuda()
        return wq[:, :q.shape[1]], ws[:, :s.shape[1]]

    (qa, sa), (qb, sb) = apart(*a), apart(*b)
    wide = torch.full((M, N + 13), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 5:5 + N]
    version = wide._version
    assert ops.gemm_mxfp4_nt(qa, qb, sa, sb, out=out) is out and wide._version > version
    assert torch.equal(out, exact_product([t.cuda() for t in a], [t.cuda() for t in b]).to(torch.bfloat16))
    assert bool((wide[:, :5] == 3).all()) and bool((wide[:, 5 + N:] == 3).all())


@pytest.mark.parametrize("M,N,blocks", [(20, 48, 6), (300, 300, 20), (2100, 2200, 18)])
def test_product_with_extreme_and_nan_scales(M, N, blocks):
    from lingua_amd import ops
    a, b = operand(M, blocks, 5), operand(N, blocks, 6)
    a[1][1, :], b[1][:, :] = 0, 127       # the smallest scale: products of 2^-129 and more, bf16 subnormals among the sums
    a[1][2, :] = 250                      # 2^123: some sums stay within fp32, others do not
    a[1][4, blocks - 1] = 255
    b[1][7, 0] = 255
    got = ops.gemm_mxfp4_nt(*(t.cuda() for t in (a[0], b[0], a[1], b[1]))).cpu()
    want = exact_product([t.cuda() for t in a], [t.cuda() for t in b]).cpu()
    nan = torch.isnan(want)
    assert bool(nan[4].all()) and bool(nan[:, 7].all()) and int(nan.sum()) == M + N - 1
    # a sum in fp32 may leave its range on the way only where the magnitudes add up to 2^128 or more: there nothing is claimed
    magnitudes = exact_product([(a[0] & 0x77).cuda(), a[1].cuda()], [(b[0] & 0x77).cuda(), b[1].cuda()]).cpu()
    fits = (magnitudes < 2.0 ** 128) | nan
    assert bool(fits[[r for r in range(M) if r != 2]].all())
    assert torch.equal(torch.isnan(got)[fits], nan[fits])
    fits[1] = False
    assert torch.equal(got[fits].nan_to_num(1.0), want.to(torch.bfloat16)[fits].nan_to_num(1.0))
    # sums of the row of smallest scales are below fp32's normal numbers, where the matrix cores may flush: off by 2^-126 at most
    assert bool(((got[1].double() - want[1]).abs().nan_to_num(0.0) <= 2.0 ** -126).all())


# Tiles of 128 x 64 and of 64 x 128 (few rows, many columns), partial in both directions, an even and an odd number of columns
@pytest.mark.parametrize("M,N,blocks", [(290, 4104, 11), (257, 4163, 24), (130, 9000, 1), (190, 9990, 6), (129, 11001, 9), (192, 9984, 32)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_products_on_oblong_tiles_are_exact(M, N, blocks, with_bias):
    test_products_are_exact(M, N, blocks, with_bias)


# The kernel of the large products: partial tiles in both directions, one tile to a workgroup and several, K from its shortest on, an odd
# and an even number of stages (8 blocks), one block to either side of a window of scales (16)
@pytest.mark.parametrize("M,N,blocks", [(4100, 2304, 9), (2500, 4104, 15), (4096, 2312, 16), (33100, 264, 17), (264, 33104, 24), (8200, 2304, 25), (8200, 2304, 33)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_large_products_are_exact(M, N, blocks, with_bias):
    """As above, with what lies behind the rows of scales and beside the result's columns guarded, and a NaN in a scale at either end."""
    from lingua_amd import ops
    a, b = operand(M, blocks, M + N), operand(N, blocks, N + blocks)
    a[1][M - 1, blocks - 1], b[1][3, 0] = 255, 255
    bias = torch.randint(-64, 64, (N,), generator=torch.Generator().manual_seed(N)).to(torch.bfloat16).cuda() if with_bias else None

    def apart(s):
        wide = torch.full((s.shape[0], s.shape[1] + 32 + -s.shape[1] % 16), 255, dtype=torch.uint8, device="cuda")
        wide[:, :s.shape[1]] = s.cuda()
        return wide[:, :s.shape[1]]

    wide = torch.full((M, N + 16), 3.0, dtype=torch.bfloat16, device="cuda")
    got = ops.gemm_mxfp4_nt(a[0].cuda(), b[0].cuda(), apart(a[1]), apart(b[1]), bias, out=wide[:, 8:8 + N])
    a[1][M - 1, blocks - 1], b[1][3, 0] = 127, 127
    want = exact_product([t.cuda() for t in a], [t.cuda() for t in b])
    if bias is not None:
        want = want + bias.double()
    want[M - 1, :] = float("nan")
    want[:, 3] = float("nan")
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(1.0), want.to(torch.bfloat16).nan_to_num(1.0))
    assert bool((wide[:, :8] == 3).all()) and bool((wide[:, 8 + N:] == 3).all())


def test_product_over_nothing_is_zero():
    from lingua_amd import ops
    q, s = torch.empty(5, 0, dtype=torch.uint8, device="cuda"), torch.empty(5, 0, dtype=torch.uint8, device="cuda")
    bias = torch.arange(5, device="cuda").to(torch.bfloat16)
    assert torch.equal(ops.gemm_mxfp4_nt(q, q, s, s), torch.zeros(5, 5, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(ops.gemm_mxfp4_nt(q, q, s, s, bias), bias.expand(5, 5))
    assert ops.gemm_mxfp4_nt(q[:0], q, s[:0], s).shape == (0, 5)


def sum_error(a, b, K):
    """What a sum of K fp32 products may be off by, whatever its order."""
    return (a.abs() @ b.abs().t()) * (K * plain.FP32)


@pytest.mark.parametrize("M,K,N", [(1, 16, 16), (1, 4096, 64), (7, 48, 32), (16, 2048, 272), (17, 2064, 48), (33, 1040, 304), (64, 4096, 96), (65, 528, 528), (333, 2048, 1040),
                                   (12, 2048, 48), (3, 11008, 64), (7, 16, 9872), (16, 48, 9872), (20, 96, 9872), (64, 528, 9872), (40, 64, 4944)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear_with_a_packed_weight(M, K, N, with_bias):
    from lingua_amd import mxfp4
    x, w = seeded_bf16((M, K), seed=M + K), seeded_bf16((N, K), std=0.02, seed=N)
    if M > 2:
        x[1] = 0.0
    bias = seeded_bf16((N,), seed=4) if with_bias else None
    code, byte = plain.mx_quantise(w)
    cb = None if bias is None else bias.cuda()
    got = mxfp4.linear_packed(x.cuda(), plain.mx_pack(code).cuda(), byte.cuda(), cb)
    xr, wr = plain.mx_rounded(x), plain.mx_rounded(w)
    want = xr @ wr.t() + (0 if bias is None else bias.double())
    assert plain.within(got, want, sum_error(xr, wr, K) + want.abs() * plain.FP32)
    assert torch.equal(got, mxfp4.linear_packed(x.cuda(), *mxfp4.pack(w.cuda()), cb))
    three = mxfp4.linear_packed(x.cuda().reshape(1, M, K), *mxfp4.pack(w.cuda()), cb)
    assert three.shape == (1, M, N) and torch.equal(three[0], got)


# Each form of the few-token kernel, one window of 512 columns a wave and several, shares that differ and waves without any: tokens
# quantised inside (M up to 8), or before on one or two tiles of weight rows (N from 4896 on) and one, two or four of tokens
@pytest.mark.parametrize("M,K,N", [(1, 11008, 64), (2, 2048, 48), (2, 11008, 80), (4, 11008, 64), (4, 512, 9872), (5, 8208, 48), (6, 8192, 64), (8, 4096, 272), (8, 48, 64),
                                   (9, 4624, 64), (12, 11008, 48), (16, 8208, 64), (20, 4624, 48), (24, 528, 5008), (32, 11008, 4912), (32, 8208, 96), (33, 4624, 48),
                                   (48, 4624, 5008), (64, 11008, 272), (64, 11008, 4912)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_few_tokens_are_exact(M, K, N, with_bias):
    """Both operands are multiples of 1/2 up to 6 times 1/2, 1 or 2, with a 4 or a 6 in every block, so that the cast of x is x.  Products
    are multiples of 1/16 and their magnitudes add up to less than 2^20: every partial sum is exact in fp32, in any order."""
    from lingua_amd import mxfp4
    blocks = (K + 31) // 32
    (qx, sx), (qw, sw) = operand(M, blocks, M + K), operand(N, blocks, N + K)
    code = plain.mx_unpack(qx)
    code[:, ::32] = code[:, ::32] & 8 | 6 + (code[:, ::32] & 1)
    x = plain.mx_values(code, sx)[:, :K]
    w = plain.mx_values(plain.mx_unpack(qw), sw)[:, :K].cuda()
    xb = x.to(torch.bfloat16).cuda()
    assert torch.equal(xb.cpu().double(), x) and torch.equal(plain.mx_rounded(xb.cpu()), x)
    if K % 32:
        qw[:, (K - 1) // 32 * 16 + K % 32 // 2:] = 0     # (codes behind the last column are zeros)
    bias = torch.randint(-64, 64, (N,), generator=torch.Generator().manual_seed(N)).to(torch.bfloat16).cuda() if with_bias else None
    got = mxfp4.linear_packed(xb, qw.cuda(), sw.cuda(), bias)
    want = x.cuda() @ w.t()
    assert float((x.abs().cuda() @ w.abs().t()).max()) + 64 < 2.0 ** 20
    if bias is not None:
        want = want + bias.double()
    assert torch.equal(got, want.to(torch.bfloat16))


@pytest.mark.parametrize("M", [1, 3, 12, 20, 70, 300])
def test_linear_over_nothing_is_its_bias(M):
    from lingua_amd import mxfp4
    q, s = torch.empty(24, 0, dtype=torch.uint8, device="cuda"), torch.empty(24, 0, dtype=torch.uint8, device="cuda")
    x, bias = torch.empty(M, 0, dtype=torch.bfloat16, device="cuda"), torch.arange(24, device="cuda").to(torch.bfloat16)
    assert torch.equal(mxfp4.linear_packed(x, q, s, bias), bias.expand(M, 24))
    assert torch.equal(mxfp4.linear_packed(x, q, s), torch.zeros(M, 24, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("M,K,N", [(5, 2608, 40), (40, 1040, 64), (40, 528, 9888), (171, 3856, 368), (700, 1296, 2064), (4200, 528, 2304)])
def test_scales_at_any_address(M, K, N, host):
    """Rows of scales an odd number of bytes apart, from an odd address on, NaN bytes between them: the product of those on lines."""
    from lingua_amd import mxfp4
    x, w = seeded_bf16((M, K), seed=M).cuda(), seeded_bf16((N, K), std=0.02, seed=N).cuda()
    codes, scales = mxfp4.pack(w)
    blocks = scales.shape[1]
    odd = torch.full((N, blocks + 5 + blocks % 2), 255, dtype=torch.uint8, device="cuda")
    odd[:, 3:3 + blocks] = scales.view(torch.uint8)
    assert odd.stride(0) % 2 == 1
    assert torch.equal(mxfp4.linear_packed(x, codes, odd[:, 3:3 + blocks]), mxfp4.linear_packed(x, codes, scales))


def test_linear_with_a_packed_weight_and_rows_that_are_not_finite():
    from lingua_amd import mxfp4
    x, w = seeded_bf16((5, 256), seed=1), seeded_bf16((64, 256), std=0.02, seed=2)
    x[1, 33], x[3, 200] = float("nan"), float("inf")
    got = mxfp4.linear_packed(x.cuda(), *mxfp4.pack(w.cuda())).cpu()
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[3]).all()) and bool(torch.isfinite(got[[0, 2, 4]]).all())


@pytest.mark.parametrize("M,K,N", [(1, 16, 32), (9, 48, 64), (33, 272, 144), (130, 512, 528), (515, 1040, 784)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear_gradients(M, K, N, with_bias, host):
    from lingua_amd import mxfp4
    x, w, gy = seeded_bf16((M, K), seed=M), seeded_bf16((N, K), std=0.02, seed=K), seeded_bf16((M, N), std=1e-3, seed=N)
    bias = seeded_bf16((N,), seed=4) if with_bias else None
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    bd = bias.cuda().requires_grad_() if with_bias else None
    y = mxfp4.mxfp4_linear(xd, wd, bd)
    grads = torch.autograd.grad(y, [xd, wd] + ([bd] if with_bias else []), gy.cuda())
    q = plain.mx_rounded
    y64 = q(x) @ q(w).t() + (bias.double() if with_bias else 0)
    assert plain.within(y.detach(), y64, sum_error(q(x), q(w), K) + y64.abs() * plain.FP32)
    gn, wn, gt, xt = q(gy), q(w.t().contiguous()).t(), q(gy.t().contiguous()), q(x.t().contiguous())
    assert plain.within(grads[0], gn @ wn, sum_error(gn, wn.t(), N))
    assert plain.within(grads[1], gt @ xt.t(), sum_error(gt, xt, M))
    if with_bias:
        assert plain.within(grads[2], gy.double().sum(0), gy.double().abs().sum(0) * M * plain.FP32)


def test_gradients_that_nobody_asks_for_are_not_made():
    from lingua_amd import mxfp4
    big, w = torch.zeros(2048, 1024, dtype=torch.bfloat16, device="cuda"), torch.zeros(1024, 1024, dtype=torch.bfloat16, device="cuda")
    for x_learns, w_learns, held in ((True, False, w.numel()), (False, True, big.numel()), (True, True, big.numel() + w.numel()), (False, False, 0)):
        xl, wl = big.clone().requires_grad_(x_learns), w.clone().requires_grad_(w_learns)
        before = torch.cuda.memory_allocated()
        y = mxfp4.mxfp4_linear(xl, wl)
        assert torch.cuda.memory_allocated() - before <= 2 * y.numel() + held * 17 // 32 + 8192
        del y
    x, w = seeded_bf16((40, 64), seed=1).cuda(), seeded_bf16((48, 64), seed=2).cuda()
    y = mxfp4.mxfp4_linear(x.clone().requires_grad_(), w)
    y.sum().backward()                                   # a gradient of stride 0
    wl = w.clone().requires_grad_()
    y = mxfp4.mxfp4_linear(x, wl)
    y.backward(torch.ones(48, 40, dtype=torch.bfloat16, device="cuda").t())
    ones = torch.ones(48, 40, dtype=torch.bfloat16)
    want = plain.mx_rounded(ones) @ plain.mx_rounded(x.cpu().t().contiguous()).t()
    assert plain.within(wl.grad, want, want.abs() * 0 + 40 * plain.FP32 * plain.mx_rounded(x.cpu().t().contiguous()).abs().sum(1))
    empty = mxfp4.mxfp4_linear(x[:0], wl)
    wl.grad = None
    empty.sum().backward()
    assert empty.shape == (0, 48) and bool((wl.grad == 0).all())


def test_modules_and_conversion():
    import lingua_amd
    from lingua_amd import mxfp4
    model = torch.nn.ModuleDict({"layers": torch.nn.ModuleList([torch.nn.Linear(64, 96, dtype=torch.bfloat16, device="cuda")]),
                                 "output": torch.nn.Linear(96, 32, dtype=torch.bfloat16, device="cuda")})
    keys, w = list(model.state_dict()), model["layers"][0].weight
    mxfp4.convert_linears_to_mxfp4(model, r"layers\.[0-9]+$")
    lin = model["layers"][0]
    assert type(lin) is mxfp4.Mxfp4Linear and lin.weight is w and type(model["output"]) is torch.nn.Linear and list(model.state_dict()) == keys
    with pytest.raises(AssertionError):
        mxfp4.convert_linears_to_mxfp4(model, r"layers\.[0-9]+$")
    x = seeded_bf16((3, 7, 64), seed=5).cuda()
    with torch.no_grad():
        y = lin(x)
        want = lin.forward(x.requires_grad_())
        assert y.shape == (3, 7, 96) and torch.equal(y, want)
        old = lingua_amd.config.cache_weight_casts
        lingua_amd.config.cache_weight_casts = True
        try:
            assert torch.equal(lin(x), y) and torch.equal(lin(x), y)
            w.mul_(2)                                     # an optimizer step: the kept copy is not used again
            assert torch.equal(lin(x), mxfp4.linear_packed(x, *mxfp4.pack(w), lin.bias))
        finally:
            lingua_amd.config.cache_weight_casts = old
            lingua_amd.clear_cast_memos()
    with torch.inference_mode():
        assert lin(x.detach()).shape == (3, 7, 96)


@pytest.mark.parametrize("M,K,N", [(1, 1024, 256), (40, 512, 128), (300, 512, 528)])
def test_captured_linears_replay(M, K, N):
    """One graph with a serving linear and a cast, replayed with other inputs and eager work in between."""
    from lingua_amd import mxfp4, ops
    x, w = seeded_bf16((M, K), seed=1).cuda(), seeded_bf16((N, K), std=0.02, seed=2).cuda()
    packed = mxfp4.pack(w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mxfp4.linear_packed(x, *packed)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mxfp4.linear_packed(x, *packed)
        back = ops.mxfp4_to_bf16(*ops.cast_mxfp4(x)[0], K)
    for i in range(3):
        x.copy_(seeded_bf16((M, K), seed=10 + i))
        want = mxfp4.linear_packed(x, *packed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(back.cpu().double(), plain.mx_rounded(x.cpu()))


def test_two_streams_at_once():
    from lingua_amd import mxfp4
    xs = [seeded_bf16((m, 1024), seed=m).cuda() for m in (1, 700)]
    packed = mxfp4.pack(seeded_bf16((528, 1024), seed=9).cuda())
    want = [mxfp4.linear_packed(x, *packed) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(mxfp4.linear_packed(x, *packed))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


@pytest.mark.parametrize("M,K,N", [(40, 80, 48), (300, 528, 272)])
@pytest.mark.parametrize("hooks", ["clones", "host", "rows apart"])
def test_kept_copies_in_other_layouts(M, K, N, hooks, host):
    """Hooks on saved tensors hand the kept copies back in layouts of their own: the gradients are the same."""
    from lingua_amd import mxfp4

    def apart(t):
        return torch.empty_strided(t.shape, (t.shape[1] + 3, 1), dtype=torch.uint8, device=t.device).copy_(t.view(torch.uint8)).view(t.dtype)

    with_hooks = {"clones": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.contiguous()),
                  "host": torch.autograd.graph.save_on_cpu,
                  "rows apart": lambda: torch.autograd.graph.saved_tensors_hooks(apart, lambda t: t)}[hooks]
    leaves = [seeded_bf16(s, std=0.1, seed=i).cuda().requires_grad_() for i, s in enumerate(((M, K), (N, K), (N,)))]
    gy = seeded_bf16((M, N), std=0.01, seed=5).cuda()
    want = torch.autograd.grad(mxfp4.mxfp4_linear(*leaves), leaves, gy)
    with with_hooks():
        y = mxfp4.mxfp4_linear(*leaves)
    for got, w in zip(torch.autograd.grad(y, leaves, gy), want):
        assert torch.equal(got, w)


def test_rows_off_their_lines(host):
    """Operands and gradients that start at odd elements, an odd number of elements apart: copied, with the results of dense ones."""
    from lingua_amd import mxfp4, ops
    M, K, N = 5, 64, 48
    x, w, gy = (seeded_bf16((r, c + 3), seed=r + c).cuda()[:, 1:1 + c] for r, c in ((M, K), (N, K), (M, N)))

    def run(x, w, gy):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = mxfp4.mxfp4_linear(x, w)
        packed = mxfp4.pack(w)
        return (y, *torch.autograd.grad(y, (x, w), gy), mxfp4.linear_packed(x, *packed), ops.mxfp4_to_bf16(*packed, K))

    for got, want in zip(run(x, w, gy), run(*(t.contiguous() for t in (x, w, gy)))):
        assert torch.equal(got, want)


def test_refusals():
    from lingua_amd import mxfp4, ops
    x = seeded_bf16((4, 64), seed=1).cuda()
    q, s = ops.cast_mxfp4(x)[0]
    for bad in (lambda: ops.cast_mxfp4(x.float()), lambda: ops.cast_mxfp4(x, rowwise=False), lambda: ops.cast_mxfp4(x[:, :20]),
                lambda: ops.cast_mxfp4(x.cpu()), lambda: ops.mxfp4_to_bf16(q, s, 65), lambda: ops.mxfp4_to_bf16(q, s[:, :1], 32),
                lambda: ops.gemm_mxfp4_nt(q, q[:, :16], s, s[:, :1]), lambda: ops.gemm_mxfp4_nt(q, q, s, s, bias=x[0, :3]),
                lambda: ops.gemm_mxfp4_nt(q, q, s, s, out=torch.empty(4, 5, dtype=torch.bfloat16, device="cuda")),
                lambda: ops.gemm_mxfp4_nt(q, q, s.float(), s), lambda: mxfp4.linear_packed(x[:, :32], q, s), lambda: mxfp4.linear_packed(x[0], q, s),
                lambda: mxfp4.mxfp4_linear(x, x[:, :32]), lambda: mxfp4.mxfp4_linear(x, seeded_bf16((5, 64)).cuda()),
                lambda: mxfp4.mxfp4_linear(x.float(), x), lambda: mxfp4.mxfp4_linear(x, x.cpu())):
        with pytest.raises(RuntimeError):
            bad()
