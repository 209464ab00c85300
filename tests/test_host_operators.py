"""What the host refuses of the residual norm, the rotary positions and MXFP4 before anything is enqueued, the plain forms against
their definitions, and the tables of rotary positions: no GPU needed."""
import copy
import ctypes
import io
import math

import pytest
import torch

import plain_operators as plain
from lingua_amd import _lib

P = 1 << 20      # an address that is aligned and never touched


def refused(name, *args):
    lib = _lib.load()
    code = getattr(lib, name)(*args)
    return code == -1 and name.split("_many")[0].encode()[:6] in lib.l8_last_error()


GEMM = dict(A=P, sa=P, B=P, sb=P, M=64, N=64, K=256, lda=128, ldsa=16, ldb=128, ldsb=16, bias=None, C=P, ldc=64, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change", [dict(M=-1), dict(C=None), dict(ldc=63), dict(A=None), dict(sb=None), dict(lda=120), dict(lda=112), dict(ldb=(1 << 23)), dict(A=P + 8),
                                    dict(ldsa=8), dict(ldsb=24), dict(sa=P + 4), dict(C=P + 1), dict(bias=P + 1), dict(K=1 << 24, lda=1 << 23), dict(M=1 << 28), dict(N=1 << 28),
                                    dict(M=8192, N=8192, ldc=8192, K=4096, lda=2048, ldb=2048, ldsa=128, ldsb=128), dict(M=8192, N=8192, ldc=8192, K=4096, lda=2048, ldb=2048, ldsa=128,
                                                                                                               ldsb=128, ws=P, ws_bytes=100),
                                    dict(M=(1 << 28) - 1, N=(1 << 28) - 1, ldc=1 << 28)])
def test_product_is_refused(change):
    assert refused("l8_gemm_mxfp4_nt", *{**GEMM, **change}.values())


def test_two_casts_are_refused():
    import struct
    good, bad = [P, 64, 64, 64, P, 32, P, 16, P, 32, P, 16], [P, 64, 60, 64, P, 32, P, 16, P, 32, P, 16]
    assert refused("l8_cast_mxfp4_two", None, None)
    assert refused("l8_cast_mxfp4_two", struct.pack("24q", *good, *bad), None) and refused("l8_cast_mxfp4_two", struct.pack("24q", *bad, *good), None)
    empty = [0, 0, 64, 64] + [0] * 8
    assert _lib.load().l8_cast_mxfp4_two(struct.pack("24q", *empty, *empty), None) == 0


def test_product_workspace():
    lib = _lib.load()
    assert lib.l8_gemm_mxfp4_workspace(64, 64, 4096) == 0 and lib.l8_gemm_mxfp4_workspace(0, 64, 64) == 0 and lib.l8_gemm_mxfp4_workspace(-1, 8192, 8192) == 0
    assert lib.l8_gemm_mxfp4_workspace(8192, 8000, 4096) == 2 * 8192 * 128     # whole tiles of 256 rows, whole windows of 512 columns
    assert lib.l8_gemm_mxfp4_workspace(8192, 8192, 4100) == 2 * 8192 * 144


CAST = dict(x=P, R=64, C=64, ldx=64, q=P, ldq=32, s=P, lds=4, qt=P, ldqt=32, st=P, ldst=4, stream=None)


@pytest.mark.parametrize("change", [dict(R=-1), dict(x=None), dict(C=60, ldx=64), dict(ldx=60), dict(ldx=56), dict(x=P + 8), dict(q=None), dict(st=None), dict(ldq=24), dict(ldq=16),
                                    dict(q=P + 8), dict(lds=2), dict(lds=1), dict(s=P + 2), dict(ldqt=16), dict(qt=P + 4), dict(ldst=6), dict(R=1048561, ldqt=1 << 20, ldst=1 << 16),
                                    dict(q=None, s=None, qt=None, st=None)])
def test_cast_is_refused(change):
    assert refused("l8_cast_mxfp4", *{**CAST, **change}.values())


BACK = dict(q=P, ldq=32, s=P, lds=2, R=8, C=64, y=P, ldy=64, stream=None)


@pytest.mark.parametrize("change", [dict(C=-1), dict(q=None), dict(y=None), dict(ldq=30), dict(ldq=16), dict(q=P + 2), dict(lds=1), dict(ldy=63), dict(R=1048561)])
def test_back_to_bf16_is_refused(change):
    assert refused("l8_mxfp4_to_bf16", *{**BACK, **change}.values())


LINEAR = dict(x=P, M=4, K=256, ldx=256, qw=P, ldqw=128, sw=P, ldsw=8, N=64, bias=None, y=P, ldy=64, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change", [dict(M=-1), dict(x=None), dict(qw=None), dict(sw=None), dict(y=None), dict(ldy=32), dict(K=252, ldx=256), dict(ldx=252), dict(x=P + 8), dict(ldqw=120),
                                    dict(ldqw=112), dict(qw=P + 8), dict(ldsw=7), dict(M=17), dict(M=17, ws=P, ws_bytes=64), dict(M=200), dict(M=1 << 20), dict(N=1 << 28), dict(y=P + 1),
                                    dict(ldx=(1 << 25) + 8)])
def test_packed_linear_is_refused(change):
    assert refused("l8_mxfp4_linear", *{**LINEAR, **change}.values())


class Operand(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("y", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("heads", "ldb", "lds", "ldh")]


ROTARY = dict(B=2, S=3, D=64, rot=64, half=0, inverse=0, cos=P, sin=P, row=32, col=1, length=8, pos=None, i32=0, pos_b=0, pos_s=0, stream=None)


@pytest.mark.parametrize("change", [dict(B=-1), dict(D=63), dict(D=514), dict(rot=0), dict(rot=3), dict(rot=66), dict(cos=None), dict(sin=P + 2), dict(length=2), dict(B=1 << 12, S=1 << 12),
                                    dict(x=None), dict(y=P + 1), dict(heads=1 << 24), dict(heads=-1)])
def test_rotary_is_refused(change):
    own = {k: change.pop(k) for k in ("x", "y", "heads") if k in change}
    fields = dict(x=P, y=P, heads=4, ldb=768, lds=256, ldh=64, **{}) | own
    two = (Operand * 2)(Operand(**fields), Operand(**{**fields, "heads": 1, "x": P, "y": P}))
    assert refused("l8_rotary", two, *{**ROTARY, **change}.values())


NORM = dict(x=P, res=P, w=P, f32=0, R=4, C=64, ldx=64, ldr=64, eps=1e-5, h=P, ldh=64, y=P, ldy=64, q=P, ldq=64, scale=P, rstd=None, col=None, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change", [dict(R=-1), dict(res=None), dict(h=None), dict(q=None), dict(C=60), dict(ldr=60), dict(ldh=56), dict(res=P + 8), dict(h=P + 8), dict(C=8200), dict(col=P),
                                    dict(col=P, ws=P, ws_bytes=8), dict(col=P, q=None, scale=None)])
def test_residual_norm_is_refused(change):
    assert refused("l8_add_rmsnorm_cast_rowwise", *{**NORM, **change}.values())


BACKWARD = dict(gy=P, gh=P, h=P, w=P, f32=0, rstd=P, R=4, C=64, ldgy=64, ldgh=64, ldh=64, gx=P, ldgx=64, gw=P, gw_f32=1, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [dict(C=-1), dict(gh=None), dict(gy=None), dict(gw=None), dict(ldgh=60), dict(gh=P + 8), dict(C=8200), dict(ws=None), dict(ws_bytes=16)])
def test_residual_norm_backward_is_refused(change):
    assert refused("l8_add_rmsnorm_bwd", *{**BACKWARD, **change}.values())


def test_no_cpu_path():
    from lingua_amd import mxfp4, norm, ops, rope
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8)
    cos = torch.zeros(4, 8)
    for call in (lambda: norm.add_rmsnorm(x, x, x[0], 1e-5), lambda: ops.cast_mxfp4(x), lambda: ops.mxfp4_to_bf16(q, s, 64), lambda: ops.gemm_mxfp4_nt(q, q, s, s),
                 lambda: mxfp4.mxfp4_linear(x, w), lambda: mxfp4.linear_packed(x, q, s), lambda: mxfp4.Mxfp4Linear(64, 64, dtype=torch.bfloat16)(x),
                 lambda: rope.rotary(x.view(1, 2, 4, 16), x.view(1, 2, 4, 16), cos, cos)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_plain_quantisation_is_the_nearest_code_to_even():
    """The quantiser that the kernels are held against, by brute force over all codes."""
    g = torch.Generator().manual_seed(0)
    x = torch.cat((torch.randn(64, 64, generator=g), torch.randint(-48, 49, (64, 64), generator=g) / 8.0), 1).to(torch.bfloat16)
    x[3, :32], x[4, 5], x[5, 70] = 0.0, float("nan"), float("inf")
    code, byte = plain.mx_quantise(x)
    for r in range(64):
        for b in range(4):
            v = [float(t) for t in x[r, 32 * b:32 * b + 32]]
            if not all(map(math.isfinite, v)):
                assert int(byte[r, b]) == 255 and not code[r, 32 * b:32 * b + 32].any()
                continue
            top = max(map(abs, v))
            want = max(math.floor(math.log2(top)) - 2 + 127, 0) if top else 0
            assert int(byte[r, b]) == want
            for i, t in enumerate(v):
                scaled = abs(t) / 2.0 ** (want - 127)
                table = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
                best = min(range(8), key=lambda k: (abs(table[k] - scaled), k % 2))
                got = int(code[r, 32 * b + i])
                assert got & 7 == best and (got >> 3) == int(math.copysign(1, t) < 0)
    assert torch.equal(plain.mx_unpack(plain.mx_pack(code)), code)


def test_tables():
    from lingua_amd import rope
    cos, sin = rope.rotary_tables(64, 200000)
    assert cos.shape == sin.shape == (200000, 32) and cos.dtype == torch.float32
    for p, i in ((0, 0), (199999, 0), (123457, 7), (199999, 31)):
        angle = p * 10000.0 ** (-2 * i / 64)
        assert abs(float(cos[p, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[p, i]) - math.sin(angle)) < 1e-7
    linear = rope.rotary_tables(64, 64, scaling="linear", factor=4)
    assert torch.equal(linear[0][::4], rope.rotary_tables(64, 16)[0])
    ntk, plain_cos = rope.rotary_tables(64, 32, scaling="ntk", factor=4), rope.rotary_tables(64, 32)
    assert torch.equal(ntk[0][:, 0], plain_cos[0][:, 0])                                    # the highest frequency stays
    assert torch.allclose(ntk[0][::4, -1], plain_cos[0][:8, -1], rtol=0, atol=2e-7)         # the lowest is interpolated
    yarn = rope.rotary_tables(64, 32, scaling="yarn", factor=4, trained_length=2048)
    size = 0.1 * math.log(4) + 1
    assert torch.allclose(yarn[0][:, 0], plain_cos[0][:, 0] * size, rtol=0, atol=2e-7)
    assert torch.allclose(yarn[0][::4, -1], plain_cos[0][:8, -1] * size, rtol=0, atol=2e-7)
    for bad in (dict(rot=3, length=4), dict(rot=4, length=-1), dict(rot=4, length=4, scaling="other"), dict(rot=4, length=4, scaling="linear", factor=0.5),
                dict(rot=4, length=4, scaling="yarn", factor=2), dict(rot=2, length=4, scaling="ntk", factor=2)):
        with pytest.raises(RuntimeError):
            rope.rotary_tables(**bad)


def test_conversion_keeps_parameters_and_refuses_other_modules():
    from bench_workloads import Llama
    from lingua_amd import mxfp4, norm
    model = Llama(n_layers=1, dim=32, n_heads=2, ffn_dim=64, vocab=16).to(torch.bfloat16)
    keys, weight = list(model.state_dict()), model.layers[0].feed_forward.w1.weight
    mxfp4.convert_linears_to_mxfp4(model, r"feed_forward\.")
    assert type(model.layers[0].feed_forward.w1) is mxfp4.Mxfp4Linear and model.layers[0].feed_forward.w1.weight is weight
    assert type(model.layers[0].attention.wq) is torch.nn.Linear and type(model.output) is torch.nn.Linear
    with pytest.raises(AssertionError):
        mxfp4.convert_linears_to_mxfp4(model, r"feed_forward\.")
    with pytest.raises(RuntimeError, match="fuse_rmsnorm first"):
        norm.fuse_residual_norm(model)
    norm.fuse_residual_norm(norm.fuse_rmsnorm(model))
    assert list(model.state_dict()) == keys and type(model.layers[0]).__name__ == "TransformerBlock"
    # a fused model can be copied and pickled
    buffer = io.BytesIO()
    torch.save(model, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(model), torch.load(buffer, weights_only=False)):
        assert type(other.layers[0]) is type(model.layers[0]) and list(other.state_dict()) == keys
        assert other.layers[0].ffn_norm is not model.layers[0].ffn_norm


def interpreted(monkeypatch):
    """The Python forms on the CPU, plain torch in the kernels' place: name -> (output, leaves) of fresh leaves."""
    from lingua_amd import float8, mxfp4, norm, ops, rope
    g = torch.Generator().manual_seed(0)
    leaf = lambda *shape: torch.randn(shape, generator=g).to(torch.bfloat16).requires_grad_()   # noqa: E731
    cos, sin = rope.rotary_tables(16, 4)
    turn = lambda t, s: None if t is None else plain.rotate(t.detach(), cos[None, :, None], s[None, :, None], False).to(torch.bfloat16)   # noqa: E731
    monkeypatch.setattr(float8.config, "share_input_casts", False)
    monkeypatch.setattr(ops, "rotary", lambda q, k, c, s, p, half, inverse=False: (turn(q, -sin if inverse else sin), turn(k, -sin if inverse else sin)))
    pair = lambda x: (x.detach().clone(), torch.zeros(()))   # noqa: E731
    monkeypatch.setattr(ops, "cast_mxfp4", lambda x, rowwise=True, transposed=False, on_lines=False: (pair(x) if rowwise else None, pair(x.t()) if transposed else None))
    monkeypatch.setattr(ops, "gemm_mxfp4_nt", lambda a, b, sa, sb, bias=None: a @ b.t() + (0 if bias is None else bias.detach()))
    monkeypatch.setattr(ops, "col_sum", lambda t: t.sum(0))

    def forward(x, r, w, eps, col_amax=None, on_lines=False):
        h, rstd, y = plain.add_rmsnorm(x.detach(), r.detach(), w.detach(), eps)
        return h.to(torch.bfloat16), y.to(torch.bfloat16), None, None, rstd

    def backward(gy, gh, h, w, rstd, gw_dtype):
        gx, gw, _, _ = plain.add_rmsnorm_gradients(h.double(), rstd, w.detach().double(), gy.double(), gh.double())
        return gx.to(torch.bfloat16), gw.to(gw_dtype)

    monkeypatch.setattr(ops, "add_rmsnorm_cast_rowwise", forward)
    monkeypatch.setattr(ops, "add_rmsnorm_bwd", backward)
    monkeypatch.setattr(ops, "rmsnorm_bwd", lambda gy, h, w, rstd, gw_dtype: backward(gy, torch.zeros_like(gy), h, w, rstd, gw_dtype))
    x, w, gain, q = leaf(4, 16), leaf(8, 16), leaf(16), leaf(1, 4, 2, 16)
    return {"add_rmsnorm": (lambda: norm.Fp8AddRMSNormFn.apply(x, x.detach(), gain, 1e-5, False)[1], (x, gain)),
            "rotary": (lambda: rope.RotaryFn.apply(q, q, cos, sin, None, False)[0], (q,)),
            "mxfp4_linear": (lambda: mxfp4.Mxfp4LinearFn.apply(x, w, gain[:8]), (x, w, gain))}


@pytest.mark.parametrize("name", ["add_rmsnorm", "rotary", "mxfp4_linear"])
@pytest.mark.parametrize("linear_loss", [False, True])
def test_python_forms_refuse_second_derivatives(name, linear_loss, monkeypatch):
    call, leaves = interpreted(monkeypatch)[name]
    for leaf in leaves:
        loss = call().float()
        loss = loss.sum() if linear_loss else loss.square().sum()
        grad, = torch.autograd.grad(loss, leaf, create_graph=True)
        if linear_loss and (name == "rotary" or (name == "mxfp4_linear" and leaf is leaves[2])):
            assert not grad.requires_grad      # these are linear: the gradient of a constant's is a constant
            continue
        with pytest.raises(RuntimeError, match=f"{name} is not differentiable twice"):
            (loss + grad.float().square().sum()).backward()


# 2^32 threads and more are not a grid: refused before anything is enqueued
def test_more_threads_than_a_grid_has_are_refused():
    wide = dict(M=(1 << 20) - 256, N=(1 << 20) - 1, ldc=1 << 20, ws=P, ws_bytes=1 << 60)     # (an odd N: tiles of 128 x 128)
    assert refused("l8_gemm_mxfp4_nt", *{**GEMM, **wide}.values())
    assert refused("l8_cast_mxfp4", *{**CAST, **dict(R=1, C=1 << 30, ldx=1 << 30, ldq=1 << 29, lds=1 << 25, ldqt=16, ldst=4)}.values())
    import struct
    small, large = [P, 64, 64, 64, P, 32, P, 16, P, 32, P, 16], [P, 1, 1 << 30, 1 << 30, P, 1 << 29, P, 1 << 25, P, 16, P, 4]
    assert refused("l8_cast_mxfp4_two", struct.pack("24q", *small, *large), None)
    assert refused("l8_mxfp4_linear", *{**LINEAR, **dict(N=(1 << 27) - 15, K=32, ldx=32, ldqw=16, ldsw=1, ldy=1 << 27)}.values())
    odd = dict(M=100, N=(1 << 27) - 16, K=(1 << 24) - 32, ldx=1 << 24, ldqw=(1 << 23) - 16, ldsw=(1 << 19) + 1, ldy=1 << 27, ws=P, ws_bytes=1 << 60)
    assert refused("l8_mxfp4_linear", *{**LINEAR, **odd}.values())
