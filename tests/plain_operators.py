"""The residual norm, the rotary positions and MXFP4 in 64 bits, from their definitions, in plain PyTorch: what the kernels are held
against.  Runs on any device and uses nothing of the package.  Beside it a fixture that the tests of these operators share."""
import pytest
import torch

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2      # a rounding to bf16 is off by at most this much of the value
FP32 = torch.finfo(torch.float32).eps / 2


def mx_quantise(x):
    """(codes uint8 [R, 32 * blocks], bytes uint8 [R, blocks]) of bf16 x, blocks along the rows."""
    R, C = x.shape
    pad = torch.zeros(R, -C % 32, dtype=torch.bfloat16, device=x.device)
    b = torch.cat((x, pad), 1).reshape(R, (C + 31) // 32, 32)
    v = b.double()
    amax = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    # floor(log2) of a finite bf16 is its exponent field; blocks below the normal numbers keep the smallest scale
    field = (b.abs().amax(2).view(torch.int16).int() >> 7)
    byte = (field - 2).clamp(min=0)
    scaled = torch.where(bad[..., None], torch.zeros_like(v), v) / torch.exp2(byte.double() - 127)[..., None]
    mag, table = scaled.abs(), E2M1.to(x.device)
    # nearest code, a tie to the even one (codes 0, 2, 4, 6 have an even mantissa), everything beyond 6 to 6
    upper = torch.searchsorted(table, mag.contiguous()).clamp(max=7)
    lower = (upper - 1).clamp(min=0)
    du, dl = (table[upper] - mag).abs(), (mag - table[lower]).abs()
    code = torch.where((du < dl) | ((du == dl) & (upper % 2 == 0)), upper, lower)
    code = (code + 8 * torch.signbit(v).long()).to(torch.uint8)
    code[bad] = 0
    byte[bad] = 255
    assert bool((amax[~bad] < 2.0 ** 128).all())
    return code.flatten(1), byte.to(torch.uint8)


def mx_values(code, byte):
    """fp64 [R, 32 * blocks] of codes and scales; NaN where the scale is."""
    c = code.long()
    v = E2M1.to(code.device)[c & 7] * (1 - 2 * (c >> 3).double())
    s = torch.exp2(byte.double() - 127)
    s[byte == 255] = float("nan")
    return (v.unflatten(1, (-1, 32)) * s[..., None]).flatten(1)


def mx_pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()


def mx_unpack(q):
    q = q.view(torch.uint8)
    return torch.stack((q & 15, q >> 4), 2).flatten(1)


def mx_rounded(x):
    """What MXFP4 makes of x, in 64 bits."""
    return mx_values(*mx_quantise(x))[:, :x.shape[1]]


def add_rmsnorm(x, residual, w, eps):
    """fp64 (h as kept, r, y) of the norm of a bf16 sum."""
    h = (x.double() + residual.double()).to(torch.bfloat16).double()
    r = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, r, h * r * w.double()


def add_rmsnorm_gradients(h, r, w, gy, gh):
    """fp64 (gradient of either operand, of the weight) and the sums of magnitudes that bound their rounding."""
    hat, t = h * r, gy * w
    dot = (t * hat).mean(-1, keepdim=True)
    g = gh + r * (t - hat * dot)
    size = gh.abs() + r * (t.abs() + hat.abs() * (t * hat).abs().mean(-1, keepdim=True))
    return g, (gy * hat).sum(0), size, (gy * hat).abs().sum(0)


def rotate(x, cos, sin, in_halves):
    """fp64 rotation of x [..., D] by cos, sin that broadcast to [..., rot / 2]."""
    rot = 2 * cos.shape[-1]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if in_halves else (2 * i, 2 * i + 1)
    y = x.double().clone()
    xa, xb = x[..., a].double(), x[..., b].double()
    y[..., a] = xa * cos.double() - xb * sin.double()
    y[..., b] = xa * sin.double() + xb * cos.double()
    return y


def within(got, want, size):
    """Is a bf16 ``got`` the rounding of something within ``size`` of ``want``?  (Subnormal results are off by a step of theirs.)"""
    got, want = got.double().cpu(), want.cpu()
    bound = want.abs() * HALF_STEP + size.cpu() * (1 + HALF_STEP) + 2.0 ** -134
    return bool(((got - want).abs() <= bound).all())


@pytest.fixture(params=["extension", "python"])
def host(request, monkeypatch):
    """Both host paths of an operator: a kernel timer wants to see single launches, which the host extension does not show."""
    if request.param == "python":
        from lingua_amd import ops
        monkeypatch.setattr(ops, "kernel_timer", [])
    return request.param
