"""Layer norm, counter-based dropout, rotary positions on several axes and low-rank adapters in 64 bits, from their definitions, in plain
PyTorch: what the kernels are held against.  Runs on any device and uses nothing of the package."""
import torch

from plain_operators import FP32


# ---- dropout ----

def philox(counter, key):
    """Four words of one counter of four words under a key of two: Philox4x32-10 in whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def keeps(numbers, site, p, n, first=0):
    """Which of the elements first .. first + n - 1 (first a multiple of 8) stay: bool [n] on the CPU."""
    seed, step = (int(v) for v in numbers.cpu())
    groups = range(first // 8, (first + n + 7) // 8)
    words = [philox((g & 0xffffffff, g >> 32, site, step & 0xffffffff), (seed & 0xffffffff, seed >> 32 & 0xffffffff)) for g in groups]
    halves = torch.tensor([h for ws in words for w in ws for h in (w & 0xffff, w >> 16)], dtype=torch.int64)[:n]
    return halves >= round(65536 * p)


def dropped(x, keep, p):
    """fp32 of a bf16 x as the kernels make it: the product with the factor, rounded to 32 bits; zero where not kept."""
    t = round(65536 * p)
    factor = torch.tensor(65536.0 / (65536 - t) if t < 65536 else 0.0, dtype=torch.float32)
    return torch.where(keep.view(x.shape).to(x.device), x.float() * factor.to(x.device), torch.zeros((), device=x.device))


# ---- layer norm ----

def layernorm(h, w, b, eps):
    """fp64 (hat, r, y) of h [R, C]; w, b fp64 [C]."""
    h = h.double()
    d = h - h.mean(1, keepdim=True)
    r = 1 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    return d * r, r, d * r * w + b


# Rounding errors of the kernels, in units of half an fp32 step.  A lane adds up at most 32 columns one after the other, six levels join the
# lanes and four the waves: a row's sum is off by at most 45 units of the sum of magnitudes.  The mean is then off by 45 |h| (|h| the mean
# magnitude); a difference from it by that and its own rounding.  The squared differences are taken about a wave's mean, where an error
# of the mean counts twice over only, and joined by n (m_wave - m)^2, whose error is 2 n |m_wave - m| (45 + 45) |h|: of 1 / deviation that is
# 90 |h| r, beside 45 / 2 of the sum and a few of root and quotient.

def hat_error(h, hat, r):
    k = h.double().abs().mean(1, keepdim=True) * r
    return FP32 * (48 * k + hat.abs() * (50 + 100 * k))


def y_error(h, hat, r, w, b):
    return w.abs() * hat_error(h, hat, r) + 3 * FP32 * ((hat * w).abs() + b.abs())


def layernorm_grads(h, hat, r, w, gy, gh):
    """fp64 (g, gw, gb) and what each may be off by; gh fp64 or None."""
    gy = gy.double()
    t, eh = gy * w, hat_error(h, hat, r)
    mt, mx = t.mean(1, keepdim=True), (t * hat).mean(1, keepdim=True)
    g = r * (t - mt - hat * mx)
    k = h.double().abs().mean(1, keepdim=True) * r
    emx = (t.abs() * eh).mean(1, keepdim=True) + FP32 * 50 * (t * hat).abs().mean(1, keepdim=True)
    err = r * (FP32 * (4 * t.abs() + 50 * t.abs().mean(1, keepdim=True) + 4 * (hat * mx).abs()) + hat.abs() * emx + eh * mx.abs()) + g.abs() * FP32 * (54 + 100 * k)
    if gh is not None:
        g = g + gh
        err = err + FP32 * 2 * (g.abs() + gh.abs())
    R = h.shape[0]
    return (g, (gy * hat).sum(0), gy.sum(0)), (err, (gy.abs() * eh).sum(0) + FP32 * (R + 8) * (gy * hat).abs().sum(0), FP32 * (R + 8) * gy.abs().sum(0))


def grad_within(got, want, error):
    """A gradient of a parameter, in bf16 or fp32: within `error` and its own rounding."""
    half = torch.finfo(got.dtype).eps / 2
    return bool(((got.double().cpu() - want.cpu()).abs() <= error.cpu() * (1 + half) + want.cpu().abs() * half + 1e-37).all())


# ---- low-rank adapters ----

# Rounding errors: a product of two bf16 is exact in 32 bits, a sum of D of them is off by at most D half steps of the sum of magnitudes in
# whatever order; h enters a product as two bf16 numbers, which leaves 2^-16 of it, and is scaled with one rounding.
SPLIT = 2.0 ** -16


def lowrank(y, x, a, b, index, scale):
    """fp64 (out, what it may be off by, h times scale, and its error) of one adapter after the other; y may be None."""
    x, a, b = (t.detach().double().cpu() for t in (x, a, b))
    index = index.cpu().long()
    n, r, D = a.shape
    T, N = x.shape[0], b.shape[2]
    s = torch.ones(n, dtype=torch.float64) if scale is None else scale.double().cpu()
    out = torch.zeros((T, N), dtype=torch.float64) if y is None else y.detach().double().cpu().clone()
    size, h, eh = torch.zeros((T, N), dtype=torch.float64), torch.zeros((T, r), dtype=torch.float64), torch.zeros((T, r), dtype=torch.float64)
    for i in range(n):
        at = (index == i).nonzero()[:, 0]
        if not len(at):
            continue
        h[at] = s[i] * (x[at] @ a[i].t())
        eh[at] = s[i].abs() * (FP32 * (D + 16)) * (x[at].abs() @ a[i].abs().t()) + (SPLIT + 4 * FP32) * h[at].abs()
        out[at] += h[at] @ b[i]
        size[at] = eh[at] @ b[i].abs() + FP32 * (2 * r + 4) * (h[at].abs() @ b[i].abs())
    size += FP32 * out.abs()
    return out, size, h, eh


def lowrank_grads(x, a, b, index, scale, gy):
    """fp64 (gx, ga, gb) and what each may be off by."""
    gx, ex, gh, egh = lowrank(None, gy, b, a, index, scale)
    _, _, h, eh = lowrank(None, x, a, b, index, scale)
    index = index.cpu().long()
    x, gy = x.detach().double().cpu(), gy.double().cpu()
    n, r, K = a.shape
    ga, gb = torch.zeros(a.shape, dtype=torch.float64), torch.zeros(b.shape, dtype=torch.float64)
    ea, eb = ga.clone(), gb.clone()
    for i in range(n):
        at = (index == i).nonzero()[:, 0]
        if not len(at):
            continue
        for grad, err, u, eu, z in ((ga, ea, gh, egh, x), (gb, eb, h, eh, gy)):
            grad[i] = u[at].t() @ z[at]
            err[i] = eu[at].t() @ z[at].abs() + FP32 * (2 * len(at) + 16) * (u[at].abs().t() @ z[at].abs())
    return (gx, ga, gb), (ex, ea, eb)
