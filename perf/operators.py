"""The operators around and inside a block's linears, as cases that can be timed and compared: residual addition with RMSNorm and
e4m3 output, rotary positions, MXFP4 quantisation, MXFP4 linears.

A case is one call (serving) or one forward + backward (training) through the public entry points.  Keys of a case:
  op      "norm"    h = x + residual, y = rmsnorm(h), and (serving) y's e4m3 copy with row scales; training: gradients too
          "rotary"  rotation of q and k by their positions; training: of their gradients too
          "cast"    a matrix to MXFP4 along its rows and along its columns, and back to bf16
          "linear"  x @ w.T (+ bias) in MXFP4; serving takes a packed weight, training quantises all it multiplies
  rows, cols            shape of the activation (norm, cast, linear: cols is the reduction)
  out                   output features (linear)
  weight                type of the norm's weight
  batch, seq, heads, kv_heads, head_dim, rot   shape of q and k, columns of a head that are rotated (rotary)
  layout                "interleaved" or "half"
  far                   tokens stand at positions of a long sequence, given as a tensor (serving)
  train, bias
"""
import math

import torch

own = False

EPS = 1e-5
FAR = 131072   # length of the rotary tables where positions are far


def listed():
    return [
        # one sequence in generation, a 1B-sized model: latency alone counts
        dict(name="norm_decode_1", op="norm", rows=1, cols=2048, weight="bf16", train=False),
        # a short ragged batch in training, weights kept in fp32
        dict(name="norm_train_ragged", op="norm", rows=1021, cols=5120, weight="fp32", train=True),
        # a 7B-sized block's norm in training, 4 x 4096 tokens
        dict(name="norm_train_7b", op="norm", rows=16384, cols=4096, weight="bf16", train=True),
        # 32 sequences in generation at far positions of a long context, half layout, half of the head, shared key heads
        dict(name="rotary_decode_32", op="rotary", batch=32, seq=1, heads=32, kv_heads=8, head_dim=128, rot=64, layout="half", far=True, train=False),
        # three ragged sequences in training, half layout, a part of the head that no vector width divides
        dict(name="rotary_train_ragged", op="rotary", batch=3, seq=341, heads=12, kv_heads=4, head_dim=96, rot=40, layout="half", far=False, train=True),
        # a 7B-sized attention in training, 4 x 4096 tokens, q and k as slices of one product
        dict(name="rotary_train_7b", op="rotary", batch=4, seq=4096, heads=32, kv_heads=32, head_dim=128, rot=128, layout="interleaved", far=False, train=True),
        # a small ragged activation with a last block that is not full
        dict(name="cast_ragged", op="cast", rows=333, cols=2064),
        # a 7B-sized MLP weight
        dict(name="cast_weight_7b", op="cast", rows=11008, cols=4096),
        # one sequence in generation through a 7B-sized projection
        dict(name="linear_decode_1", op="linear", rows=1, cols=4096, out=4096, train=False, bias=False),
        # 32 sequences in generation through a 7B-sized MLP's first linear
        dict(name="linear_decode_32", op="linear", rows=32, cols=4096, out=11008, train=False, bias=True),
        # a short ragged batch in training with a bias
        dict(name="linear_train_ragged", op="linear", rows=1021, cols=2048, out=2064, train=True, bias=True),
        # a 7B-sized MLP's linear in training, 4 x 4096 tokens: the largest case
        dict(name="linear_train_7b", op="linear", rows=16384, cols=4096, out=11008, train=True, bias=False),
    ]


_MOST_FLOPS = 6 * 16384 * 4096 * 11008
_MOST_BYTES = 16 * 16384 * 4096


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "cast", "linear", "linear"))
    train = rng.random() < 0.5
    if op == "norm":
        cols = 8 * _log_uniform(rng, 32, 1024)
        rows = _log_uniform(rng, 64, 16384) if train else _log_uniform(rng, 1, 16384)
        return dict(op=op, rows=max(1, min(rows, _MOST_BYTES // (16 * cols))), cols=cols, weight=rng.choice(("bf16", "fp32")), train=train)
    if op == "rotary":
        head_dim = 8 * rng.randint(4, 32)
        rot = head_dim if rng.random() < 0.5 else 2 * rng.randint(4, head_dim // 2)
        kv_heads = rng.choice((1, 2, 4, 7, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5))
        batch, seq = (rng.randint(1, 6), _log_uniform(rng, 16, 4096)) if train else (_log_uniform(rng, 1, 256), rng.choice((1, 1, 3, 64)))
        most = _MOST_BYTES // (8 * batch * (heads + kv_heads) * head_dim)
        return dict(op=op, batch=batch, seq=max(1, min(seq, most)), heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot=rot,
                    layout=rng.choice(("interleaved", "half")), far=not train, train=train)
    cols = 16 * _log_uniform(rng, 16, 768)
    if op == "cast":
        return dict(op=op, rows=_log_uniform(rng, 1, 16384), cols=8 * _log_uniform(rng, 16, 512))
    out = 16 * _log_uniform(rng, 16, 768)
    rows = _log_uniform(rng, 65, 16384) if train else _log_uniform(rng, *rng.choice(((1, 64), (65, 8192))))
    rows = max(1, min(rows, _MOST_FLOPS // (6 * cols * out)))
    return dict(op=op, rows=rows, cols=cols, out=out, train=train, bias=rng.random() < 0.4)


def work(case):
    op = case["op"]
    if op == "norm":
        n, w = case["rows"] * case["cols"], (2 if case["weight"] == "bf16" else 4) * case["cols"]
        if case["train"]:   # x, residual -> h, y; gy, gh, h -> one gradient for both, the weight's
            return {"bytes": 8 * n + 8 * n + 3 * w, "flops": 24 * n}
        return {"bytes": 9 * n + 4 * case["rows"] + w, "flops": 10 * n}
    if op == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        r = tokens * (case["heads"] + case["kv_heads"]) * case["rot"]
        tables = 4 * case["rot"] * (tokens if case["far"] else case["seq"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (4 * n + tables), "flops": passes * 3 * r}
    if op == "cast":   # read once, two packed copies written; the packed copies read and two bf16 ones written
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n + 2 * 17 * n // 32 + 2 * 17 * n // 32 + 4 * n, "flops": 6 * n}
    m, k, n = case["rows"], case["cols"], case["out"]
    if case["train"]:
        return {"bytes": 2 * (m * k + n * k + m * n) + 2 * (m * k + n * k + m * n), "flops": 6 * m * n * k}
    return {"bytes": 17 * n * k // 32 + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _activation(g, rows, cols):
    """What a block hands its linears: channels of different sizes, a few of them large, and padding rows of zeros."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x *= torch.exp(torch.randn((cols,), generator=g, device="cuda"))
    x[torch.rand((rows,), generator=g, device="cuda") < 0.01 * (rows > 1)] = 0
    return x.to(torch.bfloat16)


def _leaf(t):
    return t.detach().requires_grad_()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "norm":
        rows, cols, train = case["rows"], case["cols"], case["train"]
        s["x"], s["residual"] = _activation(g, rows, cols), _normal(g, rows, cols, std=3.0)
        w = 1 + 0.2 * torch.randn((cols,), generator=g, device="cuda")
        s["w"] = w.to(torch.bfloat16) if case["weight"] == "bf16" else w
        if train:
            for name in ("x", "residual", "w"):
                s[name] = _leaf(s[name])
            s["gy"], s["gh"] = _normal(g, rows, cols, std=1e-3), _normal(g, rows, cols, std=1e-3)
    elif op == "rotary":
        B, S, H, K, D, rot = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "head_dim", "rot"))
        y = _normal(g, B * S, (H + 2 * K) * D)     # the product for q, k and v, of which q and k are column slices
        q, k = y[:, :H * D].view(B, S, H, D), y[:, H * D:(H + K) * D].view(B, S, K, D)
        length = FAR if case["far"] else S
        inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        if case["far"]:
            inv = inv / 8     # positions interpolated for a context eight times as long
        angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = None
        if case["far"]:
            start = torch.randint(0, FAR - S, (B, 1), generator=g, device="cuda")
            s["positions"] = start + torch.arange(S, device="cuda")
        if case["train"]:
            s["q"], s["k"] = _leaf(q), _leaf(k)
            # gradients as attention hands them back: heads in front of tokens
            s["gq"], s["gk"] = _normal(g, B, H, S, D, std=1e-3).transpose(1, 2), _normal(g, B, K, S, D, std=1e-3).transpose(1, 2)
        else:
            s["q"], s["k"] = q, k
    elif op == "cast":
        s["x"] = _activation(g, case["rows"], case["cols"])
    else:
        m, k, n = case["rows"], case["cols"], case["out"]
        s["x"], w = _activation(g, m, k), _normal(g, n, k, std=0.02)
        s["bias"] = _normal(g, n) if case["bias"] else None
        if case["train"]:
            s["x"], s["w"] = _leaf(s["x"]), _leaf(w)
            if case["bias"]:
                s["bias"] = _leaf(s["bias"])
            s["gy"] = _normal(g, m, n, std=1e-3)
        else:   # as a checkpoint holds it: two codes a byte, the first in the low half, and a byte of scale for each 32
            code, byte = _codes(w)
            s["qw"], s["sw"] = code[:, 0::2] | code[:, 1::2] << 4, byte
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _blocks(x):
    """fp32 [R, blocks, 32], zeros behind the last column."""
    return torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))


def _codes(x):
    """e2m1 codes (uint8 [R, 32 * blocks], one a byte) and e8m0 scales (uint8 [R, blocks]) of a finite matrix, blocks along its rows."""
    b = _blocks(x)
    exponent = b.abs().amax(2).view(torch.int32) >> 23
    byte = (exponent - 2).clamp(min=0)
    up = torch.ldexp(torch.ones((), device=x.device), 127 - byte)[:, :, None]   # exact: powers of two down to 2^-125
    v = (b * up).abs()
    # the number of borders below v, of which a border itself counts where the code above it is even
    code = ((v > 0.25).byte() + (v >= 0.75).byte() + (v > 1.25).byte() + (v >= 1.75).byte() + (v > 2.5).byte() + (v >= 3.5).byte() + (v > 5).byte())
    code |= torch.signbit(b).byte() << 3
    return code.flatten(1), byte.byte()


def _values(code, byte):
    """fp32 values that codes and scales stand for, [R, 32 * blocks]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    return (table[code.int()].unflatten(1, (-1, 32)) * torch.ldexp(torch.ones((), device=code.device), byte.int() - 127)[:, :, None]).flatten(1)


def _quantised(x):
    """What MXFP4 makes of x, blocks along its rows, in fp32."""
    return _values(*_codes(x))[:, :x.shape[1]]


def _kept_scale(scale):
    """A row's scale goes by the row's largest output as bf16, whose last bit follows the order of the norm's sum: it is compared
    at that width."""
    return scale.to(torch.bfloat16)


def _plain_norm(s):
    x, res, w = (s[k].detach() for k in ("x", "residual", "w"))
    h = (x.float() + res.float()).to(torch.bfloat16)
    hf = h.float()
    r = torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS)
    y = (hf * r * w.float()).to(torch.bfloat16)
    if not s["case"]["train"]:
        scale = y.float().abs().amax(1, keepdim=True).clamp(min=1e-12) / 448
        return {"h": h, "y": y, "q": (y.float() * (1 / scale)).to(torch.float8_e4m3fn), "scale": _kept_scale(scale)}
    gy, hat = s["gy"].float(), hf * r
    gh = gy * w.float()
    g = (s["gh"].float() + r * (gh - hat * (gh * hat).mean(1, keepdim=True))).to(torch.bfloat16)
    return {"h": h, "y": y, "gx": g, "gresidual": g, "gw": (gy * hat).sum(0).to(w.dtype)}


def _rotated(x, cos, sin, rot, layout):
    """x [B, S, H, D]; cos, sin [B or 1, S, 1, rot / 2]."""
    xf = x.float()
    turned, rest = xf[..., :rot], xf[..., rot:]
    if layout == "half":
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _at_positions(s, dtype=torch.float32):
    at = torch.arange(s["case"]["seq"], device="cuda")[None] if s["positions"] is None else s["positions"]
    return s["cos"][at][:, :, None].to(dtype), s["sin"][at][:, :, None].to(dtype)


def _plain_rotary(s):
    rot, layout = s["case"]["rot"], s["case"]["layout"]
    cos, sin = _at_positions(s)
    out = {"q": _rotated(s["q"].detach(), cos, sin, rot, layout), "k": _rotated(s["k"].detach(), cos, sin, rot, layout)}
    if s["case"]["train"]:
        out["gq"], out["gk"] = _rotated(s["gq"], cos, -sin, rot, layout), _rotated(s["gk"], cos, -sin, rot, layout)
    return out


def _plain_linear(s):
    x, bias = s["x"].detach(), s["bias"]
    if not s["case"]["train"]:
        code = torch.stack((s["qw"] & 15, s["qw"] >> 4), 2).flatten(1)
        w = _values(code, s["sw"])[:, :x.shape[1]]
        y = _quantised(x) @ w.t()
        return {"y": (y if bias is None else y + bias.float()).to(torch.bfloat16)}
    w, gy = s["w"].detach(), s["gy"]
    y = _quantised(x) @ _quantised(w).t()
    out = {"y": (y if bias is None else y + bias.detach().float()).to(torch.bfloat16),
           "gx": (_quantised(gy) @ _quantised(w.t()).t()).to(torch.bfloat16),
           "gw": (_quantised(gy.t()) @ _quantised(x.t()).t()).to(torch.bfloat16)}
    if bias is not None:
        out["gbias"] = gy.float().sum(0).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _own_norm(s):
    from lingua_amd import norm, ops
    if not s["case"]["train"]:
        h, y, q, scale, _ = ops.add_rmsnorm_cast_rowwise(s["x"], s["residual"], s["w"], EPS)
        return {"h": h, "y": y, "q": q, "scale": _kept_scale(scale)}
    h, y = norm.add_rmsnorm(s["x"], s["residual"], s["w"], EPS)
    gx, gres, gw = torch.autograd.grad((h, y), (s["x"], s["residual"], s["w"]), (s["gh"], s["gy"]))
    return {"h": h, "y": y, "gx": gx, "gresidual": gres, "gw": gw}


def _own_rotary(s):
    from lingua_amd import rope
    q, k = rope.rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], layout=s["case"]["layout"])
    out = {"q": q, "k": k}
    if s["case"]["train"]:
        out["gq"], out["gk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _own_cast(s):
    from lingua_amd import ops
    x = s["x"]
    (q, scale), (qt, scale_t) = ops.cast_mxfp4(x, rowwise=True, transposed=True)
    return {"rows": ops.mxfp4_to_bf16(q, scale, x.shape[1]), "columns": ops.mxfp4_to_bf16(qt, scale_t, x.shape[0])}


def _own_linear(s):
    from lingua_amd import mxfp4
    if not s["case"]["train"]:
        return {"y": mxfp4.linear_packed(s["x"], s["qw"], s["sw"], s["bias"])}
    y = mxfp4.mxfp4_linear(s["x"], s["w"], s["bias"])
    of = [s["x"], s["w"]] + ([s["bias"]] if s["bias"] is not None else [])
    grads = torch.autograd.grad(y, of, s["gy"])
    return {"y": y, **dict(zip(("gx", "gw", "gbias"), grads))}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "cast": _own_cast, "linear": _own_linear}[op](state)
    if op == "cast":
        x = state["x"]
        return {"rows": _quantised(x).to(torch.bfloat16), "columns": _quantised(x.t()).to(torch.bfloat16)}
    return {"norm": _plain_norm, "rotary": _plain_rotary, "linear": _plain_linear}[op](state)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------

def _exact_quantised(x):
    """MXFP4 of x in 64 bits: each block in steps of its own power of two, each value rounded to the step of its own octave."""
    R, C = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -C % 32)).reshape(R, -1, 32)
    top = torch.frexp(b.abs().amax(2, keepdim=True))[1].double() - 1          # 2^top <= amax < 2^(top + 1)
    unit = torch.exp2((top - 2).clamp(min=-127))
    v = b / unit
    octave = (torch.frexp(v)[1].double() - 1).clamp(min=0, max=2)
    step = torch.exp2(octave - 1)
    return (torch.round(v / step) * step).clamp(-6, 6).mul(unit).reshape(R, -1)[:, :C]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h64 = s["x"].detach().double() + s["residual"].detach().double()
        h = h64.to(torch.bfloat16).double()    # the norm is that of the sum as it is kept
        w = s["w"].detach().double()
        r = 1 / (h.square().mean(1, keepdim=True) + EPS).sqrt()
        y = h * r * w
        if not case["train"]:
            kept = y.to(torch.bfloat16).double()   # the copy is that of the output as it is kept
            scale = kept.abs().amax(1, keepdim=True).clamp(min=1e-12) / 448
            return {"h": h64, "y": y, "q": (kept / scale).to(torch.float8_e4m3fn), "scale": scale}
        gy, hat = s["gy"].double(), h * r
        t = gy * w
        g = s["gh"].double() + (t - hat * (t * hat).mean(1, keepdim=True)) * r
        return {"h": h64, "y": y, "gx": g, "gresidual": g, "gw": (gy * hat).sum(0)}
    if op == "rotary":
        cos, sin = _at_positions(s, torch.float64)
        rot = case["rot"]
        first = torch.arange(rot // 2, device="cuda")
        i, j = (first, first + rot // 2) if case["layout"] == "half" else (2 * first, 2 * first + 1)

        def turn(x, sin):
            z = torch.complex(x[..., i].double(), x[..., j].double()) * torch.complex(cos, sin)
            out = x.detach().double().clone()
            out[..., i], out[..., j] = z.real, z.imag
            return out

        out = {"q": turn(s["q"].detach(), sin), "k": turn(s["k"].detach(), sin)}
        if case["train"]:
            out["gq"], out["gk"] = turn(s["gq"], -sin), turn(s["gk"], -sin)
        return out
    if op == "cast":
        return {"rows": _exact_quantised(s["x"]), "columns": _exact_quantised(s["x"].t())}
    x = s["x"].detach()
    bias = 0 if s["bias"] is None else s["bias"].detach().double()
    if not case["train"]:
        low, high = (s["qw"] & 15).long(), (s["qw"] >> 4).long()
        c = torch.stack((low, high), 2).flatten(1)
        e, m = (c >> 1 & 3), (c & 1).double()
        value = torch.where(e == 0, m / 2, torch.exp2(e.double() - 1) * (1 + m / 2)) * (1 - 2 * (c >> 3).double())
        w = (value.unflatten(1, (-1, 32)) * torch.exp2(s["sw"].double() - 127)[:, :, None]).flatten(1)[:, :x.shape[1]]
        return {"y": _exact_quantised(x) @ w.t() + bias}
    w, gy = s["w"].detach(), s["gy"]
    out = {"y": _exact_quantised(x) @ _exact_quantised(w).t() + bias,
           "gx": _exact_quantised(gy) @ _exact_quantised(w.t()).t(),
           "gw": _exact_quantised(gy.t()) @ _exact_quantised(x.t()).t()}
    if s["bias"] is not None:
        out["gbias"] = gy.double().sum(0)
    return out
