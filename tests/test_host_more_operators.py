"""What the host refuses of layer norm, dropout, rotary positions on several axes and low-rank adapters before anything is enqueued: no GPU
needed."""
import struct

import pytest
import torch

from lingua_amd import _lib

P = 1 << 20      # an address that is aligned and never touched


def refused(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args) == -1 and name.encode() in lib.l8_last_error()


FWD = dict(x=P, residual=P, w=P, b=P, w_f32=0, b_f32=0, centred=1, R=4, C=64, ldx=64, ldr=64, eps=1e-5, numbers=P, site=0, threshold=100, h=P, ldh=64, y=P, ldy=64, q=P, ldq=64,
           scale=P, mean=P, rstd=P, col=0, ws=0, ws_bytes=0, stream=0)


@pytest.mark.parametrize("change", [dict(R=-1), dict(C=-8), dict(x=0), dict(y=0), dict(h=0), dict(C=60, ldx=64), dict(C=8200, ldx=8200, ldr=8200, ldh=8200, ldy=8200, ldq=8200), dict(ldx=60),
                                    dict(ldx=56), dict(x=P + 8), dict(residual=P + 8), dict(residual=0), dict(ldr=60), dict(h=P + 2), dict(ldh=32), dict(y=P + 8), dict(ldy=4), dict(q=0),
                                    dict(scale=0), dict(q=P + 4), dict(ldq=60), dict(w=P + 1), dict(w=P + 2, w_f32=1), dict(b=P + 2, b_f32=1), dict(col=P), dict(col=P, ws=P, ws_bytes=8),
                                    dict(col=P, q=0, scale=0), dict(site=-1), dict(site=1 << 32), dict(threshold=-1), dict(threshold=65537), dict(numbers=P + 4), dict(centred=0),
                                    dict(centred=0, b=0, numbers=0), dict(centred=0, b=0, w=0)])
def test_norm_is_refused(change):
    assert refused("l8_norm_fwd", struct.pack("11qd16q", *{**FWD, **change}.values()))


BWD = dict(gy=P, gh=P, h=P, w=P, w_f32=0, centred=1, R=4, C=64, ldgy=64, ldgh=64, ldh=64, mean=P, rstd=P, numbers=P, site=0, threshold=100, gx=P, ldgx=64, gres=P, ldgres=64, gw=P, gw_f32=1,
           gb=P, gb_f32=1, ws=P, ws_bytes=1 << 20, stream=0)


@pytest.mark.parametrize("change", [dict(R=-1), dict(C=-8), dict(gy=0), dict(h=0), dict(gx=0), dict(rstd=0), dict(mean=0), dict(C=60), dict(C=8200, ldgy=8200, ldgh=8200, ldh=8200, ldgx=8200,
                                                                                                                                 ldgres=8200), dict(ldgy=60),
                                    dict(gh=P + 8), dict(ldgh=56), dict(ldh=60), dict(ldgx=4), dict(gres=0), dict(numbers=0), dict(ldgres=60), dict(gres=P + 8), dict(w=P + 1), dict(ws=0),
                                    dict(ws_bytes=16), dict(ws=P + 8), dict(centred=0), dict(centred=0, gb=0, w=0), dict(threshold=70000)])
def test_norm_backward_is_refused(change):
    assert refused("l8_norm_bwd", struct.pack("27q", *{**BWD, **change}.values()))


DROP = dict(x=P, residual=P, y=P, n=64, numbers=P, site=0, threshold=1, stream=0)


@pytest.mark.parametrize("change", [dict(n=-1), dict(x=None), dict(y=None), dict(numbers=None), dict(x=P + 1), dict(residual=P + 1), dict(site=-1), dict(site=1 << 32), dict(threshold=65537),
                                    dict(numbers=P + 4), dict(n=1 << 35)])
def test_dropout_is_refused(change):
    assert refused("l8_dropout", *{**DROP, **change}.values())


ROTARY = dict(B=2, S=3, D=64, sections=(16, 8, 8), axes=3, rounds=0, half=0, inverse=0, cos=P, sin=P, row=32, col=1, length=8, pos=P, i32=0, pos_a=6, pos_b=3, pos_s=1, stream=None)


@pytest.mark.parametrize("change", [dict(B=-1), dict(D=63), dict(D=514), dict(axes=0), dict(axes=5, sections=(4, 4, 4, 4, 4)), dict(sections=(0, 0, 0)), dict(sections=(16, -8, 8)),
                                    dict(sections=(16, 8, 9)), dict(sections=(1 << 60, 1 << 60, 1 << 60)), dict(sections=(256, 1, 0), D=512), dict(cos=None), dict(sin=P + 2), dict(pos=None),
                                    dict(pos=P + 4), dict(pos=P + 2, i32=1), dict(length=-1), dict(B=1 << 12, S=1 << 12), dict(x=None), dict(y=P + 1), dict(heads=-1)])
def test_rotary_axes_is_refused(change):
    own = {k: change.pop(k) for k in ("x", "y", "heads") if k in change}
    fields = dict(x=P, y=P, heads=4, ldb=768, lds=256, ldh=64) | own
    args = {**ROTARY, **change}
    args["sections"] = struct.pack(f"{len(args['sections'])}q", *args["sections"])
    two = struct.pack("12q", *[v or 0 for v in fields.values()], P, P, 1, 768, 256, 64)
    assert refused("l8_rotary_axes", two, *args.values())


ROUTE = dict(index=P, i64=0, T=64, n=4, order=P, starts=P, stream=None)
SHRINK = dict(x=P, T=64, K=128, ldx=128, f=P, n=4, r=16, order=P, starts=P, h=P, splits=2, stream=None)
EXPAND = dict(y=P, ldy=128, h=P, splits=2, scale=P, f=P, T=64, N=128, n=4, r=16, order=P, starts=P, out=P, ldo=128, stream=None)


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=1 << 24), dict(n=0), dict(n=65535), dict(T=1 << 23, n=8191), dict(index=None), dict(index=P + 2), dict(index=P + 4, i64=1), dict(order=None), dict(order=P + 2),
                                    dict(starts=None), dict(starts=P + 1)])
def test_route_is_refused(change):
    assert refused("l8_lowrank_route", *{**ROUTE, **change}.values())


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=1 << 24), dict(n=0), dict(n=1 << 17), dict(r=0), dict(r=12), dict(r=136), dict(K=0), dict(K=12, ldx=16), dict(K=1 << 24, ldx=1 << 24),
                                    dict(x=None), dict(x=P + 8), dict(ldx=120), dict(ldx=132), dict(f=None), dict(f=P + 8), dict(h=None), dict(h=P + 4), dict(order=None), dict(starts=None),
                                    dict(splits=0), dict(splits=65), dict(T=(1 << 24) - 1, n=65534, splits=64)])
def test_shrink_is_refused(change):
    assert refused("l8_lowrank_shrink", *{**SHRINK, **change}.values())


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=1 << 24), dict(n=0), dict(r=4), dict(r=130), dict(N=0), dict(N=20, ldy=24, ldo=24), dict(y=P + 8), dict(ldy=64), dict(ldy=130), dict(h=None),
                                    dict(h=P + 8), dict(splits=0), dict(scale=P + 2), dict(f=None), dict(f=P + 2), dict(out=None), dict(out=P + 8), dict(ldo=132), dict(ldo=64), dict(order=None),
                                    dict(starts=P + 2), dict(T=(1 << 24) - 1, n=1, N=1 << 16, ldy=1 << 16, ldo=1 << 16)])
def test_expand_is_refused(change):
    assert refused("l8_lowrank_expand", *{**EXPAND, **change}.values())


SIDE = dict(h=P, splits=2, z=P, ldz=128, D=128, grad=P)
OUTER = dict(scale=P, T=64, n=4, r=16, order=P, starts=P, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=1 << 24), dict(n=0), dict(r=20), dict(D=0), dict(D=20, ldz=24), dict(h=0), dict(h=P + 8), dict(splits=0), dict(z=0), dict(z=P + 8), dict(ldz=120),
                                    dict(ldz=132), dict(grad=P + 8), dict(scale=P + 2), dict(order=None), dict(starts=None), dict(T=10000), dict(T=10000, ws=P, ws_bytes=64),
                                    dict(T=10000, ws=P + 8, ws_bytes=1 << 40), dict(T=(1 << 24) - 1, n=65534, ws=P, ws_bytes=1 << 60, D=1 << 20, ldz=1 << 20)])
def test_outer_is_refused(change):
    side = {**SIDE, **{k: v for k, v in change.items() if k in SIDE}}
    rest = {**OUTER, **{k: v for k, v in change.items() if k in OUTER}}
    for first in (True, False):
        both = (side, SIDE) if first else (SIDE, side)
        assert refused("l8_lowrank_outer", struct.pack("12q", *both[0].values(), *both[1].values()), *rest.values())


BOTH = dict(scale=P, f=P, also=P, T=64, n=4, r=16, order=P, starts=P, ws=P, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change", [dict(T=0), dict(T=-1), dict(n=0), dict(r=40), dict(r=4), dict(D=20, ldz=24), dict(h=0), dict(splits=65), dict(z=P + 8), dict(ldz=120), dict(grad=0), dict(grad=P + 8),
                                    dict(f=None), dict(f=P + 8), dict(also=None), dict(also=P + 4), dict(scale=P + 2), dict(order=None), dict(starts=None), dict(ws=None), dict(ws=P + 8),
                                    dict(ws_bytes=64)])
def test_outer_with_shrink_is_refused(change):
    side = {**SIDE, **{k: v for k, v in change.items() if k in SIDE}}
    assert refused("l8_lowrank_outer_shrink", struct.pack("6q", *side.values()), *{**BOTH, **{k: v for k, v in change.items() if k in BOTH}}.values())


def test_lowrank_splits_and_workspace():
    lib = _lib.load()
    assert lib.l8_lowrank_splits(0, 4, 16, 64) == lib.l8_lowrank_splits(-5, 4, 16, 64) == lib.l8_lowrank_splits(20, 2, 64, 8) == 1
    assert all(1 <= lib.l8_lowrank_splits(T, n, r, K) <= 16 for r in (8, 128) for T in (1, 16, 300, 1 << 20) for n in (1, 40, 1 << 16) for K in (8, 4096, 1 << 20))
    assert lib.l8_lowrank_outer_workspace(100, 16, 128, 128) == 0 and lib.l8_lowrank_outer_workspace(0, 16, 128, 128) == 0
    assert lib.l8_lowrank_outer_workspace(1 << 20, 16, 128, 256) % (4 * 16 * 384) == 0


def test_lowrank_arguments_are_refused():
    from lingua_amd import adapters
    bf = torch.bfloat16
    y, x, a, b, i = torch.zeros(4, 64, dtype=bf), torch.zeros(4, 32, dtype=bf), torch.zeros(2, 8, 32, dtype=bf), torch.zeros(2, 8, 64, dtype=bf), torch.zeros(4, dtype=torch.int32)
    call = adapters.add_lowrank
    for args in ((y, x, a[0], b, i), (y, x, a, b[:, :4], i), (y, x, a, b[:1], i), (y, x[:, :24], a, b, i), (y[:, :8], x, a, b, i), (y[:3], x, a, b, i), (y, x, a, b, i[:3]), (y, x, a, b, i[:, None]),
                 (y.float(), x, a, b, i), (y, x.float(), a, b, i), (y, x, a.float(), b, i), (y, x, a[:, :4], b[:, :4], i), (y, x.repeat(1, 1)[:, :12], a[:, :, :12], b, i),
                 (y, x, a.repeat(1, 17, 1), b.repeat(1, 17, 1), i), (y.to("meta"), x, a, b, i), (y, x, a, b, i.to("meta")),
                 (y, x, a, b, adapters.Plan(i, torch.zeros(6, dtype=torch.int32), 3, (4,)))):
        with pytest.raises(RuntimeError, match="do not fit|bf16|same tokens|rank|operands on|index is on|plan is for"):
            call(*args)
    with pytest.raises(RuntimeError, match="bank"):
        adapters.route(i, 0)


def test_adapters_beside_linears_keep_parameters():
    from lingua_amd import adapters
    model = torch.nn.ModuleDict({"w1": torch.nn.Linear(32, 64), "norm": torch.nn.LayerNorm(32)}).to(torch.bfloat16)
    weight = model["w1"].weight
    adapters.add_adapters(model, adapters.Requests(2), 8, "w1")
    assert list(model.state_dict()) == ["w1.a", "w1.b", "w1.scale", "w1.linear.weight", "w1.linear.bias", "norm.weight", "norm.bias"] and model["w1"].linear.weight is weight
    assert not model["w1"].b.any() and float(model["w1"].scale[1]) == 1
    x = torch.randn(3, 32, dtype=torch.bfloat16)
    assert torch.equal(model["w1"](x), model["w1"].linear(x))     # no request has one


def test_adapters_inside_a_fused_feed_forward_are_refused():
    """It multiplies by its linears' weights and never calls them: their adapters would be lost."""
    from lingua_amd import adapters, swiglu
    lin = [torch.nn.Linear(*s, bias=False, dtype=torch.bfloat16) for s in ((32, 64), (32, 64), (64, 32))]
    model = torch.nn.ModuleDict({"feed_forward": swiglu.Fp8FeedForward(*lin), "wo": torch.nn.Linear(32, 32)}).to(torch.bfloat16)
    for match in ("w2$", "w", "feed_forward"):
        with pytest.raises(RuntimeError, match="fused feed-forward"):
            adapters.add_adapters(model, adapters.Requests(2), 8, match)
    adapters.add_adapters(model, adapters.Requests(2), 8, "wo")
    assert isinstance(model["wo"], adapters.AdaptedLinear) and model["feed_forward"].w1 is lin[0]


def test_empty_calls_do_nothing():
    lib = _lib.load()
    assert lib.l8_lowrank_shrink(*{**SHRINK, "T": 0, "x": None}.values()) == 0 and lib.l8_lowrank_expand(*{**EXPAND, "T": 0, "out": None}.values()) == 0
    assert lib.l8_lowrank_outer(struct.pack("12q", *[0] * 12), *OUTER.values()) == 0
    assert lib.l8_dropout(None, None, None, 0, None, 0, 0, None) == 0
    assert lib.l8_norm_fwd(struct.pack("11qd16q", *{**FWD, "R": 0, "x": 0}.values())) == 0
    assert lib.l8_norm_bwd(struct.pack("27q", *{**BWD, "C": 0, "gy": 0}.values())) == 0
    assert lib.l8_norm_bwd(struct.pack("27q", *{**BWD, "R": 0, "gw": 0, "gb": 0}.values())) == 0
    assert lib.l8_norm_bwd_workspace(0, 64, 1) == 0 and lib.l8_norm_bwd_workspace(5, 0, 1) == 0


def test_arguments_are_refused():
    """Before anything asks for a GPU."""
    from lingua_amd import dropout, norm
    x, n = torch.zeros(4, 64, dtype=torch.bfloat16), dropout.numbers(1, "cpu")
    Drop = dropout.Drop
    for bad in (Drop(-0.1, n), Drop(1.1, n), Drop(float("nan"), n), Drop(0.1, n, -1), Drop(0.1, n, 1 << 32), Drop(0.1, n[:1]), Drop(0.1, n.int()), Drop(0.1, n.repeat(2)[::2]),
                Drop(0.1, torch.zeros(2, dtype=torch.int64, device="meta"))):
        for call in (lambda: dropout.dropout(x, bad), lambda: dropout.dropout_add(x, x, bad), lambda: norm.add_layernorm(x, x, dropout=bad),
                     lambda: norm.add_rmsnorm(x, x, x[0], 1e-5, bad)):
            with pytest.raises(RuntimeError, match="dropped|32 bits|int64"):
                call()
    for call in (lambda: norm.layernorm(x.float()), lambda: norm.layernorm(x[0]), lambda: norm.add_layernorm(x, x[:2]), lambda: norm.add_layernorm(x, x.float()),
                 lambda: dropout.dropout(x.float(), Drop(0.1, n)), lambda: dropout.dropout_add(x, x[:2], Drop(0.1, n))):
        with pytest.raises(RuntimeError, match="bf16|same shape|leading dimension"):
            call()


def test_rotary_axes_arguments_are_refused():
    from lingua_amd import rope
    q, cos, pos = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16), torch.zeros(4, 8), torch.zeros(3, 1, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="layout"):
        rope.rotary_axes(q, q, cos, cos, pos, (4, 2, 2), layout="whole")
    with pytest.raises(RuntimeError, match="order"):
        rope.rotary_axes(q, q, cos, cos, pos, (4, 2, 2), order="turns")
    with pytest.raises(RuntimeError, match="order|shares"):
        rope.pair_axes((4, -1))
    with pytest.raises(RuntimeError, match="length"):
        rope.axes_tables((4, 4), -1)


def test_no_cpu_path():
    from lingua_amd import adapters, dropout, norm, rope
    x, n = torch.zeros(4, 64, dtype=torch.bfloat16), dropout.numbers(1, "cpu")
    drop = dropout.Drop(0.1, n)
    for call in (lambda: norm.layernorm(x), lambda: norm.add_layernorm(x, x), lambda: norm.add_layernorm(x, x, dropout=drop), lambda: norm.add_rmsnorm(x, x, x[0], 1e-5, drop),
                 lambda: dropout.dropout(x, drop), lambda: dropout.dropout_add(x, x, drop), lambda: norm.Fp8LayerNorm(64)(x), lambda: dropout.Dropout(0.1, n)(x),
                 lambda: rope.rotary_axes(x.view(1, 4, 1, 64), x.view(1, 4, 1, 64), torch.zeros(4, 32), torch.zeros(4, 32), torch.zeros(2, 1, 4).long(), (16, 16)),
                 lambda: adapters.add_lowrank(x, x, torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(4).int())):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_seed_is_any_64_bits():
    from lingua_amd import dropout
    for seed in (0, 1, -1, 2 ** 63, 2 ** 64 - 1, 2 ** 64 + 5):
        assert int(dropout.numbers(seed, "cpu")[0]) % 2 ** 64 == seed % 2 ** 64
