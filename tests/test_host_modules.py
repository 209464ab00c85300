"""What the modules of dropout and adapters do with a model's structure: no GPU needed."""
import copy
import io

import pytest
import torch

from lingua_amd import adapters, dropout, rope


class Twice(torch.nn.Module):
    """A dropout that is called twice in a forward pass, and one that is called once."""

    def __init__(self):
        super().__init__()
        self.drop, self.last = torch.nn.Dropout(0.1), torch.nn.Dropout(0.2)

    def forward(self, fail=False):
        sites = [self.drop.drop().site, self.last.drop().site, self.drop.drop().site]
        if fail:
            raise ValueError
        return sites


def test_calls_of_a_forward_pass_drop_other_elements():
    """And a forward pass that is repeated drops the same again, also one behind a pass that ended early, and in a copy of the model."""
    numbers = dropout.numbers(1, "cpu")
    model = dropout.convert_dropouts(Twice(), numbers)
    want = [0, 1, 1 << 20]
    assert model() == want and model() == want
    with pytest.raises(ValueError):
        model(fail=True)
    assert model() == want
    other = copy.deepcopy(model)
    assert other() == want and other.drop._pass is not model.drop._pass and other.drop.numbers is not numbers
    buffer = io.BytesIO()
    torch.save(model, buffer)
    assert torch.load(io.BytesIO(buffer.getvalue()), weights_only=False)() == want
    # outside a pass nothing is counted
    assert [model.drop.drop().site for _ in range(3)] == [0, 0, 0]
    model.eval()
    assert model.drop.drop() is None


def test_shared_parents():
    """A block that stands at two places: one dropout, whose calls are told apart where the model has a forward pass, and refused where it has
    none."""
    block = torch.nn.Sequential(torch.nn.Identity(), torch.nn.Dropout(0.1))

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.first, self.second = block, block

        def forward(self):
            return [part[1].drop().site for part in (self.first, self.second)]

    with pytest.raises(RuntimeError, match="several places of a ModuleList"):
        dropout.convert_dropouts(torch.nn.ModuleList([block, block]), dropout.numbers(1, "cpu"))
    assert type(block[1]) is torch.nn.Dropout
    model = dropout.convert_dropouts(Model(), dropout.numbers(1, "cpu"))
    assert model.first[1] is model.second[1] and model() == [0, 1 << 20]


def test_sites_that_are_taken():
    """By modules made by hand, also as a later call of a lower site."""
    n = dropout.numbers(1, "cpu")
    model = torch.nn.ModuleList([dropout.Dropout(0.1, n, 0), dropout.Dropout(0.1, n, (5 << 20) + 1), torch.nn.Dropout(0.3), torch.nn.Dropout(0.3)])
    dropout.convert_dropouts(model, n)
    assert [m.site for m in model] == [0, (5 << 20) + 1, 2, 3]

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.drop = torch.nn.Dropout(0.5)

        def forward(self, times):
            return [self.drop.drop().site for _ in range(times)]

    model = dropout.convert_dropouts(Model(), n)
    assert model(4096) == [k << 20 for k in range(4096)]
    with pytest.raises(RuntimeError, match="4096"):
        model(4097)
    model.drop.site = 1 << 20
    with pytest.raises(RuntimeError, match="sites below"):
        model(2)


def test_a_scale_that_asks_for_a_gradient_is_refused():
    """It would learn nothing."""
    y, x = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    a, b, index = torch.zeros(2, 8, 32, dtype=torch.bfloat16), torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    scale = torch.ones(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="scale asks for a gradient"):
        adapters.add_lowrank(y, x, a, b, index, scale)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):    # (without gradients it is as good as any)
        adapters.add_lowrank(y, x, a, b, index, scale)


def test_tables_that_ask_for_a_gradient_are_refused():
    """Of positions on several axes: they would learn nothing."""
    q, pos = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16), torch.zeros(3, 1, 2, dtype=torch.int64)
    table, learnt = torch.zeros(4, 8), torch.zeros(4, 8, requires_grad=True)
    for cos, sin in ((learnt, table), (table, learnt)):
        with pytest.raises(RuntimeError, match="tables ask for a gradient"):
            rope.rotary_axes(q, q, cos, sin, pos, (4, 2, 2))


def test_a_linear_at_several_places():
    """A bank at each place, also below one parent; one in a shared parent has one."""
    lin = torch.nn.Linear(16, 16, bias=False)
    model = torch.nn.ModuleDict({"stack": torch.nn.Sequential(lin, torch.nn.ReLU(), lin), "other": lin, "none": None})
    block = torch.nn.Sequential(torch.nn.Linear(16, 16))
    model["a"], model["b"] = block, block
    requests = adapters.Requests(2)
    for _ in range(2):      # (and not one in another)
        adapters.add_adapters(model, requests, 8, "")
        banks = [model["stack"][0], model["stack"][2], model["other"]]
        assert all(type(m) is adapters.AdaptedLinear and m.linear is lin for m in banks) and len({id(m) for m in banks}) == 3
        assert type(block[0]) is adapters.AdaptedLinear and type(block[0].linear) is torch.nn.Linear and model["a"][0] is model["b"][0]
    assert model["none"] is None


def test_a_linear_that_has_a_bank_already():
    model = adapters.add_adapters(torch.nn.Linear(16, 16), adapters.Requests(2), 8, "")
    assert adapters.add_adapters(model, model.requests, 8, "") is model and type(model.linear) is torch.nn.Linear


def test_a_filter_that_names_no_linear_is_refused():
    model = torch.nn.ModuleDict({"w1": torch.nn.Linear(16, 16), "norm": torch.nn.LayerNorm(16)})
    for match in ("w2", "norm", "w1.weight"):
        with pytest.raises(RuntimeError, match="names no linear"):
            adapters.add_adapters(model, adapters.Requests(2), 8, match)
    assert type(model["w1"]) is torch.nn.Linear


def test_a_fused_feed_forward_at_several_places_is_refused():
    """By any of its names."""
    from lingua_amd import swiglu
    fused = swiglu.Fp8FeedForward(*(torch.nn.Linear(*s, bias=False, dtype=torch.bfloat16) for s in ((32, 64), (32, 64), (64, 32))))
    model = torch.nn.ModuleDict({"first": fused, "second": fused})
    for match in ("first.w1", "second.w2"):
        with pytest.raises(RuntimeError, match="fused feed-forward"):
            adapters.add_adapters(model, adapters.Requests(2), 8, match)
    assert type(fused.w2) is torch.nn.Linear


def test_modules_that_were_pickled_before_their_calls_were_counted():
    model = dropout.convert_dropouts(Twice(), dropout.numbers(1, "cpu"))
    requests = adapters.Requests(2)
    for thing in (model.drop, requests):
        for name in ("_pass", "_calls", "_several", "_version", "_read"):
            thing.__dict__.pop(name, None)
    assert model.drop.drop().site == 0 and requests.plan is None
