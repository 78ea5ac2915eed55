"""CPU: which layers ``mx_convert`` takes, with a stand-in for the layer that needs a GPU."""
import pytest
import torch

import neuzip_amd


class Taken(torch.nn.Module):
    def __init__(self, linear):
        super().__init__()
        self.size = tuple(linear.weight.shape)


@pytest.fixture(autouse=True)
def stand_in(monkeypatch):
    monkeypatch.setattr(neuzip_amd.nn, "MXLinear", Taken)


class Holder(torch.nn.Module):
    def __init__(self, **children):
        super().__init__()
        for name, child in children.items():
            setattr(self, name, child)


@pytest.mark.parametrize("order", (("proj", "lm_head"), ("lm_head", "proj")))
@pytest.mark.parametrize("deep", (False, True))
def test_a_head_that_stands_under_another_name_is_left_alone(order, deep):
    head, other = torch.nn.Linear(4, 6), torch.nn.Linear(4, 4)
    places = {"proj": Holder(inner=head, up=other) if deep else head, "lm_head": head}
    model = neuzip_amd.mx_convert(Holder(rest=other, **{name: places[name] for name in order}))
    assert model.lm_head is head and head.weight is not None and head(torch.zeros(1, 4)).shape == (1, 6)
    assert (model.proj.inner if deep else model.proj) is head
    assert isinstance(model.rest, Taken) and other.weight is None
    assert not deep or model.proj.up is model.rest


def test_a_head_of_several_layers_is_left_alone_wherever_they_stand():
    inner, free = torch.nn.Linear(4, 4), torch.nn.Linear(4, 5)
    model = Holder(body=Holder(a=inner, b=free), lm_head=torch.nn.Sequential(inner, torch.nn.Linear(4, 7)))
    neuzip_amd.mx_convert(model)
    assert model.body.a is inner and model.lm_head[0] is inner and inner.weight is not None
    assert isinstance(model.lm_head[1], torch.nn.Linear) and isinstance(model.body.b, Taken)


def test_layers_in_several_places_and_modules_that_hold_each_other():
    shared = torch.nn.Linear(3, 3)
    block = Holder(a=shared)
    model = Holder(x=block, y=block, z=Holder(a=shared), none=None)
    model.none = None
    model.back = Holder(block=block)
    neuzip_amd.mx_convert(model)
    assert isinstance(block.a, Taken) and model.z.a is block.a and model.back.block.a is block.a
