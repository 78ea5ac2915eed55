"""CPU: which layers ``fp8_convert`` and ``fp8_activations`` take, with stand-ins for the layers that need a GPU."""
import pytest
import torch

import neuzip_amd
from neuzip_amd import nn


class Held:
    def write(self, data):
        return "0"


class Holder(torch.nn.Module):
    def __init__(self, **children):
        super().__init__()
        for name, child in children.items():
            setattr(self, name, child)


def linear():
    return torch.nn.Linear(4, 4)


@pytest.mark.parametrize("block_rows", (1, 128))
def test_layers_that_are_converted(monkeypatch, block_rows):
    class Taken(torch.nn.Module):
        def __init__(self, linear, block_rows):
            super().__init__()
            self.block_rows = block_rows

    monkeypatch.setattr(nn, "FP8Linear", Taken)
    shared, head = linear(), linear()
    model = Holder(a=shared, block=Holder(b=shared, c=linear()), lm_head=head, tied=head)
    assert neuzip_amd.fp8_convert(model, block_rows=block_rows) is model
    assert isinstance(model.a, Taken) and model.block.b is model.a and model.block.c.block_rows == block_rows
    assert model.lm_head is head and model.tied is head and shared.weight is None


def test_what_keeps_8_bits():
    block = Holder(q=nn.Linear(Held(), linear()), fc=nn.Linear(Held(), linear()), act=torch.nn.GELU(),
                   tanh=torch.nn.GELU(approximate="tanh"), dense=linear())
    model = Holder(block=block, silu=torch.nn.SiLU(inplace=True), relu=torch.nn.ReLU())
    assert block.fc.saved_bits == 16 and "saved_bits" not in repr(block.fc)
    assert neuzip_amd.fp8_activations(model, skip=("q",)) is model
    assert block.q.saved_bits == 16 and block.fc.saved_bits == 8 and "saved_bits=8" in repr(block.fc)
    assert (block.act.kind, block.tanh.kind, model.silu.kind) == ("gelu", "gelu_tanh", "silu")
    assert isinstance(model.relu, torch.nn.ReLU) and type(block.dense) is torch.nn.Linear
    neuzip_amd.fp8_activations(model)
    assert block.q.saved_bits == 8 and block.act.kind == "gelu"


def test_one_name_to_skip():
    """a text is one mark, not a mark for each of its letters"""
    block = Holder(q_proj=nn.Linear(Held(), linear()), o=nn.Linear(Held(), linear()), act=torch.nn.GELU())
    neuzip_amd.fp8_activations(Holder(block=block), skip="q_proj")
    assert (block.q_proj.saved_bits, block.o.saved_bits) == (16, 8) and isinstance(block.act, nn.FP8Activation)
    for nothing in ("", (), None):
        block = Holder(q_proj=nn.Linear(Held(), linear()))
        neuzip_amd.fp8_activations(Holder(block=block), skip=nothing)
        assert block.q_proj.saved_bits == 8
