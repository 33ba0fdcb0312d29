"""The layer in 8-bit integers as a module of a network that is moved between types, without a GPU; its product after
such a move is compared on the GPU."""
import copy

import pytest
import torch

from yolo_amd import Int8Linear

MOVES = {"half": lambda m: m.half(), "bfloat16": lambda m: m.bfloat16(), "to": lambda m: m.to(torch.float16),
         "double": lambda m: m.double(), "type": lambda m: m.type(torch.float16), "twice": lambda m: m.half().float(),
         "both": lambda m: m.to(m[0].weight.device, torch.bfloat16)}


def _net(bias=True, dev="cpu"):
    gen = torch.Generator().manual_seed(0)
    weight = torch.randint(-127, 128, (10, 70), generator=gen, dtype=torch.int8)
    layer = Int8Linear(weight, 1e-3 * torch.rand(10, generator=gen), torch.randn(10, generator=gen) if bias else None)
    return torch.nn.Sequential(torch.nn.Linear(70, 70), layer).to(dev)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("move", list(MOVES))
def test_a_network_moved_to_another_type_keeps_the_layer(move, bias):
    net = _net(bias)
    before = copy.deepcopy(net[1].state_dict())
    assert MOVES[move](net) is net
    if move != "twice":
        assert net[0].weight.dtype != torch.float32
    assert list(net[1].state_dict()) == list(before)
    for name, kept in net[1].state_dict().items():
        assert kept.dtype == before[name].dtype and torch.equal(kept, before[name]), name
    assert (net[1].bias is None) == (not bias) and net[1].weight.stride(0) == 128


def test_moves_between_devices_still_move_the_layer():
    net = _net().to("meta", torch.float16)
    assert all(t.is_meta for t in net.state_dict().values())
    assert net[1].weight_scale.dtype == torch.float32 and net[1].weight_rows.dtype == torch.int8
    net = net.to_empty(device="cpu")
    assert not any(t.is_meta for t in net.state_dict().values())
    net.load_state_dict(_net().half().state_dict())
    assert torch.equal(net[1].weight_scale, _net()[1].weight_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("move", list(MOVES))
def test_the_product_stays_the_same(dev, move):
    net = _net(dev=dev)
    x = torch.randn(5, 70, generator=torch.Generator().manual_seed(1)).to(dev)
    want = net[1](x)
    assert torch.equal(MOVES[move](net)[1](x), want)
