"""A cast of the layer leaves what the scan takes in float32 as it is."""
import copy

import pytest
import torch
from torch import nn

WIDE = ("A_log", "skip", "step_bias")


def _layer(**like):
    from rnn_kernel_amd import SelectiveScan

    torch.manual_seed(0)
    return SelectiveScan(8, states=3, **like)


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: m.half(), lambda m: m.double(), lambda m: m.type(torch.bfloat16)])
def test_casts(cast):
    model = nn.Sequential(nn.Linear(4, 8), _layer())
    for p in model.parameters():
        p.grad = torch.full_like(p, 0.3)
    before = copy.deepcopy(model[1])
    ids = [id(p) for p in model.parameters()]
    cast(model)
    new = model[0].weight.dtype
    assert new != torch.float32 and [id(p) for p in model.parameters()] == ids
    for name, p in model[1].named_parameters():
        old = before.get_parameter(name)
        assert p.dtype == p.grad.dtype == (torch.float32 if name in WIDE else new), name
        assert torch.equal(p, old.to(p.dtype)) and torch.equal(p.grad, torch.full_like(old, 0.3).to(p.dtype)) and p.requires_grad


def test_moves_and_copies():
    layer = _layer()
    layer.to(torch.bfloat16).to(torch.float32)
    assert all(p.dtype == torch.float32 for p in layer.parameters())
    other = copy.deepcopy(layer).to("meta", torch.bfloat16)
    for name, p in other.named_parameters():
        assert p.is_meta and p.dtype == (torch.float32 if name in WIDE else torch.bfloat16), name
    other.to_empty(device="cpu")
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.A_log, layer.A_log) and other.A_log.dtype == torch.float32


@pytest.mark.gpu
def test_a_cast_layer_is_one_made_of_that_type(gpu):
    cast = _layer().to(gpu).to(torch.bfloat16)
    made = _layer(dtype=torch.bfloat16, device=gpu)
    made.load_state_dict(cast.state_dict())
    x = torch.randn(2, 5, 8, device=gpu, dtype=torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(cast.state_dict().values(), made.state_dict().values()))
    for a, b in zip(cast(x), made(x)):
        assert torch.equal(a, b) if torch.is_tensor(a) else all(map(torch.equal, a, b))
    states = [m.new_states(2) for m in (cast, made)]
    assert torch.equal(cast.step(x[:, 0], states[0]), made.step(x[:, 0], states[1]))
    assert all(map(torch.equal, *states))
