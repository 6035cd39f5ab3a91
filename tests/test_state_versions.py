"""A single step changes its states in place, and autograd is told."""
import pytest
import torch


def _inputs(device="cpu"):
    q, k, v = (torch.randn(2, h, d, device=device) for h, d in ((1, 4), (1, 4), (2, 5)))
    return [q, k, v, -torch.rand(2, 2, device=device), torch.rand(2, 2, device=device)]


def test_a_step_counts_as_a_change_of_the_states(hip_lib, monkeypatch):
    """(The library's call is left out: this runs without a GPU.)"""
    from rnn_kernel_amd import delta

    monkeypatch.setattr(delta._lib, "call", lambda *a: None)
    monkeypatch.setattr(delta, "_check_inputs", lambda *a, **k: None)
    monkeypatch.setattr(delta, "_check_state", lambda *a, **k: None)
    state = torch.randn(2, 2, 4, 5)
    before = state._version
    delta.gated_delta_step(*_inputs(), state)
    assert state._version > before
    with torch.inference_mode():  # where nothing is counted
        delta.gated_delta_step(*_inputs(), torch.randn(2, 2, 4, 5))


@pytest.mark.gpu
def test_a_graph_that_saved_the_states_is_told(gpu):
    from rnn_kernel_amd import GatedDelta, gated_delta_step

    state = torch.randn(2, 2, 4, 5, device=gpu)
    w = torch.ones((), device=gpu, requires_grad=True)
    y = (w * state).sum()
    gated_delta_step(*_inputs(gpu), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    layer = GatedDelta(8, 2, 4, 5, device=gpu)
    pool = layer.new_states(3)
    y = (w * pool).sum()
    layer.step(torch.randn(2, 8, device=gpu), pool)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
