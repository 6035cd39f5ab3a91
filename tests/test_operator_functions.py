"""The operators' autograd functions, applied directly, refuse what the operators refuse."""
import pytest
import torch


def _rule_inputs():
    return [torch.randn(2, 3, 1, 4), torch.randn(2, 3, 1, 4), torch.randn(2, 3, 2, 5), -torch.rand(2, 3, 2), torch.rand(2, 3, 2)]


def test_functions_refuse_cpu_tensors():
    from rnn_kernel_amd import GatedDeltaFunction, LinearFunction

    with pytest.raises(RuntimeError, match="q must be a CUDA/HIP tensor"):
        GatedDeltaFunction.apply(*_rule_inputs(), None, None, None, False)
    with pytest.raises(RuntimeError, match="x must be a CUDA/HIP tensor"):
        LinearFunction.apply(torch.randn(2, 4), torch.randn(3, 4), None, None, "silu")


@pytest.mark.gpu
def test_functions_refuse_shapes_and_take_any_layout(gpu):
    """Refusals end before a launch; what the operators copy, the functions copy."""
    from rnn_kernel_amd import GatedDeltaFunction, LinearFunction, gated_delta_rule, linear

    a = [t.to(gpu) for t in _rule_inputs()]
    with pytest.raises(ValueError, match="same shape"):
        GatedDeltaFunction.apply(a[0][..., :3], *a[1:], None, None, None, False)
    with pytest.raises(ValueError, match="initial_state must have shape"):
        GatedDeltaFunction.apply(*a, torch.zeros(1, 2, 4, 5, device=gpu), None, None, False)
    with pytest.raises(ValueError, match="lengths must have shape"):
        GatedDeltaFunction.apply(*a, None, torch.ones(3, dtype=torch.int32, device=gpu), None, False)
    x, w = torch.randn(6, 4, device=gpu), torch.randn(3, 4, device=gpu)
    with pytest.raises(ValueError, match="x must have shape"):
        LinearFunction.apply(x[:, :3], w, None, None, None)
    with pytest.raises(ValueError, match="activation must be one of"):
        LinearFunction.apply(x, w, None, None, "tanh")
    apart = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in a[:3]]
    assert apart[2].stride(-1) != 1
    state = torch.randn(2, 2, 5, 4, device=gpu).transpose(2, 3)
    for t in (*a, *apart, state):
        t.requires_grad_(True)
    got = GatedDeltaFunction.apply(*apart, *a[3:], state, None, None, True)
    want = gated_delta_rule(*a, state, normalize=True)
    up = [torch.randn_like(t) for t in want]
    for p, q in zip((*got, *torch.autograd.grad(got, [*apart, *a[3:], state], up)),
                    (*want, *torch.autograd.grad(want, [*a, state], up))):
        assert torch.equal(p, q)
    assert torch.equal(LinearFunction.apply(x, w, None, None, "relu"), linear(x, w, activation="relu"))
