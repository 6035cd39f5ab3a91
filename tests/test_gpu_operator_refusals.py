"""What the gated delta rule and the matrix product refuse of GPU tensors: every case
ends in a Python exception before a launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(gpu, T=3):
    q, k = torch.randn(2, T, 1, 4, device=gpu), torch.randn(2, T, 1, 4, device=gpu)
    return [q, k, torch.randn(2, T, 2, 5, device=gpu), -torch.rand(2, T, 2, device=gpu), torch.rand(2, T, 2, device=gpu)]


def _with(args, i, t):
    return [t if j == i else a for j, a in enumerate(args)]


def test_rule_refuses(gpu):
    from rnn_kernel_amd import gated_delta_rule

    a = _inputs(gpu)
    for i, t, error, message in (
            (2, a[2].cpu(), RuntimeError, "v must be a CUDA/HIP tensor"), (1, a[1].bfloat16(), RuntimeError, "all float32 or all"),
            (3, a[3].bfloat16(), RuntimeError, "g and beta must be"), (3, a[3].double(), RuntimeError, "g and beta must be"),
            (0, a[0][0], ValueError, "q must have shape"), (1, a[1][..., :3], ValueError, "same shape"),
            (2, a[2][:, :2], ValueError, "batch and token"), (4, a[4][..., :1], ValueError, "g and beta must have v's shape")):
        with pytest.raises(error, match=message):
            gated_delta_rule(*_with(a, i, t))
    with pytest.raises(ValueError, match="multiple of q's"):
        gated_delta_rule(a[0].expand(2, 3, 3, 4), a[1].expand(2, 3, 3, 4), *a[2:])
    wide = torch.randn(2, 3, 1, 257, device=gpu)
    with pytest.raises(ValueError, match=r"key dim must be in \[1, 256\]"):
        gated_delta_rule(wide, wide, *a[2:])
    with pytest.raises(ValueError, match="initial_state must have shape"):
        gated_delta_rule(*a, torch.zeros(2, 2, 5, 4, device=gpu))
    with pytest.raises(RuntimeError, match="initial_state must be float32"):
        gated_delta_rule(*a, torch.zeros(2, 2, 4, 5, device=gpu, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="lengths must be an int32"):
        gated_delta_rule(*a, lengths=torch.tensor([1, 2], device=gpu))
    with pytest.raises(ValueError, match="lengths must have shape"):
        gated_delta_rule(*a, lengths=torch.ones(3, device=gpu, dtype=torch.int32))


def test_step_refuses(gpu):
    from rnn_kernel_amd import gated_delta_step

    a = [t[:, 0] for t in _inputs(gpu)]
    state = torch.zeros(3, 2, 4, 5, device=gpu)
    with pytest.raises(ValueError, match="fewer states"):
        gated_delta_step(*a, state[:1])
    with pytest.raises(ValueError, match="state must be contiguous"):
        gated_delta_step(*a, torch.zeros(3, 2, 5, 4, device=gpu).transpose(2, 3))
    with pytest.raises(ValueError, match="state must have shape"):
        gated_delta_step(*a, state[:, :1])
    with pytest.raises(RuntimeError, match="state must be float32"):
        gated_delta_step(*a, state.bfloat16())
    with pytest.raises(RuntimeError, match="state must be on"):
        gated_delta_step(*a, state.cpu())
    with pytest.raises(RuntimeError, match="slots must be an int32"):
        gated_delta_step(*a, state, slots=torch.tensor([0, 1], device=gpu))
    with pytest.raises(RuntimeError, match="has no gradients"):
        gated_delta_step(a[0].requires_grad_(True), *a[1:], state)


def test_linear_refuses(gpu):
    from rnn_kernel_amd import linear

    x, w, b, r = (torch.randn(*s, device=gpu) for s in ((5, 4), (3, 4), (3,), (5, 3)))
    for args, kw, error, message in (
            ((x, w.cpu()), {}, RuntimeError, "weight must be a CUDA/HIP tensor"), ((x, w.bfloat16()), {}, RuntimeError, "all float32"),
            ((x.double(), w.double()), {}, RuntimeError, "all float32"), ((x, w[:, :3]), {}, ValueError, "x must have shape"),
            ((x, w[0]), {}, ValueError, "weight must have shape"), ((x, w, b[:2]), {}, ValueError, "bias must have shape"),
            ((x, w, b), dict(residual=r[:4]), ValueError, "residual must have shape"),
            ((x, w, b), dict(residual=r[0]), ValueError, "residual must have shape"),
            ((x, w, b), dict(activation="tanh"), ValueError, "activation must be one of")):
        with pytest.raises(error, match=message):
            linear(*args, **kw)


def test_second_gradients_are_refused(gpu):
    from rnn_kernel_amd import gated_delta_rule, linear

    x, w = torch.randn(5, 4, device=gpu, requires_grad=True), torch.randn(3, 4, device=gpu)
    (dx,) = torch.autograd.grad(linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    a = _inputs(gpu)
    a[2].requires_grad_(True)
    (dv,) = torch.autograd.grad(gated_delta_rule(*a)[0].sum(), a[2], create_graph=True)
    with pytest.raises(RuntimeError):
        dv.sum().backward()
