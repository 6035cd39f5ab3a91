"""Forward-mode tangents are refused: the operators have no forward-mode derivative, and a
result without a tangent would be a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad

MESSAGE = "no forward-mode derivative"


def _calls(device):
    """(call, its tensors) of each operator."""
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step, linear

    q, k, v = (torch.randn(2, 3, h, d, device=device) for h, d in ((1, 4), (1, 4), (2, 5)))
    gates = [torch.rand(2, 3, 2, device=device) for _ in range(2)]
    s = torch.randn(2, 2, 4, 5, device=device)
    yield gated_delta_rule, [q, k, v, *gates, s]
    yield gated_delta_step, [t[:, 0] for t in (q, k, v, *gates)] + [s.clone()]
    x, w, b, r = (torch.randn(*n, device=device) for n in ((6, 4), (3, 4), (3,), (6, 3)))
    yield lambda *a: linear(*a[:3], residual=a[3]), [x, w, b, r]


def _refuses(device):
    for call, tensors in _calls(device):
        with forward_ad.dual_level():
            for i, t in enumerate(tensors):
                args = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else u for j, u in enumerate(tensors)]
                with pytest.raises(RuntimeError, match=MESSAGE):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError, match=MESSAGE):
                    call(*args)


def test_tangents_are_refused():
    _refuses("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu(gpu):
    _refuses(gpu)
    for call, tensors in _calls(gpu):  # tensors without tangents are taken at a dual level too
        with forward_ad.dual_level():
            call(*tensors)
