"""What the backward passes hand to the library after saved-tensor hooks have given the
tensors back in another layout: the unpacked tensors' addresses with their own strides.
Runs without a GPU: the library's calls are recorded, not made."""
import importlib

import pytest
import torch


def _recorded(monkeypatch, module, checks):
    calls = {}
    monkeypatch.setattr(module._lib, "call", lambda index, name, *args: calls.__setitem__(name, args))
    monkeypatch.setattr(module, "_index_of", lambda device: 0)
    for name in checks:
        monkeypatch.setattr(module, name, lambda *a, **k: None)
    return calls


class _Hooks:
    """Hands every saved tensor back as `change` of it, and keeps what it handed back."""

    def __init__(self, change):
        self.change, self.given = change, []

    def unpack(self, t):
        t = self.change(t)
        self.given.append(t)
        return t

    def __enter__(self):
        self.inner = torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), self.unpack)
        return self.inner.__enter__()

    def __exit__(self, *exc):
        return self.inner.__exit__(*exc)


def _apart(t):
    """The same values, neighbouring elements of the last dimension two apart."""
    return torch.stack([t, torch.zeros_like(t)], -1)[..., 0]


@pytest.mark.parametrize("change", [torch.Tensor.contiguous, torch.clone, _apart])
def test_the_rules_backward_goes_by_the_unpacked_tensors(hip_lib, monkeypatch, change):
    from rnn_kernel_amd import delta

    calls = _recorded(monkeypatch, delta, ("_check_inputs", "_check_state", "_check_ints"))
    B, T, Hk, Hv, Dk, Dv = 2, 5, 2, 4, 3, 6
    row = torch.randn(B, T, 2 * Hk * Dk + Hv * Dv)
    q, k, v = (t.unflatten(-1, (-1, d)) for t, d in zip(row.split([Hk * Dk, Hk * Dk, Hv * Dv], -1), (Dk, Dk, Dv)))
    g, beta = (torch.rand(B, T, 1).expand(B, T, Hv) for _ in range(2))
    lengths = torch.tensor([5, 2], dtype=torch.int32)
    v.requires_grad_(True)
    hooks = _Hooks(change)
    with hooks:
        o, _ = delta.GatedDeltaFunction.apply(q, k, v, g, beta, None, lengths, 1.0, False)
    o.sum().backward()
    args = calls["rka_gated_delta_backward"]
    strides = next(list(a) for a in args if hasattr(a, "_length_"))
    for at, t, group in ((0, q, 0), (1, k, 1), (2, g, 3), (3, beta, 4)):
        mine = strides[3 * group:3 * group + 3]
        given = [u for u in hooks.given if u.data_ptr() == args[at]]
        if given:  # as it came back, if a head's elements lie side by side in it
            assert tuple(mine) == given[0].stride()[:3]
            assert t.dim() == 3 or given[0].stride(-1) == 1
        else:  # a copy, which is dense
            assert change is _apart and tuple(mine) == t.contiguous().stride()[:3]
    if change is _apart:
        assert args[4] not in [u.data_ptr() for u in hooks.given]  # lengths
        assert args[5] not in [u.data_ptr() for u in hooks.given]  # what the forward saved


@pytest.mark.parametrize("change", [torch.Tensor.contiguous, _apart])
def test_the_products_backward_goes_by_the_unpacked_tensors(hip_lib, monkeypatch, change):
    linear = importlib.import_module("rnn_kernel_amd.linear")  # (the package's `linear` is the function)
    calls = _recorded(monkeypatch, linear, ("_check",))
    x, w = torch.randn(4, 9)[:, 2:7], torch.randn(3, 8)[:, :5].requires_grad_(True)
    hooks = _Hooks(change)
    with hooks:
        y = linear.LinearFunction.apply(x, w, None, None, "silu")
    y.sum().backward()
    args = calls["rka_linear_backward"]
    given = {u.data_ptr(): u for u in hooks.given}
    for at, cols in ((2, 5), (4, 5)):
        if args[at] in given:
            assert given[args[at]].stride() == (args[at + 1], 1)
        else:
            assert change is _apart and args[at + 1] == cols
    if change is _apart:
        assert args[6] not in given  # the sums before the activation


@pytest.mark.parametrize("change", [lambda t: t.to("meta"), lambda t: t.double() if t.is_floating_point() else t.long(),
                                    lambda t: t[:1] if t.size(0) > 1 else t])
def test_what_comes_back_as_something_else_is_refused(hip_lib, monkeypatch, change):
    """As torch's own operators refuse it: on another device, of another type or size."""
    from rnn_kernel_amd import delta

    linear = importlib.import_module("rnn_kernel_amd.linear")
    calls = _recorded(monkeypatch, delta, ("_check_inputs", "_check_state", "_check_ints"))
    _recorded(monkeypatch, linear, ("_check",))
    monkeypatch.setattr(linear._lib, "call", lambda index, name, *args: calls.__setitem__(name, args))
    q, k, v = (torch.randn(2, 3, h, d, requires_grad=True) for h, d in ((1, 4), (1, 4), (2, 5)))
    gates = [torch.rand(2, 3, 2) for _ in range(2)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), change):
        o, _ = delta.GatedDeltaFunction.apply(q, k, v, *gates, None, torch.tensor([3, 1], dtype=torch.int32), 1.0, False)
        y = linear.LinearFunction.apply(torch.randn(4, 5), torch.randn(3, 5, requires_grad=True), None, None, "silu")
    for t in (o, y):
        with pytest.raises(RuntimeError, match="saved tensor"):
            t.sum().backward()
    assert not any("backward" in name for name in calls)


@pytest.mark.parametrize("which", range(6))
def test_each_saved_tensor_of_the_rule_is_looked_at(hip_lib, monkeypatch, which):
    from rnn_kernel_amd import delta

    calls = _recorded(monkeypatch, delta, ("_check_inputs", "_check_state", "_check_ints"))
    seen = []

    def unpack(t):
        seen.append(t)
        return t.to("meta") if len(seen) == which + 1 else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
        o, _ = delta.GatedDeltaFunction.apply(torch.randn(2, 3, 1, 4), torch.randn(2, 3, 1, 4),
                                              torch.randn(2, 3, 2, 5, requires_grad=True), torch.rand(2, 3, 2),
                                              torch.rand(2, 3, 2), None, torch.tensor([3, 1], dtype=torch.int32), 1.0, False)
    with pytest.raises(RuntimeError, match="saved tensor"):
        o.sum().backward()
    assert len(seen) == 6 and "rka_gated_delta_backward" not in calls
