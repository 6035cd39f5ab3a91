"""The exponentials of float32 calls element by element, far from 0 too, where a rounded exponent
would cost bits: SiLU of the convolution and of the scan's gate, their slopes, and small steps.

Tolerances, of each element, by arithmetic: an exponential 2^-23, 1 + it 2^-24 and the
exponential's own, a division and a product 2^-24 each: 5 * 2^-24.  The slope s (1 + z (1 - s)): s
4 * 2^-24; for z <= -3, where s is below 1/20, z (1 - s) three roundings and s's, of which 1 +
leaves at most 3/2; two more products: 13 * 2^-24.  For z >= 3 s is next to 1, off by two roundings
or 2 * 2^-24, and 1 - s (a difference without rounding) by as much in absolute terms; z times that,
beside a result of 1 or more: (2 z + 8) * 2^-24 with the roundings of the products and sums, as in any
float32 arithmetic of this formula.  softplus far below 0: an exponential, a logarithm, a product of
them and the sum: 4 * 2^-23."""
import pytest
import torch

pytestmark = pytest.mark.gpu

VALUE, STEP = 5 * 2.0 ** -24, 4 * 2.0 ** -23


def _z(least, device):
    gen = torch.Generator().manual_seed(5)
    low = -80 + (80 - least) * torch.rand(4000, generator=gen)
    return torch.cat([low, least + 20 * torch.rand(1000, generator=gen)]).to(device)


def _silu(z):
    z = z.double()
    return z * torch.sigmoid(z)


def _slope(z):
    s = torch.sigmoid(z.double())
    return s * (1 + z.double() * torch.sigmoid(-z.double()))


def _slopes_fit(a, z):
    off = (a.double() / _slope(z) - 1).abs()
    return bool((off <= torch.where(z < 0, 13, 2 * z + 8) * 2.0 ** -24).all())


def _off(a, ref):
    return float((a.double() / ref - 1).abs().max())


def test_silu_of_the_convolution(gpu):
    from rnn_kernel_amd import causal_conv, causal_conv_step

    z = _z(3, gpu)
    w = torch.tensor([[0.0, 1.0]], device=gpu).expand(z.numel(), 2)
    x = z.view(1, 1, -1).clone().requires_grad_(True)
    y = causal_conv(x, w, activation="silu")[0]
    dx = torch.autograd.grad(y.sum(), x)[0]
    assert _off(y.detach().view(-1), _silu(z)) <= VALUE and _slopes_fit(dx.view(-1), z)
    state = torch.zeros(1, 1, z.numel(), device=gpu)
    with torch.no_grad():
        assert torch.equal(causal_conv_step(z.view(1, -1), state, w, activation="silu").view(-1), y.view(-1))


def test_silu_of_the_gate(gpu):
    """(B and C are 0: y = skip x silu(gate).)"""
    from rnn_kernel_amd import selective_scan, selective_step

    z = _z(3, gpu)
    n = z.numel()
    one, none, A = torch.ones(1, 1, n, device=gpu), torch.zeros(1, 1, 1, 2, device=gpu), -torch.ones(n, 2, device=gpu)
    skip, gate = torch.ones(n, device=gpu), z.view(1, 1, -1).clone().requires_grad_(True)
    x = one.clone().requires_grad_(True)
    y = selective_scan(x, one, A, none, none, skip=skip, gate=gate)[0]
    dx, dgate = torch.autograd.grad(y.sum(), [x, gate])
    assert _off(y.detach().view(-1), _silu(z)) <= VALUE and _off(dx.view(-1), _silu(z)) <= VALUE
    assert _slopes_fit(dgate.view(-1), z)
    with torch.no_grad():
        step = selective_step(one[0], one[0], A, none[0], none[0], torch.zeros(1, n, 2, device=gpu), skip=skip, gate=gate[0])
    assert torch.equal(step.view(-1), y.view(-1))


def test_small_steps(gpu):
    """A state of one token is the step: softplus(dt), and its gradient sigmoid(dt)."""
    from rnn_kernel_amd import selective_scan, selective_step

    z = -12 - 68 * torch.rand(4000, generator=torch.Generator().manual_seed(6)).to(gpu)
    n = z.numel()
    one, A = torch.ones(1, 1, n, device=gpu), -torch.ones(n, 1, device=gpu)
    unit = torch.ones(1, 1, 1, 1, device=gpu)
    dt = z.view(1, 1, -1).clone().requires_grad_(True)
    h = selective_scan(one, dt, A, unit, unit, softplus=True)[1]
    grad = torch.autograd.grad(h.sum(), dt)[0]
    assert _off(h.detach().view(-1), torch.log1p(z.double().exp())) <= STEP
    assert _off(grad.view(-1), torch.sigmoid(z.double())) <= STEP
    pool = torch.zeros(1, n, 1, device=gpu)
    with torch.no_grad():
        selective_step(one[0], dt[0], A, unit[0], unit[0], pool, softplus=True)
    assert torch.equal(pool.view(-1), h.view(-1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_is_not_finite_or_far(gpu, dtype):
    """As the formulas have it: silu(inf) = inf, of -inf and NaN NaN, of -1e30 0; steps inf, 0 and NaN."""
    from rnn_kernel_amd import causal_conv, selective_scan

    z = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e30, -1e30, 300.0, -300.0, 0.0, -0.0], device=gpu).to(dtype)
    n = z.numel()
    want = torch.nan_to_num(_silu(z).to(dtype).double(), nan=7.0)
    w = torch.ones(n, 2, device=gpu, dtype=dtype)
    y = causal_conv(z.view(1, 1, -1), w, activation="silu")[0]
    one, none, A = torch.ones(1, 1, n, device=gpu, dtype=dtype), torch.zeros(1, 1, 1, 2, device=gpu, dtype=dtype), -torch.ones(n, 2, device=gpu)
    gated = selective_scan(one, one, A, none, none, skip=torch.ones(n, device=gpu), gate=z.view(1, 1, -1))[0]
    for got in (y, gated):
        assert torch.equal(torch.nan_to_num(got.view(-1).double(), nan=7.0), want)
    unit = torch.ones(1, 1, 1, 1, device=gpu, dtype=dtype)
    h = selective_scan(one, z.view(1, 1, -1), A[:, :1], unit, unit, softplus=True)[1].view(-1).double()
    z = z.double()
    s = torch.where(z > 0, z, 0 * z.clamp(-1, 1)) + torch.log1p((-z.abs()).exp())
    assert torch.equal(h.isnan(), s.isnan()) and torch.equal(h.isinf(), s.isinf())
    rest = torch.isfinite(s)
    assert ((h - s)[rest].abs() <= STEP * s[rest].abs() + 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_below_0_everywhere(gpu, dtype):
    """Where exp(-z) is no float32 (z below -88.7), and next to it: silu and its slope are below 2^-115 there,
    and no NaN; steps of as much are the number itself, or 0."""
    from rnn_kernel_amd import causal_conv, causal_conv_step, selective_scan, selective_step

    z = torch.cat([torch.linspace(-400, -87, 20001), -torch.logspace(2, 38, 5001)]).to(gpu, dtype)
    n = z.numel()
    w = torch.tensor([[0.0, 1.0]], device=gpu, dtype=dtype).expand(n, 2)
    x = z.view(1, 1, -1).clone().requires_grad_(True)
    y = causal_conv(x, w, activation="silu")[0]
    found = [y, torch.autograd.grad(y.sum(), x)[0]]
    one, none = torch.ones(1, 1, n, device=gpu, dtype=dtype), torch.zeros(1, 1, 1, 2, device=gpu, dtype=dtype)
    A, skip = -torch.ones(n, 2, device=gpu), torch.ones(n, device=gpu)
    v, gate = one.clone().requires_grad_(True), z.view(1, 1, -1).clone().requires_grad_(True)
    y = selective_scan(v, one, A, none, none, skip=skip, gate=gate)[0]
    found += [y, *torch.autograd.grad(y.sum(), [v, gate])]
    with torch.no_grad():
        found.append(causal_conv_step(z.view(1, -1), torch.zeros(1, 1, n, device=gpu, dtype=dtype), w, activation="silu"))
        found.append(selective_step(one[0], one[0], A, none[0], none[0], torch.zeros(1, n, 2, device=gpu), skip=skip, gate=z.view(1, -1)))
    for t in found:
        assert (t.abs() <= 2.0 ** -115).all()
    unit = torch.ones(1, 1, 1, 1, device=gpu, dtype=dtype)
    for sign in (1, -1):
        raw = (sign * z).view(1, 1, -1).clone().requires_grad_(True)
        h = selective_scan(one, raw, A[:, :1], unit, unit, softplus=True)[1].view(-1)
        (grad,) = torch.autograd.grad(h.sum(), raw)
        want, slope = (torch.zeros_like(z), 0.0) if sign > 0 else (-z, 1.0)
        assert ((h - want.float()).abs() <= 2.0 ** -115).all() and ((grad.float() - slope).abs() <= 2.0 ** -115).all()
