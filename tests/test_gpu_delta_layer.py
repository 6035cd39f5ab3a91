"""GPU parity of the gated delta-rule layer with its formulas in float64, and its parts
used together: training, a prompt, answers token by token.

Tolerances, set before the first run, as 2-norms of the error over 2-norms of the result,
float32: the projections are off by 2^-24 (8 + 2 sqrt(40)) = 1.3e-6 at most, the rule by
2e-6 and by up to four times what each of its five inputs is off, the output's projection
by another 1.3e-6: 3e-5.  Gradients take the same way back: 6e-5; the decay's, whose terms
cancel, 3e-4.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

VALUE, GRAD, DECAY_GRAD = 3e-5, 6e-5, 3e-4


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double().cpu()
    assert a.shape == ref.shape and torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


def _oracle(layer, x, state, lengths, params):
    """The layer's formulas in float64 on the CPU, a token at a time."""
    keys, values = layer.key_heads * layer.key_dim, layer.value_heads * layer.value_dim
    B, T, _ = x.shape
    rep = layer.value_heads // layer.key_heads
    q, k, v = F.silu(x @ params["project.weight"].t()).split([keys, keys, values], dim=-1)
    q, k = (t.reshape(B, T, layer.key_heads, layer.key_dim) for t in (q, k))
    q, k = ((t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(rep, 2) for t in (q, k))
    v = v.reshape(B, T, layer.value_heads, layer.value_dim)
    g = F.logsigmoid(x @ params["decay.weight"].t() + params["decay.bias"])
    beta = torch.sigmoid(x @ params["rate.weight"].t() + params["rate.bias"])
    S, out = state, []
    for t in range(T):
        live = t < lengths
        Sd = S * g[:, t].exp()[..., None, None]
        e = v[:, t] - (k[:, t, :, :, None] * Sd).sum(-2)
        Sn = Sd + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[..., None, :]
        S = torch.where(live[:, None, None, None], Sn, S)
        o = layer.key_dim ** -0.5 * (q[:, t, :, :, None] * S).sum(-2)
        out.append(torch.where(live[:, None, None], o, torch.zeros_like(o)))
    o = torch.stack(out, 1).reshape(B, T, values)
    return x + o @ params["out.weight"].t(), S


@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim,tokens", [(2, 2, 16, 16, 1), (4, 2, 32, 24, 70), (3, 1, 20, 33, 130)])
def test_layer_matches_its_formulas(gpu, heads, key_heads, key_dim, value_dim, tokens):
    from rnn_kernel_amd import GatedDelta

    torch.manual_seed(3)
    layer = GatedDelta(40, heads, key_dim, value_dim, key_heads, device=gpu)
    x = torch.randn(3, tokens, 40)
    lengths = torch.tensor([tokens, 0, (tokens + 1) // 2])
    state, dy = torch.randn(3, heads, key_dim, value_dim), torch.randn(3, tokens, 40)
    dev = [x.to(gpu).requires_grad_(True), state.to(gpu).requires_grad_(True)]
    y, last = layer(*dev, lengths.to(gpu, torch.int32))
    names, own = zip(*layer.named_parameters())
    got = torch.autograd.grad([y, last], [*dev, *own], [dy.to(gpu), torch.ones_like(last)])

    ref = [x.double().requires_grad_(True), state.double().requires_grad_(True)]
    params = {n: p.detach().double().cpu().requires_grad_(True) for n, p in zip(names, own)}
    ry, rlast = _oracle(layer, *ref, lengths, params)
    want = torch.autograd.grad([ry, rlast], [*ref, *params.values()], [dy.double(), torch.ones_like(rlast)])
    assert _rel(y - dev[0], ry - ref[0]) <= VALUE and _rel(last, rlast) <= VALUE
    for name, a, b in zip(("x", "state", *names), got, want):
        assert _rel(a, b) <= (DECAY_GRAD if name.startswith("decay") else GRAD), (name, _rel(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_answers_continue_a_prompt(gpu, dtype):
    """Tokens one by one, with states in a pool that is larger than the batch, a request
    without a state among them, are the whole sequence's."""
    from rnn_kernel_amd import GatedDelta

    torch.manual_seed(5)
    layer = GatedDelta(64, 4, 32, 32, 2, device=gpu, dtype=dtype)
    x = torch.randn(3, 90, 64, device=gpu).to(dtype)
    slots = torch.tensor([4, -1, 1], dtype=torch.int32, device=gpu)
    with torch.no_grad():
        whole, last = layer(x)
        pool = layer.new_states(6)
        _, state = layer(x[:, :80])
        pool[4], pool[1] = state[0], state[2]
        untouched = [pool[i].clone() for i in (0, 2, 3, 5)]
        steps = torch.stack([layer.step(x[:, t], pool, slots) for t in range(80, 90)], 1)
    # bfloat16: o and y are rounded on either side, of which y - x keeps y's, of the size of y
    tol = 2 * VALUE if dtype == torch.float32 else 4 * 2.0 ** -8
    scale = 1.0 if dtype == torch.float32 else float(whole.float().norm() / (whole - x).float().norm())
    for b in (0, 2):
        assert _rel(steps[b] - x[b, 80:], whole[b, 80:] - x[b, 80:]) <= tol * scale
    assert torch.equal(steps[1], x[1, 80:])
    assert _rel(pool[4], last[0]) <= VALUE and _rel(pool[1], last[2]) <= VALUE
    assert all(torch.equal(pool[i], u) for i, u in zip((0, 2, 3, 5), untouched))


def test_the_command_trains_and_answers(gpu):
    from rnn_kernel_amd.delta_train import main

    r = main(["--size", "64", "--heads", "2", "--key-heads", "1", "--head-dim", "32", "--batch-size", "4", "--seq-len", "100",
              "--steps", "40", "--answer", "9"])
    assert r["losses"][-1] < 0.7 * r["losses"][0]
    assert r["error"] <= 2 * VALUE
