"""The operators of a language model together, as they are used: embedded tokens through
layers of norm, projections, convolution and scan, and the loss over the vocabulary; training
steps, prompts of unequal length and answers token by token.

Tolerances, set before the first run.  float32 against the same model in plain float64
operations: an output passes some eight operators of at most 4e-6 each: 3e-5; gradients twice as
many: 1e-4, as 2-norms.  bfloat16 answers against the whole sequence: every operator rounds its
result (2^-9 rms) in other places of the sums only, some ten roundings, and the states carry
them on: 0.05."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

VALUE, GRAD, BF16 = 3e-5, 1e-4, 0.05


class Model(nn.Module):
    def __init__(self, vocabulary, size, layers, device, dtype=torch.float32, **options):
        from rnn_kernel_amd import LayerNorm, LinearCrossEntropy, SelectiveScan

        super().__init__()
        self.embedding = nn.Parameter(torch.randn(vocabulary, size, device=device).to(dtype))
        self.layers = nn.ModuleList(SelectiveScan(size, device=device, dtype=dtype, **options) for _ in range(layers))
        self.norm = LayerNorm(size, device=device, dtype=dtype)
        self.head = LinearCrossEntropy(size, vocabulary, device=device, dtype=dtype)

    def hidden(self, tokens, states=None, lengths=None):
        x, new = self.embedding[tokens], []
        for i, layer in enumerate(self.layers):
            x, s = layer(x, None if states is None else states[i], lengths)
            new.append(s)
        return self.norm(x), new

    def step(self, tokens, states, slots):
        x = self.embedding[tokens]
        for layer, s in zip(self.layers, states):
            x = layer.step(x, s, slots)
        return self.norm(x)


def _plain_layer(layer, x, lengths):
    p = {k: v.double() for k, v in layer.named_parameters()}
    B, T, _ = x.shape
    D, N, G, W = layer.channels, layer.states, layer.groups, layer.width
    live = (torch.arange(T, device=x.device)[None, :] < lengths[:, None])[..., None]
    xn = nn.functional.layer_norm(x, (layer.size,), p["norm.weight"], p["norm.bias"])
    u, z = (xn @ p["project.weight"].t()).chunk(2, -1)
    u = torch.where(live, u, 0.0)
    us = torch.cat([u.new_zeros(B, W - 1, D), u], 1)
    u = nn.functional.silu(sum(p["conv_weight"][:, j] * us[:, j:j + T] for j in range(W)) + p["conv_bias"])
    d, Bm, C = (u @ p["inputs.weight"].t()).split([layer.step_rank, G * N, G * N], -1)
    s = nn.functional.softplus(d @ p["steps.weight"].t() + p["step_bias"])
    Bm, C = (t.unflatten(-1, (G, N)).repeat_interleave(D // G, 2) for t in (Bm, C))
    A, h, out = -p["A_log"].exp(), u.new_zeros(B, D, N), []
    for t in range(T):
        h = torch.exp(s[:, t, :, None] * A) * h + (s[:, t] * u[:, t])[..., None] * Bm[:, t]
        out.append(((C[:, t] * h).sum(-1) + p["skip"] * u[:, t]) * nn.functional.silu(z[:, t]))
    return x + torch.where(live, torch.stack(out, 1), 0.0) @ p["out.weight"].t()


def _rel(a, b):
    assert torch.isfinite(a).all()
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm().clamp_min(1e-30))


def test_a_training_step_against_float64(gpu):
    torch.manual_seed(0)
    model = Model(101, 48, 2, gpu, states=8, groups=2, width=3)
    tokens = torch.randint(0, 101, (3, 70), device=gpu)
    lengths = torch.tensor([70, 1, 33], dtype=torch.int32, device=gpu)
    target = torch.roll(tokens, -1, 1)
    target[torch.arange(70, device=gpu)[None, :] >= lengths[:, None] - 1] = -100
    hidden, _ = model.hidden(tokens, lengths=lengths)
    loss = model.head(hidden, target)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    ref = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    x = ref["embedding"][tokens]
    with torch.nn.utils.stateless._reparametrize_module(model, ref):
        for layer in model.layers:
            x = _plain_layer(layer, x, lengths)
        x = nn.functional.layer_norm(x, (48,), model.norm.weight, model.norm.bias)
        want = nn.functional.cross_entropy((x @ model.head.weight.t()).flatten(0, 1), target.flatten())
    live = torch.arange(70, device=gpu)[None, :] < lengths[:, None]
    assert _rel(hidden[live], x[live]) <= VALUE and _rel(loss, want) <= VALUE
    for (name, r), g in zip(ref.items(), grads):
        rg = torch.autograd.grad(want, r, retain_graph=True)[0]
        assert _rel(g, rg) <= GRAD, (name, _rel(g, rg))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_and_answers_token_by_token(gpu, dtype):
    torch.manual_seed(1)
    model = Model(64, 64, 2, gpu, dtype)
    tokens = torch.randint(0, 64, (4, 40), device=gpu)
    slots = torch.tensor([5, 0, 3, 2], dtype=torch.int32, device=gpu)
    with torch.no_grad():
        whole, _ = model.hidden(tokens)
        lengths = torch.tensor([30, 7, 0, 39], dtype=torch.int32, device=gpu)
        _, states = model.hidden(tokens, lengths=lengths)
        pools = [layer.new_states(6) for layer in model.layers]
        for pool, state in zip(pools, states):
            for p, s in zip(pool, state):
                p[slots.long()] = s
        at = lengths.clone()
        out = whole.clone()
        while int(at.min()) < 40:  # rows that are through stand aside as padding
            todo = at < 40
            y = model.step(tokens[torch.arange(4, device=gpu), at.clamp(max=39).long()], pools, torch.where(todo, slots, -1))
            for b in range(4):
                if todo[b]:
                    out[b, at[b]] = y[b]
            at = at + todo.int()
        answered = torch.arange(40, device=gpu)[None, :] >= lengths[:, None]
        assert _rel(out[answered], whole[answered]) <= (VALUE if dtype == torch.float32 else BF16)


def test_steps_of_training_change_every_parameter(gpu):
    from rnn_kernel_amd import AdamW

    torch.manual_seed(2)
    model = Model(50, 32, 1, gpu)
    before = [p.detach().clone() for p in model.parameters()]
    optimizer = AdamW(model.parameters(), lr=1e-2)
    for _ in range(3):
        tokens = torch.randint(0, 50, (2, 25), device=gpu)
        optimizer.zero_grad()
        model.head(model.hidden(tokens[:, :-1])[0], tokens[:, 1:]).backward()
        optimizer.step()
    assert all(torch.isfinite(p).all() and not torch.equal(p, b) for p, b in zip(model.parameters(), before))


def test_a_captured_step_replays(gpu):
    """One token through a layer as a graph, its states updated by every replay."""
    torch.manual_seed(3)
    model = Model(50, 64, 2, gpu)
    tokens = torch.randint(0, 50, (3,), device=gpu)
    slots = torch.tensor([2, 0, -1], dtype=torch.int32, device=gpu)
    pools, check = ([layer.new_states(4) for layer in model.layers] for _ in range(2))
    with torch.no_grad():
        model.step(tokens, check, slots)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model.step(tokens, pools, slots)
        for pool in (pools, check):
            for s in pool:
                for t in s:
                    t.zero_()
        for _ in range(4):
            tokens.copy_(torch.randint(0, 50, (3,), device=gpu))
            graph.replay()
            want = model.step(tokens, check, slots)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            assert all(torch.equal(a, b) for p, q in zip(pools, check) for a, b in zip(p, q))
