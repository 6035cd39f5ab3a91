"""The operators of a language model on a selective state space, as cases to be timed.

Four operators, each through the package's public entry points where ``own`` is set
and in plain torch operations where it is not:

* the short causal convolution of each channel, y = act(b + sum_j w_j x_{t-W+1+j}):
  ``conv`` over sequences with every gradient, ``conv_step`` for one token of each of a
  batch of requests;
* the selective scan.  Per channel d and state n, with step sizes
  s = softplus(dt + bias),

      h_t[d, n] = exp(s A[d, n]) h_{t-1}[d, n] + s x_t[d] B_t[n]
      y_t[d] = (sum_n C_t[n] h_t[d, n] + skip[d] x_t[d]) silu(gate_t[d])

  ``scan`` over prompts, ``scan_train`` with every gradient, ``scan_step`` for single
  tokens, states in a pool;
* layer norm with its gradients: ``norm``;
* the cross entropy of a product with a vocabulary, -log softmax(x W^T + b)[target]:
  ``loss`` (a loss for each row) and ``loss_train`` (their mean, with every gradient).

``exact`` gives the same results in float64: recurrence and convolution token by token
with their adjoints, norm and loss from their formulas.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5  # of the norm
IGNORED = -100  # a row without a target


def _conv(name, kind, B, T, D, W, dtype="bf16", act="silu", lengths=False, s0=False, slots=0):
    return dict(name=name, kind=kind, B=B, T=T, D=D, W=W, dtype=dtype, act=act, lengths=lengths, s0=s0, slots=slots)


def _scan(name, kind, B, T, D, N, G=1, dtype="bf16", gate=True, lengths=False, s0=False, slots=0):
    return dict(name=name, kind=kind, B=B, T=T, D=D, N=N, G=G, dtype=dtype, gate=gate, lengths=lengths, s0=s0, slots=slots)


def _norm(name, M, K, dtype="bf16"):
    return dict(name=name, kind="norm", M=M, K=K, dtype=dtype)


def _loss(name, kind, M, K, V, dtype="bf16", bias=False, ignored=0.0):
    return dict(name=name, kind=kind, M=M, K=K, V=V, dtype=dtype, bias=bias, ignored=ignored)


def listed():
    return [
        # a training batch through the convolution
        _conv("conv_train", "conv", 4, 2048, 2048, 4),
        # a full serving batch, one token each, inputs kept in a pool
        _conv("conv_step", "conv_step", 256, 1, 2048, 4, slots=320),
        # one request answering, one token: launch latency is all there is
        _scan("scan_step_one", "scan_step", 1, 1, 256, 16, slots=1),
        # a full serving batch: every state is read and written once
        _scan("scan_step_batch", "scan_step", 256, 1, 4096, 16, slots=320),
        # one long prompt: the serial axis is long, the channels few
        _scan("scan_long", "scan", 1, 16384, 2048, 16),
        # prompts of unequal lengths (some empty) that continue earlier states, in groups of uneven sizes
        _scan("scan_ragged", "scan", 16, 1000, 520, 24, G=2, dtype="f32", lengths=True, s0=True),
        # training on whole sequences
        _scan("scan_train", "scan_train", 4, 2048, 2048, 16),
        # the norm in front of a layer, in training
        _norm("norm_train", 16384, 2048),
        # the same in 32 bits, odd sizes
        _norm("norm_f32_odd", 1000, 385, dtype="f32"),
        # training over a large vocabulary, some rows without a target
        _loss("loss_train", "loss_train", 8192, 2048, 64000, ignored=0.1),
        # 32 bits, odd sizes
        _loss("loss_f32_odd", "loss_train", 1000, 257, 10007, dtype="f32", bias=True, ignored=0.3),
        # how likely given texts are: a loss for each token, no gradients
        _loss("loss_rows", "loss", 2048, 1024, 100000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("conv", "conv_step", "scan_step", "scan", "scan_train", "norm", "loss_train", "loss"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    even = rng.random() < 0.5  # widths of real layers are mostly multiples of 64

    def width(lo, hi):
        d = _log_int(rng, lo, hi)
        return -(-d // 64) * 64 if even else d

    if kind == "norm":
        while True:
            m, k = _log_int(rng, 1, 32768), width(16, 8192)
            if m * k <= 16384 * 2048:
                break
        c = _norm("", m, k, dtype)
    elif kind.startswith("loss"):
        # (32-bit products run at a small share of the bf16 rate)
        most = 8192 * 2048 * 64000 // (1 if dtype == "bf16" else 8) // (1 if kind == "loss_train" else 2)
        while True:
            m, k, v = _log_int(rng, 1, 16384), width(16, 4096), width(50, 130000)
            if m * k * v <= most and m * v <= 8192 * 64000:
                break
        c = _loss("", kind, m, k, v, dtype, rng.random() < 0.4, rng.choice((0.0, 0.1, 0.5)))
    elif kind.startswith("conv"):
        step = kind == "conv_step"
        while True:
            b, t, d = _log_int(rng, 1, 512 if step else 32), 1 if step else _log_int(rng, 1, 8192), width(16, 8192)
            if b * t * d <= (512 * 2048 if step else 4 * 2048 * 2048):
                break
        c = _conv("", kind, b, t, d, rng.randint(2, 5), dtype, rng.choice(("none", "silu", "silu")),
                  not step and rng.random() < 0.4, step or rng.random() < 0.5, b + rng.randint(0, b) if step else 0)
    else:
        while True:
            g = rng.choice((1, 1, 2, 4))
            d, n = width(16, 4096) // g * g, rng.choice((16, 16, _log_int(rng, 1, 64)))
            if kind == "scan_step":
                b, t, most = _log_int(rng, 1, 256), 1, 256 * 4096 * 16
            elif kind == "scan":
                b, t, most = _log_int(rng, 1, 32), _log_int(rng, 1, 16384), 16384 * 2048 * 16
            else:
                b, t, most = _log_int(rng, 1, 16), _log_int(rng, 1, 4096), 4 * 2048 * 2048 * 16 // 2
            if b * t * d * n <= most:
                break
        step = kind == "scan_step"
        c = _scan("", kind, b, t, d, n, g, dtype, rng.random() < 0.7, not step and rng.random() < 0.4,
                  step or rng.random() < 0.6, b + rng.randint(0, b) if step else 0)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs ---


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    kind = case["kind"]

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def leaves(s, names):
        for n in names:
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_(True)
        return s

    if kind == "norm":
        M, K = case["M"], case["K"]
        s = dict(case=case, x=(2 * rand(M, K) + 0.5 * rand(M, 1)).to(dt), w=(1 + 0.2 * rand(K)).to(dt),
                 b=(0.2 * rand(K)).to(dt), dy=rand(M, K).to(dt))
        return leaves(s, "xwb")
    if kind.startswith("loss"):
        M, K, V = case["M"], case["K"], case["V"]
        target = torch.randint(0, V, (M,), generator=gen, device=DEVICE)
        if case["ignored"]:
            away = torch.rand(M, generator=gen, device=DEVICE) < case["ignored"]
            away[0] = False  # (one row has a target)
            target = torch.where(away, IGNORED, target)
        s = dict(case=case, x=rand(M, K).to(dt), w=(2 * rand(V, K) / math.sqrt(K)).to(dt),
                 b=rand(V).to(dt) if case["bias"] else None, target=target)
        if kind == "loss_train":
            s["dloss"] = 0.5 + torch.rand((), generator=gen, device=DEVICE)
            leaves(s, "xwb")
        return s

    B, T, D = case["B"], case["T"], case["D"]
    s = dict(case=case, lengths=None, s0=None, slots=None)
    if case["lengths"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device=DEVICE, dtype=torch.int32)
    if case["slots"]:
        s["slots"] = torch.randperm(case["slots"], generator=gen, device=DEVICE)[:B].to(torch.int32)
    # what goes into the convolution and the gate leave one projection: columns of a common row
    xz = rand(B, T, 2 * D).to(dt)
    if kind.startswith("conv"):
        W = case["W"]
        s.update(x=xz[..., :D], w=(rand(D, W) / math.sqrt(W)).to(dt), b=(0.3 * rand(D)).to(dt))
        if kind == "conv_step":
            s["x"] = s["x"][:, 0]
            s["state"] = rand(case["slots"], W - 1, D).to(dt)
            return s
        if case["s0"]:
            s["s0"] = rand(B, W - 1, D).to(dt)
        s.update(dy=rand(B, T, D).to(dt), ds=rand(B, W - 1, D).to(dt))
        return leaves(s, ("x", "w", "b", "s0"))

    N, G = case["N"], case["G"]
    x = rand(B, T, D)
    bc = rand(B, T, 2 * G * N).to(dt)
    first = torch.exp(torch.rand(D, generator=gen, device=DEVICE) * math.log(100.0) + math.log(1e-3))  # steps of 0.001 to 0.1
    A = -torch.arange(1, N + 1, device=DEVICE, dtype=torch.float32) * torch.exp(0.1 * rand(D, N))
    s.update(x=(x * torch.sigmoid(x)).to(dt), dt=(0.5 * rand(B, T, D)).to(dt), gate=xz[..., D:] if case["gate"] else None,
             A=A, B=bc[..., :G * N].view(B, T, G, N), C=bc[..., G * N:].view(B, T, G, N), skip=1 + 0.1 * rand(D),
             bias=first + torch.log(-torch.expm1(-first)))
    if kind == "scan_step":
        for n in ("x", "dt", "gate", "B", "C"):
            s[n] = s[n][:, 0] if s[n] is not None else None
        s["state"] = rand(case["slots"], D, N)
        return s
    if case["s0"]:
        s["s0"] = rand(B, D, N)
    if kind == "scan_train":
        s.update(dy=rand(B, T, D).to(dt), ds=rand(B, D, N))
        leaves(s, SCANNED)
    return s


# ------------------------------------------------------------- plain forms ---


def _silu(z):
    return z * torch.sigmoid(z)


def _plain_conv(x, w, b, s0, act, lengths):
    B, T, D = x.shape
    W = w.size(1)
    before = x.new_zeros(B, W - 1, D) if s0 is None else s0
    xs = torch.cat([before, x], 1)
    windows = xs.float().unfold(1, W, 1)  # [B, T, D, W]
    z = (windows * w.float()).sum(-1) + b.float()
    y = _silu(z) if act == "silu" else z
    if lengths is None:
        return y.to(x.dtype), xs[:, T:]
    live = torch.arange(T, device=x.device)[None, :] < lengths[:, None]
    last = lengths.long()[:, None] + torch.arange(W - 1, device=x.device)
    return torch.where(live[..., None], y, 0.0).to(x.dtype), xs.gather(1, last[..., None].expand(-1, -1, D))


def _plain_conv_step(x, state, w, b, act, slots):
    at = slots.long()
    xs = torch.cat([state[at], x[:, None]], 1)
    z = (xs.float() * w.float().t()).sum(1) + b.float()
    state[at] = xs[:, 1:]
    return (_silu(z) if act == "silu" else z).to(x.dtype)


def _steps(dt, bias):
    r = dt.float() + bias
    return torch.clamp(r, min=0) + torch.log1p(torch.exp(-torch.abs(r)))


def _read_out(h, C, x, skip, gate, dtype):
    y = (C * h).sum(-1) + skip * x
    return (y if gate is None else y * _silu(gate.float())).to(dtype)


def _plain_scan(x, dt, A, Bm, C, s0, skip, gate, bias, lengths):
    """All tokens at once: after the pass with reach k every h is the sum over the 2k last
    tokens, and a the decay over them."""
    T, rep = x.size(1), x.size(2) // Bm.size(2)
    step, xf = _steps(dt, bias), x.float()
    if lengths is not None:
        live = torch.arange(T, device=x.device)[None, :] < lengths[:, None]
        step, xf = torch.where(live[..., None], step, 0.0), torch.where(live[..., None], xf, 0.0)
    a = torch.exp(step[..., None] * A)
    h = (step * xf)[..., None] * Bm.float().repeat_interleave(rep, 2)
    if s0 is not None:
        h = torch.cat([h[:, :1] + a[:, :1] * s0[:, None], h[:, 1:]], 1)
    k = 1
    while k < T:
        h = torch.cat([h[:, :k], h[:, k:] + a[:, k:] * h[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1) if 2 * k < T else a
        k *= 2
    y = _read_out(h, C.float().repeat_interleave(rep, 2), xf, skip, gate, x.dtype)
    return (y if lengths is None else torch.where(live[..., None], y, 0.0)), h[:, -1]


def _plain_scan_step(x, dt, A, Bm, C, state, skip, gate, bias, slots):
    rep, at = x.size(1) // Bm.size(1), slots.long()
    step, xf = _steps(dt, bias), x.float()
    h = torch.exp(step[..., None] * A) * state[at] + (step * xf)[..., None] * Bm.float().repeat_interleave(rep, 1)
    state[at] = h
    return _read_out(h, C.float().repeat_interleave(rep, 1), xf, skip, gate, x.dtype)


def _plain_norm(x, w, b):
    xf = x.float()
    c = xf - xf.mean(-1, keepdim=True)
    return (c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * w.float() + b.float()).to(x.dtype)


def _plain_loss(x, w, b, target):
    """A loss for each row, 0 for those without a target."""
    z = torch.matmul(x.float(), w.float().t())
    if b is not None:
        z = z + b.float()
    top = z.detach().amax(-1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(-1))
    of = z.gather(1, target.clamp(min=0)[:, None])[:, 0]
    return torch.where(target == IGNORED, 0.0, lse - of)


# --------------------------------------------------------------------- run ---

SCANNED = ("x", "dt", "A", "B", "C", "s0", "skip", "gate", "bias")


def _with_gradients(s, outs, names, douts):
    names = [n for n in names if s[n] is not None]
    grads = torch.autograd.grad(list(outs.values()), [s[n] for n in names], douts, allow_unused=True, materialize_grads=True)
    return dict(outs, **{"d" + n: t for n, t in zip(names, grads)})


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import rnn_kernel_amd as rka
    if kind == "norm":
        y = rka.layer_norm(s["x"], s["w"], s["b"], EPS) if own else _plain_norm(s["x"], s["w"], s["b"])
        return _with_gradients(s, dict(y=y), ("x", "w", "b"), [s["dy"]])
    if kind == "loss":
        if own:
            return rka.linear_cross_entropy(s["x"], s["w"], s["target"], s["b"], reduction="none")
        return _plain_loss(s["x"], s["w"], s["b"], s["target"])
    if kind == "loss_train":
        if own:
            loss = rka.linear_cross_entropy(s["x"], s["w"], s["target"], s["b"])
        else:
            loss = _plain_loss(s["x"], s["w"], s["b"], s["target"]).sum() / (s["target"] != IGNORED).sum()
        return _with_gradients(s, dict(loss=loss), ("x", "w", "b"), [s["dloss"]])
    if kind == "conv_step":
        args = (s["x"], s["state"], s["w"], s["b"])
        if own:
            y = rka.causal_conv_step(*args, activation=case["act"], slots=s["slots"])
        else:
            y = _plain_conv_step(*args, case["act"], s["slots"])
        return dict(y=y, state=s["state"])
    if kind == "conv":
        args = (s["x"], s["w"], s["b"], s["s0"])
        if own:
            y, state = rka.causal_conv(*args, activation=case["act"], lengths=s["lengths"])
        else:
            y, state = _plain_conv(*args, case["act"], s["lengths"])
        return _with_gradients(s, dict(y=y, state=state), ("x", "w", "b", "s0"), [s["dy"], s["ds"]])
    args = [s[n] for n in ("x", "dt", "A", "B", "C")]
    if kind == "scan_step":
        if own:
            y = rka.selective_step(*args, s["state"], skip=s["skip"], gate=s["gate"], dt_bias=s["bias"], softplus=True,
                                   slots=s["slots"])
        else:
            y = _plain_scan_step(*args, s["state"], s["skip"], s["gate"], s["bias"], s["slots"])
        return dict(y=y, state=s["state"])
    if own:
        y, state = rka.selective_scan(*args, s["s0"], skip=s["skip"], gate=s["gate"], dt_bias=s["bias"], softplus=True,
                                      lengths=s["lengths"])
    else:
        y, state = _plain_scan(*args, s["s0"], s["skip"], s["gate"], s["bias"], s["lengths"])
    outs = dict(y=y, state=state)
    return _with_gradients(s, outs, SCANNED, [s["dy"], s["ds"]]) if kind == "scan_train" else outs


# -------------------------------------------------------------------- work ---


def work(case):
    e, kind = 4 if case["dtype"] == "f32" else 2, case["kind"]
    if kind == "norm":
        M, K = case["M"], case["K"]
        return {"bytes": e * (5 * M * K + 4 * K), "flops": 20 * M * K}
    if kind.startswith("loss"):
        M, K, V = case["M"], case["K"], case["V"]
        mats = e * (M * K + V * K + V * case["bias"])
        if kind == "loss":
            return {"bytes": mats + 12 * M, "flops": 2 * M * K * V}
        # the products of rows without a target need not be made
        return {"bytes": 2 * mats + 8 * M, "flops": 6 * M * K * V * (1 - case["ignored"])}
    B, T, D = case["B"], case["T"], case["D"]
    tokens = B * T * (0.5 if case["lengths"] else 1.0)  # lengths are drawn evenly from 0 to T
    if kind.startswith("conv"):
        W = case["W"]
        if kind == "conv_step":
            return {"bytes": e * B * D * (2 + 2 * (W - 1)) + e * D * (W + 1), "flops": 2 * B * D * W}
        return {"bytes": e * D * (3 * tokens + 2 * B * T + 2 * (W + 1) + 2 * B * (W - 1) * (1 + case["s0"])),
                "flops": 6 * tokens * D * W}
    N, G = case["N"], case["G"]
    fixed = 4 * D * (N + 2)
    inputs = e * tokens * (D * (2 + case["gate"]) + 2 * G * N)
    y, state = e * B * T * D, 4 * B * D * N
    flops = 7 * tokens * D * N  # decay, its exponential, update and output of a state
    if kind != "scan_train":
        s0 = case["s0"] or kind == "scan_step"
        return {"bytes": fixed + inputs + y + state * (1 + s0), "flops": flops}
    return {"bytes": 2 * (fixed + inputs + y + state * (1 + case["s0"])), "flops": 3 * flops}


# ------------------------------------------------------------------- exact ---


def exact(case, seed):
    kind = case["kind"]
    with torch.no_grad():
        s = {n: t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t
             for n, t in prepare(case, seed).items()}
        if kind == "norm":
            return _exact_norm(s)
        if kind.startswith("loss"):
            return _exact_loss(s, kind)
        if kind.startswith("conv"):
            return _exact_conv(s, case)
        return _exact_scan(s, case)


def _exact_norm(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    unit = (x - mean) / (var + EPS).sqrt()
    g = dy * w
    dx = (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True)) / (var + EPS).sqrt()
    return dict(y=unit * w + s["b"], dx=dx, dw=(dy * unit).sum(0), db=dy.sum(0))


def _exact_loss(s, kind):
    x, w, target = s["x"], s["w"], s["target"]
    M = x.size(0)
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"]
    logp = torch.log_softmax(z, -1)
    del z
    rows = torch.arange(M, device=x.device)
    on = target != IGNORED
    at = torch.where(on, target, 0)
    loss = torch.where(on, -logp[rows, at], 0.0)
    if kind == "loss":
        return loss
    count = on.sum()
    dz = logp.exp_()
    dz[rows, at] -= 1.0
    dz *= (on * s["dloss"] / count)[:, None]
    out = dict(loss=loss.sum() / count, dx=dz @ w, dw=dz.t() @ x)
    if s["b"] is not None:
        out["db"] = dz.sum(0)
    return out


def _silu_and_slope(z):
    sig = torch.sigmoid(z)
    return z * sig, sig * (1 + z * (1 - sig))


def _exact_conv(s, case):
    x, w, b = s["x"], s["w"], s["b"]
    W = case["W"]
    if case["kind"] == "conv_step":
        at = s["slots"].long()
        xs = torch.cat([s["state"][at], x[:, None]], 1)
        z = torch.einsum("bwd,dw->bd", xs, w) + b
        pool = s["state"].clone()
        pool[at] = xs[:, 1:]
        return dict(y=_silu_and_slope(z)[0] if case["act"] == "silu" else z, state=pool)
    B, T, D = x.shape
    before = torch.zeros(B, W - 1, D, dtype=x.dtype, device=x.device) if s["s0"] is None else s["s0"]
    xs = torch.cat([before, x], 1)
    z = b.expand(B, T, D).clone()
    for j in range(W):
        z += w[:, j] * xs[:, j:j + T]
    y, slope = _silu_and_slope(z) if case["act"] == "silu" else (z, torch.ones_like(z))
    n = torch.full((B,), T, device=x.device) if s["lengths"] is None else s["lengths"].long()
    live = (torch.arange(T, device=x.device)[None, :] < n[:, None])[..., None]
    dz = torch.where(live, s["dy"] * slope, 0.0)
    dxs = torch.zeros_like(xs)
    dw = torch.zeros_like(w)
    for j in range(W):
        dxs[:, j:j + T] += w[:, j] * dz
        dw[:, j] = (dz * xs[:, j:j + T]).sum((0, 1))
    state = torch.empty_like(before)
    rows = torch.arange(B, device=x.device)
    for j in range(W - 1):
        state[:, j] = xs[rows, n + j]
        dxs[rows, n + j] += s["ds"][:, j]
    out = dict(y=torch.where(live, y, 0.0), state=state, dx=dxs[:, W - 1:], dw=dw, db=dz.sum((0, 1)))
    if s["s0"] is not None:
        out["ds0"] = dxs[:, :W - 1]
    return out


def _exact_scan(s, case):
    kind, D, N, G = case["kind"], case["D"], case["N"], case["G"]
    x, dt, A, Bm, C, skip, gate = (s[n] for n in ("x", "dt", "A", "B", "C", "skip", "gate"))
    if kind == "scan_step":
        x, dt, Bm, C = (t[:, None] for t in (x, dt, Bm, C))
        gate = None if gate is None else gate[:, None]
    B, T = x.shape[:2]
    raw = dt + s["bias"]
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    live = torch.ones(B, T, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=x.device)[None, :] < s["lengths"][:, None]
    on = live[..., None]
    sizes = (D // G, N)

    def wide(t):  # [B, G, N] -> [B, D, N]
        return t[:, :, None].expand(-1, -1, *sizes).reshape(B, D, N)

    if kind == "scan_step":
        h = s["state"][s["slots"].long()]
    else:
        h = torch.zeros(B, D, N, dtype=x.dtype, device=x.device) if s["s0"] is None else s["s0"]
    train = kind == "scan_train"
    read, before = torch.zeros_like(x), []
    for t in range(T):
        if train:
            before.append(h)
        new = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * x[:, t])[..., None] * wide(Bm[:, t])
        h = torch.where(on[:, t, :, None], new, h)
        read[:, t] = (wide(C[:, t]) * h).sum(-1)
    ungated = read + skip * x
    open_, slope = _silu_and_slope(gate) if gate is not None else (torch.ones_like(x), None)
    y = torch.where(on, ungated * open_, 0.0)
    if kind == "scan_step":
        pool = s["state"].clone()
        pool[s["slots"].long()] = h
        return dict(y=y[:, 0], state=pool)
    out = dict(y=y, state=h)
    if not train:
        return out
    dy = torch.where(on, s["dy"], 0.0)
    if gate is not None:
        out["dgate"] = dy * ungated * slope
    dr = dy * open_
    dh = s["ds"]
    dA = torch.zeros_like(A)
    dB, dC, dx, dstep = torch.zeros_like(Bm), torch.zeros_like(C), skip * dr, torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        m = on[:, t, :, None]
        h0, st, xt, Bt = before[t], step[:, t], x[:, t], wide(Bm[:, t])
        a = torch.exp(st[..., None] * A)
        ht = a * h0 + (st * xt)[..., None] * Bt
        full = dh + dr[:, t, :, None] * wide(C[:, t])
        live_h = torch.where(m, full, 0.0)
        dC[:, t] = (dr[:, t, :, None] * ht).unflatten(1, (G, D // G)).sum(2)
        dB[:, t] = ((st * xt)[..., None] * live_h).unflatten(1, (G, D // G)).sum(2)
        of_b, of_a = (live_h * Bt).sum(-1), live_h * a * h0
        dx[:, t] += st * of_b
        dstep[:, t] = xt * of_b + (of_a * A).sum(-1)
        dA += (of_a * st[..., None]).sum(0)
        dh = torch.where(m, a * full, dh)
    ddt = dstep * torch.sigmoid(raw)
    out.update(dx=dx, ddt=ddt, dA=dA, dB=dB, dC=dC, dskip=(dr * x).sum((0, 1)), dbias=ddt.sum((0, 1)))
    if s["s0"] is not None:
        out["ds0"] = dh
    return out
