"""The operators of a gated delta-rule layer, as cases to be timed.

Two operators, each through the package's public entry points where ``own`` is
set and in plain torch operations where it is not:

* the gated delta rule.  Per head, with a state S [Dk, Dv] held in 32 bits,

      S_t = exp(g_t) S_{t-1} + k_t (beta_t (v_t - k_t^T exp(g_t) S_{t-1}))^T
      o_t = scale * S_t^T q_t

  ``step`` is one token for each of a batch of requests whose states live in a
  pool (serving), ``rule`` whole sequences with or without lengths and an
  initial state, ``train`` the same with every gradient;
* the matrix product with its epilogue, y = act(x W^T + b) + r: ``linear``
  forward, ``linear_train`` with every gradient.

``exact`` gives the same results in float64: the recurrence token by token with
its adjoint, and the product's gradients from their formulas.
"""
import math

import torch

own = False

DEVICE = "cuda"
CHUNK = 64
EPS = 1e-6  # under the root of a normalised query or key


def _delta(name, kind, B, T, Hk, Hv, Dk, Dv, dtype="bf16", lengths=False, s0=True, normalize=True, slots=0):
    return dict(name=name, kind=kind, B=B, T=T, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=dtype, lengths=lengths, s0=s0,
                normalize=normalize, slots=slots)


def _linear(name, kind, M, N, K, dtype="bf16", act="none", bias=True, residual=False):
    return dict(name=name, kind=kind, M=M, N=N, K=K, dtype=dtype, act=act, bias=bias, residual=residual)


def listed():
    return [
        # one request answering, one token: launch latency is all there is
        _delta("step_one", "step", 1, 1, 4, 8, 64, 64, slots=1),
        # a full serving batch, one token each, states scattered over a pool:
        # every state is read and written once
        _delta("step_batch", "step", 256, 1, 16, 32, 128, 128, slots=320),
        # one long prompt on few heads: the serial axis is long, the rows few
        _delta("rule_long", "rule", 1, 16384, 8, 16, 128, 128, s0=False),
        # prompts of unequal lengths (some empty) that continue earlier states,
        # with heads of unequal and uneven sizes
        _delta("rule_ragged", "rule", 16, 1000, 8, 8, 64, 96, lengths=True),
        # training on whole sequences, query and key heads shared by two
        # value heads each
        _delta("train_bf16", "train", 4, 2048, 8, 16, 128, 128),
        # training in 32 bits with head sizes that are no multiple of anything
        _delta("train_f32_odd", "train", 2, 333, 3, 3, 96, 129, dtype="f32", lengths=True, normalize=False),
        # a projection while answering: few rows, all of the weight is read
        _linear("linear_token", "linear", 4, 4096, 2048, act="silu"),
        # the gates of a layer: many rows, few columns
        _linear("linear_gates", "linear", 8192, 32, 2048, act="logsigmoid"),
        # the output projection over a large prompt batch, with its residual
        _linear("linear_prefill", "linear", 16384, 4096, 4096, act="gelu", residual=True),
        # a projection in training
        _linear("linear_train", "linear_train", 8192, 2048, 2048, act="silu", residual=True),
        # training in 32 bits, odd sizes
        _linear("linear_f32_odd", "linear_train", 1000, 385, 257, dtype="f32", act="gelu", residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


ACTIVATIONS = ("none", "relu", "gelu", "silu", "sigmoid", "logsigmoid")


def draw(rng):
    kind = rng.choice(("step", "rule", "train", "linear", "linear_train"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind.startswith("linear"):
        train = kind == "linear_train"
        # 32-bit products run at a small share of the bf16 rate
        most = (8192 * 2048 * 2048 if train else 16384 * 4096 * 4096) // (1 if dtype == "bf16" else 4)
        while True:
            m, n, k = _log_int(rng, 1, 16384), _log_int(rng, 8, 4096), _log_int(rng, 16, 4096)
            if rng.random() < 0.5:  # widths of real layers are mostly multiples of 64
                n, k = -(-n // 64) * 64, -(-k // 64) * 64
            if m * n * k <= most and 3072 not in (m, n, k):
                break
        c = _linear("", kind, m, n, k, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.7, rng.random() < 0.5)
    else:
        while True:
            hk = rng.randint(1, 16)
            hv = hk * rng.choice((1, 1, 2, 4))
            dk, dv = _log_int(rng, 16, 256), _log_int(rng, 16, 256)
            if rng.random() < 0.5:
                dk, dv = -(-dk // 32) * 32, -(-dv // 32) * 32
            if kind == "step":
                b, t, most = _log_int(rng, 1, 256), 1, 256 * 32 * 128 * 128
            elif kind == "rule":
                b, t, most = _log_int(rng, 1, 32), _log_int(rng, 1, 16384), 16384 * 16 * 128 * 128
            else:
                b, t, most = _log_int(rng, 1, 16), _log_int(rng, 1, 2048), 4 * 2048 * 16 * 128 * 128 // 2
            if b * t * hv * dk * dv <= most:
                break
        c = _delta("", kind, b, t, hk, hv, dk, dv, dtype, kind != "step" and rng.random() < 0.4,
                   kind == "step" or rng.random() < 0.6, rng.random() < 0.6, b + rng.randint(0, b) if kind == "step" else 0)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs ---


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = _dtype(case)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    if case["kind"].startswith("linear"):
        M, N, K = case["M"], case["N"], case["K"]
        s = dict(case=case, x=rand(M, K).to(dt), w=(rand(N, K) / math.sqrt(K)).to(dt),
                 b=(0.5 * rand(N)).to(dt) if case["bias"] else None, r=rand(M, N).to(dt) if case["residual"] else None)
        if case["kind"] == "linear_train":
            s["dy"] = rand(M, N).to(dt)
            for n in ("x", "w", "b", "r"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
        return s

    B, T, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    # queries, keys and values as they leave one projection: columns of a
    # common row
    qkv = rand(B, T, 2 * Hk * Dk + Hv * Dv)
    if not case["normalize"]:  # already of length one or so, as a layer without the norm would have them
        qkv[..., :2 * Hk * Dk] /= math.sqrt(Dk)
    qkv = qkv.to(dt)
    q = qkv[..., :Hk * Dk].view(B, T, Hk, Dk)
    k = qkv[..., Hk * Dk:2 * Hk * Dk].view(B, T, Hk, Dk)
    v = qkv[..., 2 * Hk * Dk:].view(B, T, Hv, Dv)
    g = torch.nn.functional.logsigmoid(rand(B, T, Hv) + 3.0)
    beta = torch.sigmoid(rand(B, T, Hv))
    s = dict(case=case, q=q, k=k, v=v, g=g, beta=beta, lengths=None, s0=None, scale=Dk ** -0.5)
    if case["kind"] == "step":
        for n in ("q", "k", "v", "g", "beta"):
            s[n] = s[n][:, 0]
        s["state"] = rand(case["slots"], Hv, Dk, Dv) / math.sqrt(Dk)
        s["slots"] = torch.randperm(case["slots"], generator=gen, device=DEVICE)[:B].to(torch.int32)
        return s
    if case["s0"]:
        s["s0"] = rand(B, Hv, Dk, Dv) / math.sqrt(Dk)
    if case["lengths"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device=DEVICE, dtype=torch.int32)
    if case["kind"] == "train":
        s["do"] = rand(B, T, Hv, Dv).to(dt)
        s["ds"] = rand(B, Hv, Dk, Dv) / math.sqrt(Dk)
        for n in ("q", "k", "v", "g", "beta", "s0"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_(True)
    return s


# ------------------------------------------------------------- plain forms ---


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "logsigmoid":
        return torch.clamp(z, max=0) - torch.log1p(torch.exp(-torch.abs(z)))
    return z


def _plain_linear(x, w, b, r, act):
    z = torch.matmul(x.float(), w.float().t())
    if b is not None:
        z = z + b.float()
    y = _act(z, act)
    if r is not None:
        y = y + r.float()
    return y.to(x.dtype)


def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)


def _plain_step(q, k, v, g, beta, state, slots, scale, normalize):
    rep = v.size(1) // q.size(1)
    qf, kf = q.float(), k.float()
    if normalize:
        qf, kf = _unit(qf), _unit(kf)
    qf, kf = qf.repeat_interleave(rep, 1), kf.repeat_interleave(rep, 1)
    s = state[slots.long()] * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v.float() - (kf[..., None] * s).sum(-2))
    s = s + kf[..., None] * u[..., None, :]
    state[slots.long()] = s
    return ((scale * qf)[..., None] * s).sum(-2).to(q.dtype)


def _plain_rule(q, k, v, g, beta, s0, lengths, scale, normalize):
    """Chunks of 64 tokens: everything but the state's way from chunk to chunk
    is done for all chunks at once; that way is a loop, as it is serial."""
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    qf, kf, vf = q.float(), k.float(), v.float()
    gf, bf = g.float(), beta.float()
    if normalize:
        qf, kf = _unit(qf), _unit(kf)
    if lengths is not None:
        live = torch.arange(T, device=q.device)[None, :] < lengths[:, None]
        qf, kf, vf = (torch.where(live[..., None, None], t, 0.0) for t in (qf, kf, vf))
        gf, bf = (torch.where(live[..., None], t, 0.0) for t in (gf, bf))
    n = -(-T // CHUNK)
    pad = n * CHUNK - T

    def chunks(t):  # [B, T, H, ...] -> [n, B, H, CHUNK, ...]
        t = torch.cat([t, t.new_zeros((B, pad) + t.shape[2:])], 1) if pad else t
        return t.unflatten(1, (n, CHUNK)).movedim(1, 0).transpose(2, 3)

    rep = Hv // Hk
    qc = chunks((qf * scale).repeat_interleave(rep, 2))
    kc, vc, gc, bc = chunks(kf.repeat_interleave(rep, 2)), chunks(vf), chunks(gf), chunks(bf)
    G = gc.cumsum(-1)
    i = torch.arange(CHUNK, device=q.device)
    decay = torch.exp(torch.where(i[:, None] >= i[None, :], G[..., :, None] - G[..., None, :], float("-inf")))
    kk = torch.matmul(kc, kc.transpose(-1, -2)) * decay
    # the inverse of I + N, N strictly lower triangular: that of its diagonal
    # blocks of two, four, ... rows from that of blocks of half the rows
    lower = torch.where(i[:, None] > i[None, :], kk, 0.0) * bc[..., None, :]
    inverse = torch.eye(CHUNK, device=q.device).expand_as(lower)
    for level in range(CHUNK.bit_length() - 1):
        half = (i[:, None] >> level == (i[None, :] >> level) + 1) & (i[:, None] >> (level + 1) == i[None, :] >> (level + 1))
        inverse = inverse - torch.matmul(torch.matmul(inverse, torch.where(half, lower, 0.0)), inverse)
    gamma = torch.exp(G)[..., None]
    ev, ek = torch.matmul(inverse, vc), torch.matmul(inverse, gamma * kc)
    last = torch.exp(G[..., -1])[..., None, None]
    kw = (kc * torch.exp(G[..., -1:] - G)[..., None]).transpose(-1, -2)
    state = s0 if s0 is not None else q.new_zeros((B, Hv, Dk, Dv), dtype=torch.float32)
    states, us = [], []
    for c in range(n):
        u = bc[c][..., None] * (ev[c] - torch.matmul(ek[c], state))
        states.append(state)
        us.append(u)
        state = last[c] * state + torch.matmul(kw[c], u)
    o = torch.matmul(qc * gamma, torch.stack(states)) + torch.matmul(torch.matmul(qc, kc.transpose(-1, -2)) * decay, torch.stack(us))
    o = o.transpose(2, 3).movedim(0, 1).flatten(1, 2)[:, :T]
    return o.to(q.dtype), state


# --------------------------------------------------------------------- run ---

GRADS = ("q", "k", "v", "g", "beta", "s0")


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import rnn_kernel_amd as rka
    if kind.startswith("linear"):
        if own:
            y = rka.linear(s["x"], s["w"], s["b"], activation=case["act"], residual=s["r"])
        else:
            y = _plain_linear(s["x"], s["w"], s["b"], s["r"], case["act"])
        if kind == "linear":
            return y
        names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        return dict(y=y, **{"d" + n: t for n, t in zip(names, grads)})
    args = [s[n] for n in ("q", "k", "v", "g", "beta")]
    norm = case["normalize"]
    if kind == "step":
        if own:
            o = rka.gated_delta_step(*args, s["state"], slots=s["slots"], scale=s["scale"], normalize=norm)
        else:
            o = _plain_step(*args, s["state"], s["slots"], s["scale"], norm)
        return dict(o=o, state=s["state"])
    if own:
        o, state = rka.gated_delta_rule(*args, s["s0"], scale=s["scale"], normalize=norm, lengths=s["lengths"])
    else:
        o, state = _plain_rule(*args, s["s0"], s["lengths"], s["scale"], norm)
    if kind == "rule":
        return dict(o=o, state=state)
    names = [n for n in GRADS if s[n] is not None]
    grads = torch.autograd.grad([o, state], [s[n] for n in names], [s["do"], s["ds"]])
    return dict(o=o, state=state, **{"d" + n: t for n, t in zip(names, grads)})


# -------------------------------------------------------------------- work ---


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"].startswith("linear"):
        M, N, K = case["M"], case["N"], case["K"]
        mats = M * K + N * K + M * N * (1 + case["residual"]) + N * case["bias"]
        if case["kind"] == "linear":
            return {"bytes": e * mats, "flops": 2 * M * N * K}
        # the gradients of x, W and b are written, dy is read
        return {"bytes": e * (mats + M * K + N * K + M * N + N * case["bias"]), "flops": 6 * M * N * K}
    B, T, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    tokens = B * T * (0.5 if case["lengths"] else 1.0)  # lengths are drawn evenly from 0 to T
    qkv = e * tokens * (2 * Hk * Dk + Hv * Dv) + 8 * tokens * Hv
    o = e * B * T * Hv * Dv
    state = 4 * B * Hv * Dk * Dv
    flops = 7 * tokens * Hv * Dk * Dv  # decay, read, write and output of a state
    if case["kind"] != "train":
        return {"bytes": qkv + o + state * (1 + case["s0"]), "flops": flops}
    return {"bytes": 2 * (qkv + o) + 2 * state * (1 + case["s0"]), "flops": 3 * flops}


# ------------------------------------------------------------------- exact ---


def _act_and_slope(z, act):
    sig = torch.sigmoid(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return z * sig, sig * (1 + z * (1 - sig))
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    if act == "logsigmoid":
        return -torch.logaddexp(-z, torch.zeros_like(z)), torch.sigmoid(-z)
    return z, torch.ones_like(z)


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["kind"].startswith("linear"):
            x, w = s["x"].detach().double(), s["w"].detach().double()
            z = x @ w.t()
            if s["b"] is not None:
                z = z + s["b"].double()
            y, slope = _act_and_slope(z, case["act"])
            if s["r"] is not None:
                y = y + s["r"].double()
            if case["kind"] == "linear":
                return y
            dy = s["dy"].double()
            dz = dy * slope
            out = dict(y=y, dx=dz @ w, dw=dz.t() @ x)
            if s["b"] is not None:
                out["db"] = dz.sum(0)
            if s["r"] is not None:
                out["dr"] = dy
            return out
        return _exact_delta(s, case)


def _exact_delta(s, case):
    kind, rep = case["kind"], case["Hv"] // case["Hk"]
    q, k, v, g, beta = (s[n].detach().double() for n in ("q", "k", "v", "g", "beta"))
    if kind == "step":
        q, k, v, g, beta = (t[:, None] for t in (q, k, v, g, beta))
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    cq = torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) if case["normalize"] else torch.ones_like(q[..., :1])
    ck = torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS) if case["normalize"] else torch.ones_like(k[..., :1])
    qn, kn = q * cq, k * ck
    qh = qn.repeat_interleave(rep, 2) * s["scale"]
    kh = kn.repeat_interleave(rep, 2)
    a = g.exp()
    S = s["state"][s["slots"].long()].double() if kind == "step" else (
        torch.zeros(B, Hv, Dk, Dv, dtype=torch.float64, device=q.device) if s["s0"] is None else s["s0"].detach().double())
    live = torch.ones(B, T, dtype=torch.bool, device=q.device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=q.device)[None, :] < s["lengths"][:, None]
    train = kind == "train"
    o = torch.zeros_like(v)
    before, errs = [], []
    for t in range(T):
        m = live[:, t, None, None, None]
        if train:
            before.append(S)
        Sd = S * a[:, t, :, None, None]
        e = v[:, t] - torch.einsum("bhd,bhde->bhe", kh[:, t], Sd)
        errs.append(e)
        Sn = Sd + kh[:, t, :, :, None] * (beta[:, t, :, None] * e)[:, :, None, :]
        S = torch.where(m, Sn, S)
        o[:, t] = torch.where(m[..., 0], torch.einsum("bhd,bhde->bhe", qh[:, t], S), 0.0)
    if kind == "step":
        pool = s["state"].double()
        pool[s["slots"].long()] = S
        return dict(o=o[:, 0], state=pool)
    out = dict(o=o, state=S)
    if not train:
        return out
    do = torch.where(live[..., None, None], s["do"].double(), 0.0)
    dS = s["ds"].double()
    dq, dk, dv = torch.zeros_like(qh), torch.zeros_like(kh), torch.zeros_like(v)
    dg, db = torch.zeros_like(g), torch.zeros_like(beta)
    for t in range(T - 1, -1, -1):
        m = live[:, t, None, None, None]
        S0, at, bt, kt, e = before[t], a[:, t, :, None, None], beta[:, t, :, None], kh[:, t], errs[t]
        u = bt * e
        St = at * S0 + kt[..., None] * u[..., None, :]
        D = dS + qh[:, t, :, :, None] * do[:, t, :, None, :]
        dq[:, t] = torch.einsum("bhde,bhe->bhd", St, do[:, t])
        du = torch.einsum("bhd,bhde->bhe", kt, D)
        de = bt * du
        dkt = torch.einsum("bhde,bhe->bhd", D, u) - torch.einsum("bhde,bhe->bhd", at * S0, de)
        D = D - kt[..., None] * de[..., None, :]
        dk[:, t] = torch.where(m[..., 0], dkt, 0.0)
        dv[:, t] = torch.where(m[..., 0], de, 0.0)
        db[:, t] = torch.where(m[..., 0, 0], (du * e).sum(-1), 0.0)
        dg[:, t] = torch.where(m[..., 0, 0], (at * S0 * D).sum((-1, -2)), 0.0)
        dS = torch.where(m, at * D, dS)
    dq = (dq * s["scale"]).unflatten(2, (Hk, rep)).sum(3)
    dk = dk.unflatten(2, (Hk, rep)).sum(3)
    if case["normalize"]:
        dq = cq * (dq - qn * (qn * dq).sum(-1, keepdim=True))
        dk = ck * (dk - kn * (kn * dk).sum(-1, keepdim=True))
    out.update(dq=dq, dk=dk, dv=dv, dg=dg, dbeta=db)
    if s["s0"] is not None:
        out["ds0"] = dS
    return out
