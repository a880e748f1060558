"""The selective state scan and its short causal convolution, as cases that can be timed.

A selective scan keeps a [P, N] state per head, as the framework's linear memory does, but each
token chooses how much of the state stays and how strongly it writes:
``S_t = exp(d_t A) S_{t-1} + d_t x_t k_t^T``, ``y_t = S_t q_t + D x_t``.  The convolution in front
of it mixes the last few tokens of each channel.  Both are called on whole prompts, in training
(with every gradient) and for single tokens with their states kept between calls.

``run`` computes a case in plain float32 torch operations, or, with ``own`` set, through this
framework's entry points.  ``exact`` follows the definition token by token in float64.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_DEV = "cuda"


def listed():
    return [
        # Prompts of eight users through the convolution of a block of 32 heads of 64 values with one
        # shared key and query row of 128: its channels are values, keys and queries side by side.
        {"name": "conv_prompt_bf16", "op": "conv", "dtype": "bf16", "B": 8, "T": 2048, "C": 2304, "W": 4,
         "train": False, "ragged": False},
        # A padded batch of prompts of different lengths (one of them empty), half precision.
        {"name": "conv_ragged_f16", "op": "conv", "dtype": "f16", "B": 5, "T": 777, "C": 1000, "W": 3,
         "train": False, "ragged": True},
        # The same convolution's training step: output, final state and every gradient.
        {"name": "conv_train_bf16", "op": "conv", "dtype": "bf16", "B": 8, "T": 2048, "C": 2304, "W": 4,
         "train": True, "ragged": False},
        # One token of each of 256 served sequences.
        {"name": "conv_step_bf16", "op": "conv_step", "dtype": "bf16", "B": 256, "C": 2304, "W": 4},
        # One token of a single float32 sequence, where only latency counts.
        {"name": "conv_step_one_f32", "op": "conv_step", "dtype": "f32", "B": 1, "C": 640, "W": 4},
        # Prompts of eight users through the scan.
        {"name": "scan_prompt_bf16", "op": "scan", "dtype": "bf16", "B": 8, "T": 2048, "H": 32, "P": 64, "G": 1,
         "N": 128, "train": False, "ragged": False},
        # One long document: few heads in flight, a long walk.
        {"name": "scan_long_bf16", "op": "scan", "dtype": "bf16", "B": 1, "T": 32768, "H": 16, "P": 64, "G": 1,
         "N": 128, "train": False, "ragged": False},
        # A padded batch of different lengths (one of them empty), two groups, narrow keys, half precision.
        {"name": "scan_ragged_f16", "op": "scan", "dtype": "f16", "B": 5, "T": 777, "H": 12, "P": 64, "G": 2,
         "N": 64, "train": False, "ragged": True},
        # Training: outputs and all eight gradients.
        {"name": "scan_train_bf16", "op": "scan", "dtype": "bf16", "B": 8, "T": 2048, "H": 32, "P": 64, "G": 1,
         "N": 128, "train": True, "ragged": False},
        # Training of a float32 model of modest size, a length that is no multiple of any tile.
        {"name": "scan_train_f32", "op": "scan", "dtype": "f32", "B": 4, "T": 1000, "H": 8, "P": 64, "G": 2,
         "N": 64, "train": True, "ragged": False},
        # One token of each of 64 served sequences: the states are read and written once.
        {"name": "step_bf16", "op": "step", "dtype": "bf16", "B": 64, "H": 32, "P": 64, "G": 1, "N": 128},
        # One token of a single sequence of a small model.
        {"name": "step_one_bf16", "op": "step", "dtype": "bf16", "B": 1, "H": 8, "P": 64, "G": 1, "N": 64},
    ]


# ---------------------------------------------------------------------------
# Drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "conv":
        B, C = _log_int(rng, 1, 16), _log_int(rng, 48, 2304)
        T = _log_int(rng, 1, max(1, min(32768, 8 * 2048 * 2304 // (B * C))))
        return {"op": op, "dtype": dtype, "B": B, "T": T, "C": C, "W": rng.choice([2, 3, 4, 4]),
                "train": rng.random() < 0.5, "ragged": rng.random() < 0.3}
    if op == "conv_step":
        return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, 256), "C": _log_int(rng, 48, 2304),
                "W": rng.choice([2, 3, 4, 4])}
    G = rng.choice([1, 1, 1, 2, 4])
    H = G * _log_int(rng, 1, 32 // G)
    P, N = rng.choice([16, 32, 48, 64, 64, 64, 80, 128]), rng.choice([16, 32, 40, 64, 64, 96, 128, 128])
    if op == "step":
        return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, 64), "H": H, "P": P, "G": G, "N": N}
    B, train = _log_int(rng, 1, 8), rng.random() < 0.5
    T = _log_int(rng, 1, max(1, min(32768, 8 * 2048 * 32 * 64 // (B * H * max(P, 32)) // (1 if dtype == "bf16" else 4))))
    return {"op": op, "dtype": dtype, "B": B, "T": T, "H": H, "P": P, "G": G, "N": N, "train": train,
            "ragged": rng.random() < 0.3}


# ---------------------------------------------------------------------------
# Inputs

def _lengths(case, gen):
    if not case.get("ragged"):
        return None
    n = torch.randint(0, case["T"] + 1, (case["B"],), generator=gen, device=_DEV)
    n[0] = case["T"]
    if case["B"] > 1:
        n[-1] = 0
    return n


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=_DEV)

    s = {"case": case}
    B = case["B"]
    if case["op"] in ("conv", "conv_step"):
        C, W = case["C"], case["W"]
        # The convolution's usual start: uniform in +-1/sqrt(W).
        s["weight"] = ((torch.rand(C, W, generator=gen, device=_DEV) * 2 - 1) / math.sqrt(W)).to(dt)
        s["bias"] = ((torch.rand(C, generator=gen, device=_DEV) * 2 - 1) / math.sqrt(W)).to(dt)
        s["state"] = normal(B, W - 1, C).to(dt)
        if case["op"] == "conv_step":
            s["x"] = normal(B, C).to(dt)
            return s
        # The channels are a slice of a wider projection (gate in front, steps behind).
        wide = normal(B, case["T"], C + 136).to(dt)
        s["x"] = wide[..., 128:128 + C]
        s["lengths"] = _lengths(case, gen)
        if case["train"]:
            s["grads"] = (normal(B, case["T"], C).to(dt), normal(B, W - 1, C).to(dt))
            for k in ("x", "weight", "bias", "state"):
                s[k] = s[k].detach().requires_grad_()
        return s
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    T = case.get("T", 1)
    # What the convolution hands over: values, keys and queries side by side, through SiLU.
    rows = torch.nn.functional.silu(normal(B, T, H * P + 2 * G * N)).to(dt)
    s["values"] = rows[..., :H * P].unflatten(-1, (H, P))
    s["keys"] = rows[..., H * P:H * P + G * N].unflatten(-1, (G, N))
    s["queries"] = rows[..., H * P + G * N:].unflatten(-1, (G, N))
    # Step sizes of 0.001 to 0.1 around which the projection moves them, decay rates of 1 to 16.
    s["steps"] = (normal(B, T, H) * 0.5).to(dt)
    d0 = torch.exp(torch.rand(H, generator=gen, device=_DEV) * math.log(100.0) + math.log(0.001))
    s["step_bias"] = d0 + torch.log(-torch.expm1(-d0))
    s["rates"] = -(1 + 15 * torch.rand(H, generator=gen, device=_DEV))
    s["skip"] = 1 + 0.1 * normal(H)
    s["memory"] = 0.2 * normal(B, H, P, N)
    if case["op"] == "step":
        for k in ("values", "keys", "queries", "steps"):
            s[k] = s[k][:, 0]
        return s
    s["lengths"] = _lengths(case, gen)
    if case["train"]:
        s["grads"] = (normal(B, T, H, P).to(dt), 0.1 * normal(B, H, P, N))
        for k in _SCAN_LEAVES:
            s[k] = s[k].detach().requires_grad_()
    return s


_CONV_LEAVES = ("x", "weight", "bias", "state")
_SCAN_LEAVES = ("keys", "values", "queries", "steps", "rates", "memory", "skip", "step_bias")


# ---------------------------------------------------------------------------
# Plain forms: float32 torch operations, rounded once at the end

def _plain_conv(x, weight, bias, state, lengths):
    B, T, C = x.shape
    W = weight.size(1)
    xf, wf = x.float(), weight.float()
    t = torch.arange(T, device=x.device)
    if lengths is not None:
        xf = torch.where((t < lengths[:, None])[..., None], xf, 0.0)
    full = torch.cat([state.float(), xf], 1)
    pre = bias.float() + (full.unfold(1, W, 1) * wf).sum(-1)
    out = pre * torch.sigmoid(pre)
    if lengths is None:
        return out.to(x.dtype), full[:, T:].to(x.dtype)
    out = torch.where((t < lengths[:, None])[..., None], out, 0.0)
    last = lengths[:, None] + torch.arange(W - 1, device=x.device)
    return out.to(x.dtype), full.gather(1, last[..., None].expand(B, W - 1, C)).to(x.dtype)


def _plain_step_size(steps, step_bias):
    z = steps.float() + step_bias
    return torch.where(z > 20, z, torch.log1p(torch.exp(z.clamp(max=20))))


def _plain_scan(keys, values, queries, steps, rates, memory, skip, step_bias, lengths, L=64):
    B, T, H, P = values.shape
    G, N = keys.shape[2:]
    d = _plain_step_size(steps, step_bias)
    x, k, q = values.float(), keys.float(), queries.float()
    if lengths is not None:
        live = (torch.arange(T, device=x.device) < lengths[:, None])[..., None]
        d, x = torch.where(live, d, 0.0), torch.where(live[..., None], x, 0.0)
        k, q = torch.where(live[..., None], k, 0.0), torch.where(live[..., None], q, 0.0)
    c = -(-T // L)
    pad = c * L - T
    rows = lambda v: torch.nn.functional.pad(v, (0, 0, 0, 0, 0, pad)).unflatten(1, (c, L))  # noqa: E731
    dp = torch.nn.functional.pad(d, (0, 0, 0, pad)).unflatten(1, (c, L)).permute(0, 3, 1, 2)     # B H c L
    xh = rows(x).permute(0, 3, 1, 2, 4)                                                          # B H c L P
    kg, qg = rows(k).permute(0, 3, 1, 2, 4), rows(q).permute(0, 3, 1, 2, 4)                      # B G c L N
    cum = (dp.double() * rates.double()[:, None, None]).cumsum(-1)                               # log decay
    lower = torch.ones(L, L, dtype=torch.bool, device=x.device).tril()
    decay = torch.exp(torch.where(lower, cum[..., :, None] - cum[..., None, :], -math.inf)).float()
    heads = lambda v: v.repeat_interleave(H // G, dim=1)  # noqa: E731
    mix = heads(torch.matmul(qg, kg.transpose(-1, -2))) * decay * dp[..., None, :]
    # Each chunk's own contribution to the state, then the state at every chunk's start.
    tail = torch.exp(cum[..., -1:] - cum).float() * dp
    kh, qh = heads(kg), heads(qg)
    local = torch.matmul((xh * tail[..., None]).transpose(-1, -2), kh)                           # B H c P N
    total = torch.nn.functional.pad(cum[..., -1].cumsum(-1), (1, 0))                             # B H c+1
    n = torch.arange(c + 1, device=x.device)
    carry = torch.exp(torch.where(n[:, None] > n[None, :-1], total[..., :, None] - total[..., None, 1:],
                                  -math.inf)).float()
    states = torch.matmul(carry, local.flatten(-2)).unflatten(-1, (P, N))
    states = states + torch.exp(total).float()[..., None, None] * memory[:, :, None]
    y = torch.matmul(mix, xh)
    y = y + torch.exp(cum).float()[..., None] * torch.matmul(qh, states[:, :, :-1].transpose(-1, -2))
    y = y.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :T] + skip[:, None] * x
    return y.to(values.dtype), states[:, :, -1]


def _plain_step(keys, values, queries, steps, rates, memory, skip, step_bias):
    H, G = values.size(1), keys.size(1)
    d = _plain_step_size(steps, step_bias)
    k, q = (v.float().repeat_interleave(H // G, dim=1) for v in (keys, queries))
    x = values.float()
    new = memory * torch.exp(d * rates)[..., None, None] + (d[..., None] * x)[..., None] * k[:, :, None]
    y = (new * q[:, :, None]).sum(-1) + skip[:, None] * x
    return y.to(values.dtype), new


# ---------------------------------------------------------------------------
# One pass

def _conv(s):
    if own:
        from rnn_with_grm_amd import cuda_ops
        return cuda_ops.cuda_short_conv(s["x"], s["weight"], s["bias"], s["state"], activation="silu",
                                        lengths=s["lengths"])
    return _plain_conv(s["x"], s["weight"], s["bias"], s["state"], s["lengths"])


def _scan(s):
    if own:
        from rnn_with_grm_amd import cuda_ops
        return cuda_ops.cuda_selective_scan(s["keys"], s["values"], s["queries"], s["steps"], s["rates"], s["memory"],
                                            skip=s["skip"], step_bias=s["step_bias"], softplus=True,
                                            lengths=s["lengths"])
    return _plain_scan(s["keys"], s["values"], s["queries"], s["steps"], s["rates"], s["memory"], s["skip"],
                       s["step_bias"], s["lengths"])


def run(s):
    op = s["case"]["op"]
    if op == "conv_step":
        if own:
            from rnn_with_grm_amd import cuda_ops
            return cuda_ops.cuda_short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu")
        out, state = _plain_conv(s["x"][:, None], s["weight"], s["bias"], s["state"], None)
        return out[:, 0], state
    if op == "step":
        if own:
            from rnn_with_grm_amd import cuda_ops
            return cuda_ops.cuda_selective_step(s["keys"], s["values"], s["queries"], s["steps"], s["rates"],
                                                s["memory"], skip=s["skip"], step_bias=s["step_bias"], softplus=True)
        return _plain_step(s["keys"], s["values"], s["queries"], s["steps"], s["rates"], s["memory"], s["skip"],
                           s["step_bias"])
    one = _conv if op == "conv" else _scan
    if not s["case"]["train"]:
        return one(s)
    leaves = [s[k] for k in (_CONV_LEAVES if op == "conv" else _SCAN_LEAVES)]
    outs = one(s)
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, s["grads"]))


# ---------------------------------------------------------------------------
# What a pass cannot do without

def work(case):
    es, B, T = _SIZE[case["dtype"]], case["B"], case.get("T", 1)
    train = bool(case.get("train"))
    if case["op"] in ("conv", "conv_step"):
        C, W = case["C"], case["W"]
        rows, par, state = B * T * C * es, C * (W + 1) * es, B * (W - 1) * C * es
        if train:  # x and the output's gradient read, the output and x's gradient written
            return {"bytes": 4 * rows + 2 * par + 4 * state, "flops": B * T * C * (6 * W + 20)}
        return {"bytes": 2 * rows + par + 2 * state, "flops": B * T * C * (2 * W + 5)}
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    val, key, stp, state, par = B * T * H * P * es, B * T * G * N * es, B * T * H * es, B * H * P * N * 4, 12 * H
    cells = B * T * H * P * N  # state elements over all tokens: decay, write and read of each
    if train:
        return {"bytes": 4 * val + 4 * key + 2 * stp + 4 * state + 2 * par, "flops": 5 * cells + 12 * cells}
    return {"bytes": 2 * val + 2 * key + stp + 2 * state + par, "flops": 5 * cells}


# ---------------------------------------------------------------------------
# The definition in float64, token by token

def _live(case, lengths):
    B, T = case["B"], case.get("T", 1)
    n = torch.full((B,), T, device=_DEV) if lengths is None else lengths
    return torch.arange(T, device=_DEV)[None] < n[:, None], n


def _exact_conv(case, s):
    x, w, b, st = (s[k].detach().double() for k in _CONV_LEAVES)
    if case["op"] == "conv_step":
        x = x[:, None]
    B, T, C = x.shape
    W = w.size(1)
    live, n = _live(case, s.get("lengths"))
    x = x.masked_fill(~live[..., None], 0.0)
    full = torch.cat([st, x], 1)
    pre = b.expand(B, T, C).clone()
    for i in range(W):
        pre += full[:, i:i + T] * w[:, i]
    sig = 1 / (1 + torch.exp(-pre))
    out = (pre * sig).masked_fill(~live[..., None], 0.0)
    state = torch.stack([full[i, int(m):int(m) + W - 1] for i, m in enumerate(n.tolist())])
    if case["op"] == "conv_step":
        return out[:, 0], state
    if not case["train"]:
        return out, state
    dy, ds = (g.double() for g in s["grads"])
    g = (dy * sig * (1 + pre * (1 - sig))).masked_fill(~live[..., None], 0.0)
    dfull = torch.zeros_like(full)
    dw = torch.zeros_like(w)
    for i in range(W):
        dfull[:, i:i + T] += g * w[:, i]
        dw[:, i] = (g * full[:, i:i + T]).sum((0, 1))
    for i, m in enumerate(n.tolist()):
        dfull[i, int(m):int(m) + W - 1] += ds[i]
    return out, state, dfull[:, W - 1:].masked_fill(~live[..., None], 0.0), dw, g.sum((0, 1)), dfull[:, :W - 1]


def _exact_scan(case, s, train):
    k, x, q, z, A, S, D, zb = (s[n].detach().double() for n in _SCAN_LEAVES)
    if case["op"] == "step":
        k, x, q, z = (v[:, None] for v in (k, x, q, z))
    B, T, H, P = x.shape
    G, N = k.shape[2:]
    live, _ = _live(case, s.get("lengths"))
    z = z + zb
    d = torch.where(z > 40, z, torch.log1p(torch.exp(z.clamp(max=40)))) * live[..., None]
    x = x.masked_fill(~live[..., None, None], 0.0)
    k, q = (v.masked_fill(~live[..., None, None], 0.0) for v in (k, q))
    a = torch.exp(d * A)
    group = lambda v: v.reshape(B, G, H // G, P, v.size(-1))  # noqa: E731

    def advance(S, t):
        wr = (d[:, t, :, None] * x[:, t])[..., None]
        return S * a[:, t, :, None, None] + (group(wr) * k[:, t, :, None, None]).reshape(B, H, P, N)

    y = torch.zeros_like(x)
    block = max(1, min(64, int(2e9 // (S.numel() * 8))))
    marks = []
    for t in range(T):
        if train and t % block == 0:
            marks.append(S)
        S = advance(S, t)
        y[:, t] = (group(S) * q[:, t, :, None, None]).sum(-1).reshape(B, H, P)
    y = y + D[:, None] * x
    if case["op"] == "step":
        return y[:, 0], S
    if not train:
        return y, S
    dy, dS = (g.double() for g in s["grads"])
    dy = dy.masked_fill(~live[..., None, None], 0.0)
    dk, dq, dx, dl, dd = (torch.zeros_like(v) for v in (k, q, x, d, d))
    for m in range(len(marks) - 1, -1, -1):
        t0, t1 = m * block, min(T, (m + 1) * block)
        states = [marks[m]]
        for t in range(t0, t1):
            states.append(advance(states[-1], t))
        for t in range(t1 - 1, t0 - 1, -1):
            dyt = group(dy[:, t][..., None])
            dq[:, t] = (group(states[t - t0 + 1]) * dyt).sum((2, 3))
            dS = dS + (dyt * q[:, t, :, None, None]).reshape(B, H, P, N)
            u = group((d[:, t, :, None] * x[:, t])[..., None])
            dk[:, t] = (group(dS) * u).sum((2, 3))
            du = (group(dS) * k[:, t, :, None, None]).sum(-1).reshape(B, H, P)
            dx[:, t] = du * d[:, t, :, None]
            dd[:, t] = (du * x[:, t]).sum(-1)
            dl[:, t] = a[:, t] * (dS * states[t - t0]).sum((-1, -2))
            dS = dS * a[:, t, :, None, None]
    dx = dx + D[:, None] * dy
    dd = (dd + dl * A) * live[..., None]
    dz = dd / (1 + torch.exp(-z))
    return y, S, dk, dx, dq, dz, (dl * d).sum((0, 1)), dS, (dy * x).sum((0, 1, 3)), dz.sum((0, 1))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("conv", "conv_step"):
            return _exact_conv(case, s)
        return _exact_scan(case, s, bool(case.get("train")))
