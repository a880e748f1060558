"""The gated delta rule and the group norm behind it, as cases that can be timed.

The delta rule keeps a [P, N] state per head, as the framework's other linear memories do, but a
token first takes out what the state holds under its key and then writes:
``u_t = b_t (v_t - a_t M_{t-1} k_t)``, ``M_t = a_t M_{t-1} + u_t k_t^T``, ``h_t = M_t q_t`` with
``a_t = exp(log_decay_t)``.  The group norm takes each head's outputs of a token to unit scale and
multiplies them with an activated gate.  Both are called on whole prompts, in training (with every
gradient) and for single tokens.

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
        # Prompts of eight users: 16 heads of 128 x 128 states, a key row for every two of them.
        {"name": "delta_prompt_bf16", "op": "delta", "dtype": "bf16", "B": 8, "T": 2048, "H": 16, "P": 128, "G": 8,
         "N": 128, "train": False, "ragged": False},
        # One long document: few heads in flight, a long walk.
        {"name": "delta_long_bf16", "op": "delta", "dtype": "bf16", "B": 1, "T": 32768, "H": 16, "P": 128, "G": 16,
         "N": 128, "train": False, "ragged": False},
        # A padded batch of different lengths (one of them empty), narrow states, half precision.
        {"name": "delta_ragged_f16", "op": "delta", "dtype": "f16", "B": 5, "T": 777, "H": 12, "P": 64, "G": 12,
         "N": 64, "train": False, "ragged": True},
        # Training: outputs and all six gradients.
        {"name": "delta_train_bf16", "op": "delta", "dtype": "bf16", "B": 8, "T": 2048, "H": 16, "P": 128, "G": 8,
         "N": 128, "train": True, "ragged": False},
        # Training of a float32 model of modest size, a length that is no multiple of any tile.
        {"name": "delta_train_f32", "op": "delta", "dtype": "f32", "B": 4, "T": 1000, "H": 8, "P": 64, "G": 2,
         "N": 64, "train": True, "ragged": False},
        # One token of each of 64 served sequences: the states are read and written once.
        {"name": "delta_step_bf16", "op": "step", "dtype": "bf16", "B": 64, "H": 16, "P": 128, "G": 8, "N": 128},
        # One token of a single sequence of a small model, where only latency counts.
        {"name": "delta_step_one_bf16", "op": "step", "dtype": "bf16", "B": 1, "H": 8, "P": 64, "G": 8, "N": 64},
        # The norm of those prompts' outputs, gated.
        {"name": "norm_prompt_bf16", "op": "norm", "dtype": "bf16", "rows": 16384, "groups": 16, "width": 128,
         "gate": True, "center": False, "train": False},
        # Its training step: output and every gradient.
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bf16", "rows": 16384, "groups": 16, "width": 128,
         "gate": True, "center": False, "train": True},
        # Groups of an odd width, centred, the activation on the norm itself, float32.
        {"name": "norm_train_odd_f32", "op": "norm", "dtype": "f32", "rows": 4000, "groups": 7, "width": 45,
         "gate": False, "center": True, "train": True},
        # One token of each of 64 served sequences.
        {"name": "norm_step_bf16", "op": "norm", "dtype": "bf16", "rows": 64, "groups": 16, "width": 128,
         "gate": True, "center": False, "train": False},
    ]


# ---------------------------------------------------------------------------
# Drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        width = rng.choice([_log_int(rng, 2, 512), 8 * _log_int(rng, 1, 64), 64, 128])
        groups = _log_int(rng, 1, max(1, 2048 // width))
        rows = _log_int(rng, 1, max(1, 16384 * 2048 // (groups * max(width, 32)) // (1 if dtype != "f32" else 2)))
        return {"op": op, "dtype": dtype, "rows": min(rows, 65536), "groups": groups, "width": width,
                "gate": rng.random() < 0.6, "center": rng.random() < 0.5, "train": rng.random() < 0.5}
    G = rng.choice([1, 2, 4, 8, 16])
    H = G * rng.choice([n for n in (1, 1, 2, 3, 4, 8) if G * n <= 16])
    P, N = rng.choice([16, 32, 48, 64, 64, 80, 128, 128]), rng.choice([16, 32, 40, 64, 64, 96, 128, 128])
    if op == "step":
        return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, 64), "H": H, "P": P, "G": G, "N": N}
    B, train = _log_int(rng, 1, 8), rng.random() < 0.5
    cells = 8 * 2048 * 16 * 128 // (1 if dtype == "bf16" else 4)
    T = _log_int(rng, 1, max(1, min(32768 if not train else 4096, cells // (B * H * max(P, N)))))
    return {"op": op, "dtype": dtype, "B": B, "T": T, "H": H, "P": P, "G": G, "N": N, "train": train,
            "ragged": rng.random() < 0.3}


# ---------------------------------------------------------------------------
# Inputs

_DELTA_LEAVES = ("keys", "values", "queries", "strengths", "log_decays", "memory")
_NORM_LEAVES = ("x", "weight", "bias", "gate")


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
    if case["op"] == "norm":
        R, C = case["rows"], case["groups"] * case["width"]
        # The memory's outputs, of a scale that differs from group to group, and a slice of the projection as gate.
        scale = torch.exp(normal(R, case["groups"], 1)) * 0.1
        s["x"] = ((normal(R, case["groups"], case["width"]) + 0.3) * scale).reshape(R, C).to(dt)
        s["weight"] = (1 + 0.1 * normal(C)).to(dt)
        s["bias"] = (0.1 * normal(C)).to(dt) if case["center"] else None
        s["gate"] = normal(R, C + 64).to(dt)[:, 64:] if case["gate"] else None
        if case["train"]:
            s["grads"] = (normal(R, C).to(dt),)
            for k in _NORM_LEAVES:
                s[k] = None if s[k] is None else s[k].detach().requires_grad_()
        return s
    B, H, P, G, N = case["B"], case["H"], case["P"], case["G"], case["N"]
    T = case.get("T", 1)
    # What a projection hands over: keys and queries of unit length, values beside each other in one row.
    s["keys"] = torch.nn.functional.normalize(normal(B, T, G, N), dim=-1).to(dt)
    s["queries"] = torch.nn.functional.normalize(normal(B, T, G, N), dim=-1).to(dt)
    s["values"] = normal(B, T, H * P + 64).to(dt)[..., 64:].unflatten(-1, (H, P))
    s["strengths"] = torch.sigmoid(normal(B, T, H)).to(dt)
    # Rates of 1 to 16 and steps of 0.001 to 0.1 around which the projection moves them.
    d0 = torch.exp(torch.rand(H, generator=gen, device=_DEV) * math.log(100.0) + math.log(0.001))
    bias = d0 + torch.log(-torch.expm1(-d0))
    rates = 1 + 15 * torch.rand(H, generator=gen, device=_DEV)
    s["log_decays"] = -rates * torch.nn.functional.softplus(0.5 * normal(B, T, H) + bias)
    s["memory"] = 0.2 * normal(B, H, P, N)
    if case["op"] == "step":
        for k in ("values", "keys", "queries", "strengths", "log_decays"):
            s[k] = s[k][:, 0]
        return s
    s["lengths"] = _lengths(case, gen)
    if case["train"]:
        s["grads"] = (normal(B, T, H, P).to(dt), 0.1 * normal(B, H, P, N))
        for k in _DELTA_LEAVES:
            s[k] = s[k].detach().requires_grad_()
    return s


# ---------------------------------------------------------------------------
# Plain forms: float32 torch operations, rounded once at the end

def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower triangular matrices whose size is a power of two: blocks of twice the size from
    the inverses of their two diagonal blocks."""
    n = A.size(-1)
    inv = torch.ones(*A.shape[:-2], n, 1, 1, dtype=A.dtype, device=A.device)
    while inv.size(-3) > 1:
        m, w = inv.size(-3) // 2, inv.size(-1)
        low = A.unflatten(-1, (m, 2 * w)).unflatten(-3, (m, 2 * w)).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)[..., w:, :w]
        top, end = inv.unflatten(-3, (m, 2)).unbind(-3)
        below = -torch.matmul(torch.matmul(end, low), top)
        inv = torch.cat([torch.cat([top, torch.zeros_like(top)], -1), torch.cat([below, end], -1)], -2)
    return inv.squeeze(-3)


def _plain_delta(keys, values, queries, strengths, log_decays, memory, lengths, L=64):
    B, T, H, P = values.shape
    G = keys.size(2)
    b, g = strengths.float(), log_decays.double()
    v, k, q = values.float(), keys.float(), queries.float()
    if lengths is not None:
        live = (torch.arange(T, device=v.device) < lengths[:, None])[..., None]
        b, g = torch.where(live, b, 0.0), torch.where(live, g, 0.0)
        v, k, q = (torch.where(live[..., None], t, 0.0) for t in (v, k, q))
    c = -(-T // L)
    pad = c * L - T
    rows = lambda t: torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).unflatten(1, (c, L)).permute(0, 3, 1, 2, 4)  # noqa: E731
    each = lambda t: torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(1, (c, L)).permute(0, 3, 1, 2)  # noqa: E731
    vh, kg, qg, bh = rows(v), rows(k), rows(q), each(b)[..., None]                # B H c L P, B G c L N
    cum = each(g).cumsum(-1)                                                      # B H c L
    lower = torch.ones(L, L, dtype=torch.bool, device=v.device).tril()
    decay = torch.exp(torch.where(lower, cum[..., :, None] - cum[..., None, :], -math.inf)).float()
    heads = lambda t: t.repeat_interleave(H // G, dim=1)  # noqa: E731
    mix = heads(torch.matmul(qg, kg.transpose(-1, -2))) * decay
    solve = _unit_lower_inverse((heads(torch.matmul(kg, kg.transpose(-1, -2))) * decay * bh).tril(-1))
    kh, qh = heads(kg), heads(qg)
    start = torch.exp(cum).float()[..., None]
    own_part, of_state = torch.matmul(solve, bh * vh), torch.matmul(solve, bh * start * kh)
    tail = torch.exp(cum[..., -1:] - cum).float()[..., None] * kh
    end = torch.exp(cum[..., -1]).float()[..., None, None]
    state, out = memory, []
    for i in range(c):
        turned = state.transpose(-1, -2)
        u = own_part[:, :, i] - torch.matmul(of_state[:, :, i], turned)
        out.append(torch.matmul(start[:, :, i] * qh[:, :, i], turned) + torch.matmul(mix[:, :, i], u))
        state = end[:, :, i] * state + torch.matmul(u.transpose(-1, -2), tail[:, :, i])
    y = torch.stack(out, 2).permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :T]
    return y.to(values.dtype), state


def _plain_step(keys, values, queries, strengths, log_decays, memory):
    H, G = values.size(1), keys.size(1)
    k, q = (t.float().repeat_interleave(H // G, dim=1)[:, :, None] for t in (keys, queries))
    kept = memory * torch.exp(log_decays.float())[..., None, None]
    u = strengths.float()[..., None] * (values.float() - (kept * k).sum(-1))
    new = kept + u[..., None] * k
    return (new * q).sum(-1).to(values.dtype), new


def _plain_norm(x, weight, bias, gate, groups, center, eps=1e-5):
    xf = x.float().unflatten(-1, (groups, -1))
    if center:
        xf = xf - xf.mean(-1, keepdim=True)
    y = (xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)).flatten(-2) * weight.float()
    if bias is not None:
        y = y + bias.float()
    z = y if gate is None else gate.float()
    act = z * torch.sigmoid(z)
    return (act if gate is None else y * act).to(x.dtype)


# ---------------------------------------------------------------------------
# One pass

def _delta(s):
    if own:
        from rnn_with_grm_amd import cuda_ops
        return cuda_ops.cuda_delta_scan(s["keys"], s["values"], s["queries"], s["strengths"], s["log_decays"],
                                        s["memory"], lengths=s["lengths"])
    return _plain_delta(s["keys"], s["values"], s["queries"], s["strengths"], s["log_decays"], s["memory"],
                        s["lengths"])


def _norm(s):
    case = s["case"]
    if own:
        from rnn_with_grm_amd import cuda_ops
        return (cuda_ops.cuda_group_norm(s["x"], case["groups"], s["weight"], s["bias"], s["gate"], activation="silu",
                                         center=case["center"]),)
    return (_plain_norm(s["x"], s["weight"], s["bias"], s["gate"], case["groups"], case["center"]),)


def run(s):
    op = s["case"]["op"]
    if op == "step":
        if own:
            from rnn_with_grm_amd import cuda_ops
            return cuda_ops.cuda_delta_step(s["keys"], s["values"], s["queries"], s["strengths"], s["log_decays"],
                                            s["memory"])
        return _plain_step(s["keys"], s["values"], s["queries"], s["strengths"], s["log_decays"], s["memory"])
    one = _delta if op == "delta" else _norm
    if not s["case"]["train"]:
        return one(s)
    leaves = [s[k] for k in (_DELTA_LEAVES if op == "delta" else _NORM_LEAVES) if s[k] is not None]
    outs = one(s)
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, s["grads"]))


# ---------------------------------------------------------------------------
# What a pass cannot do without

def work(case):
    es, train = _SIZE[case["dtype"]], bool(case.get("train"))
    if case["op"] == "norm":
        C = case["groups"] * case["width"]
        rows, par, ins = case["rows"] * C * es, C * es * (2 if case["center"] else 1), 2 if case["gate"] else 1
        if train:  # x, the gate and the output's gradient read, the output and their gradients written
            return {"bytes": (2 * ins + 2) * rows + 2 * par, "flops": case["rows"] * C * 35}
        return {"bytes": (ins + 1) * rows + par, "flops": case["rows"] * C * 12}
    B, T, H, P, G, N = case["B"], case.get("T", 1), case["H"], case["P"], case["G"], case["N"]
    val, key, stp, state = B * T * H * P * es, B * T * G * N * es, B * T * H * (es + 4), B * H * P * N * 4
    cells = B * T * H * P * N  # state elements over all tokens: decay, read, write and query of each
    if train:
        return {"bytes": 4 * val + 4 * key + 2 * stp + 4 * state, "flops": 7 * cells + 18 * cells}
    return {"bytes": 2 * val + 2 * key + stp + 2 * state, "flops": 7 * cells}


# ---------------------------------------------------------------------------
# The definition in float64, token by token

def _exact_delta(case, s, train):
    k, v, q, b, g, M = (s[n].detach().double() for n in _DELTA_LEAVES)
    if case["op"] == "step":
        k, v, q, b, g = (t[:, None] for t in (k, v, q, b, g))
    B, T, H, P = v.shape
    G, N = k.shape[2:]
    n = torch.full((B,), T, device=_DEV) if s.get("lengths") is None else s["lengths"]
    dead = torch.arange(T, device=_DEV)[None] >= n[:, None]
    b, a = b.masked_fill(dead[..., None], 0.0), torch.exp(g.masked_fill(dead[..., None], 0.0))
    k, v, q = (t.masked_fill(dead[..., None, None], 0.0) for t in (k, v, q))
    wide = lambda t: t[:, :, None].expand(B, G, H // G, N).reshape(B, H, 1, N)  # noqa: E731

    def advance(M, t):
        kept, kt = M * a[:, t, :, None, None], wide(k[:, t])
        miss = v[:, t] - (kept * kt).sum(-1)
        u = b[:, t, :, None] * miss
        return kept + u[..., None] * kt, kept, miss, u

    y = torch.zeros_like(v)
    block = max(1, min(64, int(4e9 // (M.numel() * 8))))
    marks = []
    for t in range(T):
        if train and t % block == 0:
            marks.append(M)
        M = advance(M, t)[0]
        y[:, t] = (M * wide(q[:, t])).sum(-1)
    if case["op"] == "step":
        return y[:, 0], M
    if not train:
        return y, M
    dy, dM = (t.double() for t in s["grads"])
    dy = dy.masked_fill(dead[..., None, None], 0.0)
    dk, dq, dv, db, dg = (torch.zeros_like(t) for t in (k, q, v, b, g))
    shared = lambda t: t.reshape(B, G, H // G, N).sum(2)  # noqa: E731
    for m in range(len(marks) - 1, -1, -1):
        t0, t1 = m * block, min(T, (m + 1) * block)
        states = [marks[m]]
        for t in range(t0, t1):
            states.append(advance(states[-1], t)[0])
        for t in range(t1 - 1, t0 - 1, -1):
            new, kept, miss, u = advance(states[t - t0], t)
            dyt, kt = dy[:, t][..., None], wide(k[:, t])
            dM = dM + dyt * wide(q[:, t])
            du = (dM * kt).sum(-1)
            dmiss = b[:, t, :, None] * du
            dq[:, t] = shared((new * dyt).sum(-2))
            db[:, t] = (du * miss).sum(-1)
            dv[:, t] = dmiss
            dk[:, t] = shared((dM * u[..., None] - kept * dmiss[..., None]).sum(-2))
            dkept = dM - dmiss[..., None] * kt
            dg[:, t] = (dkept * kept).sum((-1, -2))
            dM = dkept * a[:, t, :, None, None]
    alive = ~dead[..., None]
    return y, M, dk * alive[..., None], dv, dq, db * alive, dg * alive, dM


def _exact_norm(case, s, eps=1e-5):
    x, w, b, z = (None if s[n] is None else s[n].detach().double() for n in _NORM_LEAVES)
    R, groups, width = case["rows"], case["groups"], case["width"]
    xg = x.view(R, groups, width)
    mean = xg.sum(-1, keepdim=True) / width if case["center"] else torch.zeros_like(xg[..., :1])
    r = 1 / torch.sqrt(((xg - mean) ** 2).sum(-1, keepdim=True) / width + eps)
    nrm = ((xg - mean) * r).view(R, -1)
    y = nrm * w + (0 if b is None else b)
    arg = y if z is None else z
    sig = 1 / (1 + torch.exp(-arg))
    act, slope = arg * sig, sig * (1 + arg * (1 - sig))
    out = act if z is None else y * act
    if not case["train"]:
        return (out,)
    do = s["grads"][0].double()
    dy = do * slope if z is None else do * act
    dn = (dy * w).view(R, groups, width)
    ng = nrm.view(R, groups, width)
    dx = dn - ng * (dn * ng).sum(-1, keepdim=True) / width
    if case["center"]:
        dx = dx - dn.sum(-1, keepdim=True) / width
    grads = [(dx * r).reshape(R, -1), (dy * nrm).sum(0)]
    if b is not None:
        grads.append(dy.sum(0))
    if z is not None:
        grads.append(do * y * slope)
    return (out, *grads)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(case, s)
        return _exact_delta(case, s, bool(case.get("train")))
