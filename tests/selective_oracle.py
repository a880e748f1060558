"""Float64 definitions of the short convolution and the selective scan, token by token.

Each takes tensors of any floating type and returns float64 results on the CPU; gradients come from
autograd through these definitions (or from differences of them)."""

import torch


def to64(*tensors, grad=False):
    return [None if t is None else t.detach().to("cpu", torch.float64).requires_grad_(grad) for t in tensors]


def lengths_of(lengths, batch, seq_len):
    return [seq_len] * batch if lengths is None else [min(max(int(n), 0), seq_len) for n in lengths.tolist()]


def short_conv(x, weight, bias, state, lengths, silu):
    B, T, C = x.shape
    W = weight.shape[1]
    outs, states = [], []
    for b, n in enumerate(lengths_of(lengths, B, T)):
        rows = list(torch.zeros(W - 1, C, dtype=torch.float64) if state is None else state[b]) + list(x[b, :n])
        out = []
        for t in range(T):
            if t >= n:
                out.append(torch.zeros(C, dtype=torch.float64))
                continue
            pre = sum(weight[:, w] * rows[t + w] for w in range(W))
            pre = pre if bias is None else pre + bias
            out.append(pre / (1 + torch.exp(-pre)) if silu else pre)
        outs.append(torch.stack(out) if out else 1.0 * x[b])
        states.append(torch.stack(rows[n:n + W - 1]))
    return torch.stack(outs), torch.stack(states)


def selective_scan(keys, values, queries, steps, rates, memory, skip, step_bias, lengths, softplus):
    B, T, H, P = values.shape
    G, N = keys.shape[2:]
    hidden, finals = [], []
    for b, n in enumerate(lengths_of(lengths, B, T)):
        M = torch.zeros(H, P, N, dtype=torch.float64) if memory is None else memory[b]
        rows = []
        for t in range(T):
            if t >= n:
                rows.append(torch.zeros(H, P, dtype=torch.float64))
                continue
            d = steps[b, t] if step_bias is None else steps[b, t] + step_bias
            if softplus:
                d = torch.logaddexp(d, torch.zeros_like(d))
            k, q = (v[b, t].repeat_interleave(H // G, 0) for v in (keys, queries))
            rate = rates if rates.ndim == 1 else rates[b, t]  # [B, T, H]: one a token, whose gradients are apart
            M = torch.exp(d * rate)[:, None, None] * M + (d[:, None] * values[b, t])[..., None] * k[:, None]
            h = (M * q[:, None]).sum(-1)
            rows.append(h if skip is None else h + skip[:, None] * values[b, t])
        hidden.append(torch.stack(rows) if rows else 1.0 * values[b])
        finals.append(M)
    return torch.stack(hidden), torch.stack(finals)
