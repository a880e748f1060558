"""Float64 definitions of the gated delta rule and the group norm.

Each takes tensors of any floating type and returns float64 results on the CPU; gradients come from
autograd through these definitions (or from differences of them)."""

import torch

from selective_oracle import lengths_of, to64  # noqa: F401

NAMES = ("keys", "values", "queries", "strengths", "log_decays", "memory")


def delta_scan(keys, values, queries, strengths, log_decays, memory, lengths):
    """Token by token."""
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
            k, q = (v[b, t].repeat_interleave(H // G, 0) for v in (keys, queries))
            if log_decays is not None:
                M = torch.exp(log_decays[b, t])[:, None, None] * M
            u = strengths[b, t][:, None] * (values[b, t] - (M * k[:, None]).sum(-1))
            M = M + u[..., None] * k[:, None]
            rows.append((M * q[:, None]).sum(-1))
        hidden.append(torch.stack(rows) if rows else 1.0 * values[b])
        finals.append(M)
    return torch.stack(hidden), torch.stack(finals)


def group_norm(x, groups, weight, bias, gate, silu, center, eps=1e-5):
    """Group by group of the rows [rows, channels]."""
    C = x.size(-1)
    W = C // groups
    outs = []
    for i in range(groups):
        part = slice(i * W, (i + 1) * W)
        v = x[:, part]
        if center:
            v = v - v.sum(1, keepdim=True) / W
        y = v / torch.sqrt((v * v).sum(1, keepdim=True) / W + eps)
        y = y if weight is None else y * weight[part]
        y = y if bias is None else y + bias[part]
        z = y if gate is None else gate[:, part]
        act = z / (1 + torch.exp(-z)) if silu else z
        outs.append(act if gate is None else y * act)
    return torch.cat(outs, 1)
