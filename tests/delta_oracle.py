"""Float64 definitions of the gated delta rule and the group norm.

Each takes tensors of any floating type and returns float64 results on the CPU; gradients come from
autograd through these definitions (or from differences of them)."""

import torch

from selective_oracle import lengths_of, to64  # noqa: F401


def delta_scan(keys, values, queries, strengths, log_decays, memory, lengths, absolute=False):
    """Token by token.  ``absolute``: the sum of the magnitudes of everything that is added up, for inputs whose signs
    are gone (strengths and decays as they are, what is taken out is added)."""
    B, T, H, P = values.shape
    G, N = keys.shape[2:]
    sign = 1.0 if absolute else -1.0
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
            u = strengths[b, t][:, None] * (values[b, t] + sign * (M * k[:, None]).sum(-1))
            M = M + u[..., None] * k[:, None]
            rows.append((M * q[:, None]).sum(-1))
        hidden.append(torch.stack(rows) if rows else 1.0 * values[b])
        finals.append(M)
    return torch.stack(hidden), torch.stack(finals)
