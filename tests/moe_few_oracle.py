"""The routed SwiGLU layer from its definition in 64 bits, with the magnitude that bounds what rounding can lose."""
import math

import torch


def choose(row, top_k):
    """(expert, weight) pairs of one token: list of floats -> the top_k largest, ties to the lower expert, -inf never."""
    if any(math.isnan(v) for v in row):
        return None
    best = sorted((e for e in range(len(row)) if row[e] != -math.inf), key=lambda e: (-row[e], e))[:top_k]
    p = [math.exp(row[e] - row[best[0]]) if row[e] != row[best[0]] else 1.0 for e in best]
    return [(e, v / sum(p)) for e, v in zip(best, p)]


def layer(x, logits, w13, w2, top_k):
    """(out, bound): the layer, and how far bf16 rounding of the intermediate (2^-8 of each of its values, some slack for
    32-bit sums included) and 32-bit arithmetic can carry a result, before its own rounding."""
    xd = x.double()
    out, bound = torch.zeros_like(xd), torch.zeros_like(xd)
    per_expert = {}
    for t, row in enumerate(logits.double().tolist()):
        pairs = choose(row, top_k)
        if pairs is None:
            out[t] = math.nan
            continue
        for e, p in pairs:
            per_expert.setdefault(e, []).append((t, p))
    for e, pairs in per_expert.items():
        rows = torch.tensor([t for t, _ in pairs], device=x.device)
        p = torch.tensor([p for _, p in pairs], dtype=torch.float64, device=x.device)[:, None]
        w = w13[e].double()
        gu = xd[rows] @ w.t()
        mag = xd[rows].abs() @ w.abs().t()
        gate, up, gm, um = gu[:, 0::2], gu[:, 1::2], mag[:, 0::2], mag[:, 1::2]
        mid = torch.nn.functional.silu(gate) * up
        # 32-bit sums of H products: 2^-24 per addition on the longest chain (a lane's H / 256 multiplications of 16 terms, taken as
        # H / 16 + 32), |silu'| <= 1.1; 2^-20 for the exponentials and the division.  A bf16 value has 8 significant bits: rounding
        # to it moves v in [2^n, 2^(n+1)) by at most half of the step 2^(n-7), so by 2^-8 of v
        sums = (x.shape[1] / 16 + 32) * 2.0 ** -24
        err = sums * (1.1 * up.abs() * gm + gate.abs() * um) + mid.abs() * (2.0 ** -20 + 2.0 ** -8 * 1.01)
        v = w2[e].double()
        out.index_add_(0, rows, p * (mid @ v.t()))
        bound.index_add_(0, rows, p * (err @ v.abs().t() + (v.shape[1] * top_k / 16 + 256) * 2.0 ** -24 * (mid.abs() @ v.abs().t())))
    return out, bound
