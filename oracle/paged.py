"""The paged cache's definition in 64 bits, sequence by sequence on the host:
what its operators are tested against, with the bounds on their rounding."""
import math

import torch


def rows(pages, table, n):
    """[kv_heads, n, head_dim] of a sequence's slots [0, n), in its own type."""
    ps = pages.shape[2]
    used = table[:-(-n // ps)].long()
    return pages[used].permute(1, 0, 2, 3).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def attend(q, k_pages, v_pages, table, lengths, scale=None):
    """Per sequence (out [heads, D], weights [kv_heads, n] summed over each
    group, lse [heads]) in fp64, and bounds of what fp32 accumulation and one
    rounding to q's type may change: of out, weights and lse.

    A score is a sum of D products: in fp32 off by at most (D + 8) 2^-24 of
    sum |q_i k_i| (the order is free; the 8 cover the scaling); with delta the
    largest such error of a head's scores, a weight is off by a factor within
    2 delta (its own and the denominator's) and the exponentials' and the
    sums' own steps, 2^-20 + n 2^-24.  bf16 multiplies V with P as three terms,
    which is exact, fp16 as two, 2^-22 and, as each is 2^-39 of the largest weight
    at least, 2^-38 |v| a slot."""
    B, heads, D = q.shape
    H = k_pages.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    eps = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[q.dtype]
    results = []
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            zero = torch.zeros(heads, D, dtype=torch.float64)
            results.append(((zero, torch.zeros(H, 0, dtype=torch.float64),
                             torch.full((heads,), -math.inf, dtype=torch.float64)),
                            (zero, torch.zeros(H, 0, dtype=torch.float64), torch.zeros(heads, dtype=torch.float64))))
            continue
        k = rows(k_pages, table[b], n).double().repeat_interleave(heads // H, 0)
        v = rows(v_pages, table[b], n).double().repeat_interleave(heads // H, 0)
        qd = q[b].double()[:, None]
        s = (qd * k).sum(-1) * scale
        delta = ((qd * k).abs().sum(-1).amax(-1) * abs(scale)) * (D + 8) * 2.0 ** -24
        lse = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[:, None])
        out = (p[:, :, None] * v).sum(1)
        rel = 2 * delta + 2.0 ** -20 + n * 2.0 ** -24
        spread = (p[:, :, None] * v.abs()).sum(1)
        split, least = (2.0 ** -22, 2.0 ** -38) if q.dtype == torch.float16 else (0, 0)
        # (a subnormal output is off by half of the type's smallest step)
        floor = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[q.dtype]
        lost = spread * (rel[:, None] + split) + least * (p.amax(-1)[:, None, None] * v.abs()).sum(1)
        out_bound = out.abs() * eps + lost * (1 + eps) + floor
        group = heads // H
        weights = p.view(H, group, n).sum(1)
        weights_bound = (p * rel[:, None]).view(H, group, n).sum(1) + weights * (group + 2) * 2.0 ** -24
        lse_bound = delta + 2.0 ** -20 + n * 2.0 ** -24 + lse.abs() * 2.0 ** -22
        results.append(((out, weights, lse), (out_bound, weights_bound, lse_bound)))
    return results


def evict(scores, positions, n, keep, seen, recent=0, sinks=0):
    """The moves [(source, destination)] that cut one sequence's slots of one
    head: Python lists in, by the definition."""
    m = min(n, keep)

    def rank(t):
        held = positions[t] >= seen - recent or positions[t] < sinks
        nan = not held and scores[t] != scores[t]
        return (not held, not nan, 0.0 if held or nan else -scores[t], t)

    kept = set(sorted(range(n), key=rank)[:m])
    sources = [t for t in range(m, n) if t in kept]
    holes = [t for t in range(m) if t not in kept]
    return list(zip(sources, holes))
