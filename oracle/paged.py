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
    at least, 2^-38 |v| a slot.  A weight below 2^-126 of the largest is below fp32's
    least normal number, and may be 0, and so may its product with V: 2^-126 (1 + |v|) a
    slot, over a sum of 1 at least, and the same again for the sum's share."""
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
        out_bound = out.abs() * eps + lost * (1 + eps) + floor + 2.0 ** -125 * (1 + v.abs()).sum(1)
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


# ------------------------------------------------------------------ whole prompts

def prompt(q, k, v, new, dtype=None, scale=None):
    """Causal attention of one sequence's last `new` slots: q [new, heads, D], its rows
    k, v [kv_heads, n, D] -> (out [new, heads, D], lse [new, heads]) in fp64 and bounds
    of what the device may change of them.

    As for `attend`, and P is rounded once to q's type (half a step, `half`, of
    each weight; fp16 weights below 2^-29 of the largest, and at least 2^-39 of
    it, by 2^-39 more), which fp32 is not.  A row is divided by the sum of what was not
    rounded but for its largest weight (in fp16 that is a power of two): with p_t
    (1 + e_t) in place of p_t the output is off by the sum of p_t e_t v_t, of which the
    largest's is p_k e_k (v_k - out), over 1 + p_k e_k.  k is any slot whose score the
    device may find the largest, and none where scores pass 2^22."""
    m, heads, D = q.shape
    H, n = k.shape[0], k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    dtype = q.dtype if dtype is None else dtype
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    out, bound = (torch.zeros(m, heads, D, dtype=torch.float64) for _ in range(2))
    lse, lse_bound = torch.full((m, heads), -math.inf, dtype=torch.float64), torch.zeros(m, heads, dtype=torch.float64)
    later = torch.arange(n)[None] > (n - m + torch.arange(m))[:, None]
    for g in range(heads):
        kd, vd, qd = k[g * H // heads].double(), v[g * H // heads].double(), q[:, g].double()
        s = (qd @ kd.T * scale).masked_fill(later, -math.inf)
        delta = ((qd.abs() @ kd.abs().T).masked_fill(later, 0).amax(-1) * abs(scale)) * (D + 8) * 2.0 ** -24
        lse[:, g] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[:, g, None])
        p[torch.isinf(lse[:, g])] = 0
        out[:, g] = p @ vd
        rel = 2 * delta + 2.0 ** -20 + n * 2.0 ** -24
        lost = (p @ vd.abs()) * rel[:, None]
        if dtype != torch.float32:
            rounded = p @ vd.abs()
            for i in range(m):
                if p[i].amax() > 0 and s[i].amax().abs() < 2.0 ** 21:
                    best = s[i] >= s[i].amax() - 2 * delta[i]
                    rounded[i] += (p[i, best, None] * ((vd[best] - out[i, g]).abs() - vd[best].abs())).amax(0)
            lost += rounded * half / (1 - half)
        if dtype == torch.float16:
            lost += 2.0 ** -38 * p.amax(-1)[:, None] * ((~later).double() @ vd.abs())
        floor = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[dtype]
        # (below fp32's least normal number: as for `attend`)
        bound[:, g] = out[:, g].abs() * half + lost * (1 + half) + floor + 2.0 ** -125 * (1 + vd.abs()).sum(0)
        lse_bound[:, g] = delta + 2.0 ** -20 + n * 2.0 ** -24 + lse[:, g].abs() * 2.0 ** -22
    return (out, lse), (bound, lse_bound)


# ------------------------------------------------------------------ 4 bits

SIZES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def hold(x):
    """Codes [..., D] (0 .. 15) and scale bytes [..., D / 32] of rows [..., D], by the
    definition: the smallest power of two, in 2^-125 .. 2^125 or for fp16 rows 2^-23 .. 2^13,
    for which no value is above 7 times it; the nearest of the sizes, the even code on ties."""
    y = x.double().unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1)
    special = ~torch.isfinite(amax)
    least, most = (-23, 13) if x.dtype == torch.float16 else (-125, 125)
    e = torch.full(amax.shape, least, dtype=torch.int32)
    for power in range(least, most):
        e[amax > 7 * 2.0 ** power] = power + 1
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
    size = torch.nan_to_num(y.abs() / unit, nan=0.0, posinf=0.0)
    distance = (size[..., None] - torch.tensor(SIZES, dtype=torch.float64)).abs()
    nearest = distance.amin(-1, keepdim=True)
    even = torch.tensor([i % 2 == 0 for i in range(8)])
    tie = ((distance == nearest) & even).any(-1) & ((distance == nearest).sum(-1) > 1)
    code = torch.where(tie, ((distance == nearest) & even).double().argmax(-1), distance.argmin(-1))
    code = code + 8 * torch.signbit(y).long()
    byte = torch.where(special, 255, e + 127)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def pack(codes):
    """Two codes a byte, the even dim's in the lower half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def value(codes, scales):
    """What codes [..., D] (0 .. 15) and scale bytes stand for, in fp64."""
    sizes = torch.tensor(SIZES + tuple(-s for s in SIZES), dtype=torch.float64)[codes.long()]
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127)
    unit[scales == 255] = math.nan
    return (sizes.unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)


def unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


# ------------------------------------------------------------------ rotary positions

def turn(x, positions, frequencies, amplitude=1.0, interleaved=False):
    """Rows x [rows, heads, D] turned by positions [rows] in fp64, and the bound of what
    the device may change: its angle is off by 2^-22 (a fraction of a turn in fp32 and
    the sine's own error), sine, cosine, their products and the sum by 2^-22 of their
    terms, and the result is rounded once to x's type."""
    part = 2 * len(frequencies)
    angle = torch.remainder(positions.double()[:, None] * frequencies[None].double(), 2 * math.pi)[:, None]
    cos, sin = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
    y = x.double().clone()
    spread = torch.zeros_like(y)
    first, second = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    spread[..., first] = spread[..., second] = (a.abs() + b.abs()) * abs(amplitude)
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[x.dtype]
    floor = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[x.dtype]
    bound = y.abs() * half * (spread > 0) + spread * 2.0 ** -21 * (1 + half) + floor * (spread > 0)
    return y, bound
