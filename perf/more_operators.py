"""The work that the paged cache's operators of a whole serving path are
measured on, through `prismkv_amd.PagedCache`: what a program has them do
beside the single-token attention over 16-bit pages.

* prompt       `attend_prompt`: causal attention of many new rows of every
               sequence, packed, over all that its pages hold, the new rows
               last (they were appended before); a prompt, a chunk of one, a
               turn behind a long history, single tokens among them;
* rotate       `append` with a `Rotary`: queries and keys turned by the
               positions that the cache knows, the keys and values into their
               pages;
* four_append  `append` to a cache in 4 bits and `read` of the appended rows as
               the values that its codes stand for;
* four_attend  `attend`: one new token of every sequence over a cache in 4 bits;
* four_prompt  `attend_prompt` over a cache in 4 bits.

Pages are [pages, kv_heads, page_size, head_dim].  In 4 bits a row holds, for
every 32 dims, a power of two 2^e (a byte, e + 127) and the dims as multiples of
it, 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign (codes 0 to 7, +8 if negative; the
even dim in the low half of a byte): e is the smallest with amax <= 7 2^e, at
least -125, and the code the nearest one, ties to even, at most 6.

The default geometry is this package's: 8 KV heads x 4 query heads, head_dim
128, bf16.  Keys and values are N(0, 1), queries N(0, 2): some slots then stand
out among the weights, as they do in a model.  Calls that append write their
lengths into a fork of the cache, so that a pass can be repeated.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, batch, longest, mix="even", tokens=0, kv_heads=8, group=4, dim=128, dtype="bf16", page=64, **more):
    return dict(kind=kind, batch=batch, longest=longest, mix=mix, tokens=tokens, kv_heads=kv_heads, group=group, dim=dim,
                dtype=dtype, page=page, **more)


def _rotary(layout="half", part=128, base=1e6, scaling="none"):
    return dict(layout=layout, part=part, base=base, scaling=scaling)


def listed():
    return [
        # the smallest request: one short prompt; launch and host latency count
        dict(_case("prompt", 1, 0, tokens=75, page=16), name="prompt_short"),
        # a long document, the whole prompt at once: the largest
        dict(_case("prompt", 1, 0, tokens=16384), name="prompt_long"),
        # the next turn of a long conversation: few rows over many slots
        dict(_case("prompt", 1, 65000, tokens=48), name="prompt_turn"),
        # a server's batch: prompts and chunks, ragged, other heads and type, pages that end inside any tile
        dict(_case("prompt", 9, 3001, "ragged", tokens=9007, kv_heads=4, group=6, dim=64, dtype="fp16", page=24),
             name="prompt_ragged_fp16"),
        # full precision of wide heads
        dict(_case("prompt", 3, 700, "near", tokens=4097, kv_heads=2, group=8, dim=256, dtype="fp32", page=32),
             name="prompt_fp32"),
        # the decode step of a large batch: latency
        dict(_case("rotate", 128, 1000, "ragged", **_rotary()), name="rotate_step"),
        # chunks of prompts far behind what a bounded cache still holds; part of the head, pairs side by side
        dict(_case("rotate", 4, 500, "ragged", tokens=20011, dim=64, dtype="fp16", scored=True,
                   **_rotary("interleaved", 32, 5e5, "llama3")), name="rotate_prompts_fp16"),
        # one token each of a large batch into 4 bits: latency again
        dict(_case("four_append", 128, 1000, "ragged"), name="four_append_tokens"),
        # prompts into 4 bits
        dict(_case("four_append", 4, 500, "ragged", tokens=20011), name="four_append_prompts"),
        # the kernel-check geometry (64K history, 256-row tail), every row read, in 4 bits
        dict(_case("four_attend", 1, 65792), name="four_attend_64k"),
        # a server's batch of long requests in 4 bits
        dict(_case("four_attend", 32, 8192, "near", dtype="fp16", page=16), name="four_attend_batch_fp16"),
        # chunks of prompts over histories in 4 bits
        dict(_case("four_prompt", 5, 9001, "near", tokens=6007), name="four_prompt_chunks"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "rotate", "rotate", "four_append", "four_attend", "four_attend",
                       "four_prompt"])
    dim, dtype = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("four"):
        dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    page, mix = rng.choice([16, 16, 32, 64, 64, 128, 24, 17]), rng.choice(["even", "near", "ragged"])
    row = kv_heads * dim * TYPES[dtype].itemsize * 2
    most = 700_000_000 // row  # rows of all sequences together
    batch = _between(rng, 1, 64)
    shape = dict(kv_heads=kv_heads, group=group, dim=dim, dtype=dtype, page=page)
    if kind == "four_attend":
        longest = _between(rng, 1, max(1, min(65536, most // batch)))
        return _case(kind, batch, longest, mix, **shape)
    if kind in ("rotate", "four_append"):
        tokens = rng.choice([0, _between(rng, batch, max(batch, min(30000, most // (8 + 4 * group))))])
        more = {}
        if kind == "rotate":
            part = rng.choice([16, 32, dim // 2, dim, dim])
            more = dict(scored=rng.random() < 0.5, **_rotary(rng.choice(["half", "half", "interleaved"]), part,
                                                             rng.choice([1e4, 5e5, 1e6]),
                                                             rng.choice(["none", "linear", "llama3", "yarn"])))
        return _case(kind, batch, _between(rng, 1, 2000), mix, tokens, **shape, **more)
    # pairs of a row and a slot stay well under those of the largest listed case
    tokens = _between(rng, 1, 16384)
    batch = min(batch, tokens)
    longest = rng.choice([0, _between(rng, 1, 65536)])
    pairs = 2_000_000_000 * 128 // (max(dim, 128) * kv_heads * group * (2 if dtype == "fp32" else 1))
    longest = max(0, min(longest, pairs // tokens, most // batch - tokens))
    tokens = max(batch, min(tokens, int(math.sqrt(pairs)), most // (1 + group)))
    return _case(kind, batch, longest, mix if longest else "even", tokens, **shape)


# ------------------------------------------------------------------ sizes of a case

def _lengths(case):
    """Slots that every sequence holds before the call's new rows."""
    batch, longest, mix = case["batch"], case["longest"], case["mix"]
    rng = random.Random(batch * 1000003 + longest)
    if mix == "even" or longest < 1:
        return [longest] * batch
    if mix == "near":
        return [longest] + [rng.randint((longest + 1) // 2, longest) for _ in range(batch - 1)]
    out = [longest] + [_between(rng, 1, longest) for _ in range(batch - 1)]
    if batch > 3:
        out[2] = 0
    return out


def _new(case):
    """New rows of every sequence: one each, or `tokens` cut at random places."""
    batch, tokens = case["batch"], case["tokens"]
    if case["kind"] == "four_attend":
        return [0] * batch
    if not tokens:
        return [1] * batch
    rng = random.Random(tokens)
    cuts = sorted(rng.randint(0, tokens) for _ in range(batch - 1))
    return [hi - lo for lo, hi in zip([0] + cuts, cuts + [tokens])]


def _four(case):
    return case["kind"].startswith("four")


def work(case):
    es, H, G, D = TYPES[case["dtype"]].itemsize, case["kv_heads"], case["group"], case["dim"]
    lengths, new, kind = _lengths(case), _new(case), case["kind"]
    held = D // 2 + D // 32 if _four(case) else D * es  # bytes of a row in the pages
    bytes_, flops = 0, 0
    if kind == "rotate":
        bytes_ = sum(new) * D * es * (2 * H * G + 4 * H) + (sum(new) * H * 16 if case.get("scored") else 0)
        flops = sum(new) * 3 * case["part"] * (H * G + H)
    elif kind == "four_append":
        bytes_ = sum(new) * H * 2 * (2 * D * es + 2 * held)  # rows in and out, their codes written and read
    elif kind == "four_attend":
        bytes_ = sum(lengths) * H * 2 * held + case["batch"] * H * G * (2 * D * es + 4)
        flops = 4 * sum(lengths) * H * G * D
    else:
        for n, m in zip(lengths, new):
            bytes_ += (n + m) * H * 2 * held * (m > 0) + m * H * G * (2 * D * es + 4)
            flops += 4 * H * G * D * (m * n + m * (m + 1) // 2)
    return {"bytes": int(bytes_), "flops": int(flops)}


# ------------------------------------------------------------------ 4 bits, plainly

def _quantise(x):
    """Codes [..., D / 2] and scale bytes [..., D / 32] of rows [..., D]."""
    y = x.float().unflatten(-1, (-1, 32))
    part, power = torch.frexp(y.abs().amax(-1))  # part in [0.5, 1): above 0.875 the next power of two
    e = (power - 3 + (part > 0.875).int()).clamp(min=-125, max=125)
    y = torch.ldexp(y, -e[..., None])
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)
    code = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = (code + 8 * (y < 0).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _widen(codes, scales):
    """The rows [..., D] that codes and scale bytes stand for, in 32 bits."""
    sizes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    x = torch.stack((sizes[(codes & 15).int()], sizes[(codes >> 4).int()]), -1).flatten(-2)
    return torch.ldexp(x.unflatten(-1, (-1, 32)), (scales.int() - 127)[..., None]).flatten(-2)


# ------------------------------------------------------------------ inputs (plain torch)

def _inputs(case, seed):
    """The cache's tensors and the call's, from the seed alone."""
    dev, dtype = "cuda", TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 1009 + 7)
    B, H, G, D, ps, kind = case["batch"], case["kv_heads"], case["group"], case["dim"], case["page"], case["kind"]
    lengths, new = _lengths(case), _new(case)
    own_pages = [(n + m + ps - 1) // ps for n, m in zip(lengths, new)]
    width, pages = max(1, max(own_pages)), sum(own_pages) + 3
    order = torch.randperm(pages, generator=gen, device=dev).int().cpu()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(own_pages):
        table[b, :count] = order[at:at + count]
        at += count
    x = dict(table=table.to(dev))
    shape = (pages, H, ps)
    for name in ("k", "v"):
        if _four(case):
            x[name] = torch.empty(*shape, D // 2, dtype=torch.uint8, device=dev)
            x[name + "_scales"] = torch.empty(*shape, D // 32, dtype=torch.uint8, device=dev)
        else:
            x[name] = torch.empty(*shape, D, dtype=dtype, device=dev)
        for lo in range(0, pages, 256):
            part = torch.randn((min(256, pages - lo),) + shape[1:] + (D,), generator=gen, device=dev)
            if _four(case):
                x[name][lo:lo + 256], x[name + "_scales"][lo:lo + 256] = _quantise(part)
            else:
                x[name][lo:lo + 256] = part
    appended = kind in ("rotate", "four_append")  # the rows that the others appended are in their lengths
    x["lengths"] = torch.tensor([n + (0 if appended else m) for n, m in zip(lengths, new)], dtype=torch.int32, device=dev)
    if case.get("scored"):  # positions go on from the tokens seen, most of which were cut away
        rng = random.Random(sum(lengths))
        x["seen"] = torch.tensor([n + rng.randint(0, 900_000) for n in lengths], dtype=torch.int32, device=dev)
        x["scores"] = torch.rand(B, H, width * ps, generator=gen, device=dev)
        x["positions"] = torch.arange(width * ps, device=dev, dtype=torch.int32).expand(B, H, -1).contiguous()
    rows = B if kind == "four_attend" else sum(new)
    if appended:  # parts of one projection's rows
        x["rows"] = torch.randn(rows, H * G + 2 * H, D, generator=gen, device=dev).to(dtype)
        if kind == "rotate":
            x["q"] = x["rows"][:, :H * G]
        x["new_k"], x["new_v"] = x["rows"][:, H * G:H * G + H], x["rows"][:, H * G + H:]
    else:
        x["q"] = (2 * torch.randn(rows, H * G, D, generator=gen, device=dev)).to(dtype)
    ends = [0]
    for m in new:
        ends.append(ends[-1] + m)
    x["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    return x


SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, **x)
    # the fork's own tensors: what an append writes beside the pages
    state["next"] = {name: x[name].clone() for name in ("lengths", "seen", "scores", "positions") if name in x}
    if case["kind"] in ("prompt", "four_prompt", "four_attend"):
        state["lse"] = torch.empty(x["q"].shape[:2], dtype=torch.float32, device="cuda")
    if own:
        from prismkv_amd import PagedCache, Rotary
        four = dict(k_scales=x["k_scales"], v_scales=x["v_scales"], dtype=TYPES[case["dtype"]]) if _four(case) else {}
        for name, t in (("cache", x), ("fork", state["next"])):
            meta = {key: t[key] for key in ("seen", "scores", "positions") if key in t}
            state[name] = PagedCache.from_tensors(x["k"], x["v"], x["table"], t["lengths"], **four, **meta)
        if case["kind"] == "rotate":
            state["rotary"] = Rotary(case["dim"], base=case["base"], rotary_dim=case["part"],
                                     interleaved=case["layout"] == "interleaved", scaling=SCALINGS[case["scaling"]])
    elif case["kind"] == "rotate":
        state["frequencies"], state["amplitude"] = _frequencies(case)
    return state


# ------------------------------------------------------------------ the plain form

def _frequencies(case):
    """The angle of every pair of dims at position 1 (64 bits), and the factor of
    the turned dims."""
    part, base = case["part"], case["base"]
    freq = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device="cuda") / part)
    s = SCALINGS[case["scaling"]]
    if s is None:
        return freq, 1.0
    if s["rope_type"] == "linear":
        return freq / s["factor"], 1.0
    original = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        turns = original * freq / (2 * math.pi)  # within the original context
        mix = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0, 1)
        return freq * (mix + (1 - mix) / s["factor"]), 1.0

    def pair_of(turns):  # the pair that makes so many turns
        return part * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), part - 1)
    ramp = ((torch.arange(part // 2, dtype=torch.float64, device="cuda") - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq * (1 - ramp + ramp / s["factor"]), 0.1 * math.log(s["factor"]) + 1


def _turn(x, position, state):
    """Rows [rows, heads, D] turned by their positions, in 32 bits."""
    case = state["case"]
    angle = position.double()[:, None, None] * state["frequencies"]
    cos, sin = ((f(angle) * state["amplitude"]).float() for f in (torch.cos, torch.sin))
    x, part = x.float(), case["part"]
    if case["layout"] == "half":
        a, b = x[..., :part // 2], x[..., part // 2:part]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:part:2], x[..., 1:part:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., part:]), -1)


def _held(s, name, b=None):
    """[.., kv_heads, slots, head_dim] in 32 bits of one sequence or all, by the page table."""
    pages = (s["table"] if b is None else s["table"][b:b + 1]).clamp(min=0).long()
    x = _widen(s[name][pages], s[name + "_scales"][pages]) if name + "_scales" in s else s[name][pages].float()
    B, P, H, ps, D = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(B, H, P * ps, D)
    return x if b is None else x[0]


def _softmax_product(logits, v):
    """Attention from its masked scores: the products and the sums' logarithm."""
    peak = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(logits - peak)
    z = p.sum(-1, keepdim=True)
    return (p / torch.where(z > 0, z, 1.0)) @ v, (peak + torch.log(z))[..., 0]


def _plain_attend(s):
    """One query token of every sequence over all its slots."""
    k, v = _held(s, "k"), _held(s, "v")
    B, H, slots, D = k.shape
    q = s["q"].float().reshape(B, H, -1, D) * (1.0 / math.sqrt(D))
    valid = (torch.arange(slots, device="cuda")[None] < s["lengths"][:, None])[:, None, None]
    out, lse = _softmax_product((q @ k.transpose(-1, -2)).masked_fill(~valid, -math.inf), v)
    return out.reshape(B, -1, D).to(s["q"].dtype), lse.reshape(B, -1)


def _plain_prompt(s):
    """Sequence by sequence, so many rows at a time that their scores fit."""
    case, q = s["case"], s["q"]
    H, G, D = case["kv_heads"], case["group"], case["dim"]
    out, lse = torch.empty_like(q), torch.empty_like(s["lse"])
    row = 0
    for b, (n, m) in enumerate(zip(_lengths(case), _new(case))):
        if m == 0:
            continue
        k, v = _held(s, "k", b), _held(s, "v", b)
        most = max(1, (1 << 28) // ((n + m) * H * G))
        for lo in range(0, m, most):
            hi = min(m, lo + most)
            x = q[row + lo:row + hi].float().reshape(hi - lo, H, G, D).permute(1, 0, 2, 3).reshape(H, -1, D)
            scores = (x * (1.0 / math.sqrt(D))) @ k[:, :n + hi].transpose(-1, -2)
            last = n + torch.arange(lo, hi, device="cuda").repeat_interleave(G)
            later = torch.arange(n + hi, device="cuda")[None] > last[:, None]
            y, l = _softmax_product(scores.masked_fill_(later, -math.inf), v[:, :n + hi])
            out[row + lo:row + hi] = y.reshape(H, -1, G, D).permute(1, 0, 2, 3).reshape(hi - lo, H * G, D).to(q.dtype)
            lse[row + lo:row + hi] = l.reshape(H, -1, G).permute(1, 0, 2).reshape(hi - lo, H * G)
        row += m
    return out, lse


def _plain_append(s, k, into):
    """Writes the rows into their pages; returns their places."""
    ps = s["k"].shape[2]
    offsets, lengths = s["offsets"].long(), s["lengths"].long()
    rows = torch.arange(k.shape[0], device="cuda")
    b = torch.searchsorted(offsets, rows, right=True) - 1
    step = rows - offsets[b]
    slot = lengths[b] + step
    page = s["table"][b, slot // ps].long()
    for name, x in (("k", k), ("v", s["new_v"])):
        if name + "_scales" in s:
            s[name][page, :, slot % ps], s[name + "_scales"][page, :, slot % ps] = _quantise(x)
        else:
            s[name][page, :, slot % ps] = x.to(s[name].dtype)
    into["lengths"].copy_(lengths + offsets[1:] - offsets[:-1])
    if "seen" in s:
        into["seen"].copy_(s["seen"] + (offsets[1:] - offsets[:-1]))
        for scores in (s["scores"], into["scores"]):
            scores[b, :, slot] = 0.0
        for positions in (s["positions"], into["positions"]):
            positions[b, :, slot] = (s["seen"][b] + step).int()[:, None].expand(-1, positions.shape[1])
    return page, slot % ps


def run(state):
    case, into = state["case"], state["next"]
    kind = case["kind"]
    packed = state["offsets"] if case["tokens"] else None
    if kind in ("prompt", "four_prompt"):
        if own:
            return {"out": state["cache"].attend_prompt(state["q"], packed, lse=state["lse"]), "lse": state["lse"]}
        return dict(zip(("out", "lse"), _plain_prompt(state)))
    if kind == "four_attend":
        if own:
            return {"out": state["cache"].attend(state["q"], lse=state["lse"]), "lse": state["lse"]}
        return dict(zip(("out", "lse"), _plain_attend(state)))
    if kind == "rotate":
        if own:
            q = state["cache"].append(state["new_k"], state["new_v"], packed, q=state["q"], rotary=state["rotary"],
                                      into=state["fork"])
        else:
            offsets = state["offsets"].long()
            rows = torch.arange(state["q"].shape[0], device="cuda")
            b = torch.searchsorted(offsets, rows, right=True) - 1
            position = (state["seen"] if "seen" in state else state["lengths"])[b] + rows - offsets[b]
            q = _turn(state["q"], position, state).to(state["q"].dtype)
            _plain_append(state, _turn(state["new_k"], position, state), into)
        return {"q": q, "k": state["k"], "v": state["v"], **into}
    if own:
        state["cache"].append(state["new_k"], state["new_v"], packed, into=state["fork"])
        k, v = state["fork"].read(packed, rows=state["new_k"].shape[0])
    else:
        place = _plain_append(state, state["new_k"], into)
        k, v = (_widen(state[name][place[0], :, place[1]], state[name + "_scales"][place[0], :, place[1]])
                .to(state["new_k"].dtype) for name in ("k", "v"))
    return {"k": k, "v": v, **into}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_values(x):
    """The values that rows stand for in 4 bits, from the borders between the sizes."""
    y = x.double().unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 7)).clamp(min=-125, max=125)
    unit = torch.pow(torch.full_like(e, 2.0), e)
    # (the logarithm's rounding beside a power of two: the definition decides)
    unit = torch.where(amax > 7 * unit, 2 * unit, unit)
    unit = torch.where((amax <= 3.5 * unit) & (e > -125), unit / 2, unit)
    size = y.abs() / unit
    got = torch.zeros_like(size)
    # a border's own value goes to the even of its two codes
    for border, below, above, up in ((0.25, 0, 0.5, False), (0.75, 0.5, 1, True), (1.25, 1, 1.5, False),
                                     (1.75, 1.5, 2, True), (2.5, 2, 3, False), (3.5, 3, 4, True), (5, 4, 6, False)):
        got = torch.where((size >= border) if up else (size > border), above, got)
    return (torch.sign(y) * got * unit).flatten(-2)


def _exact_frequency(case, j):
    """Angle per position of pair j, and the factor of the turned dims."""
    d, base, s = case["part"], case["base"], SCALINGS[case["scaling"]]
    f = math.exp(-2 * j / d * math.log(base))
    if s is None:
        return f, 1.0
    factor = s["factor"]
    if s["rope_type"] == "linear":
        return f / factor, 1.0
    length = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        wave = 2 * math.pi / f
        lo, hi = s["low_freq_factor"], s["high_freq_factor"]
        if wave < length / hi:
            return f, 1.0
        if wave > length / lo:
            return f / factor, 1.0
        smooth = (length / wave - lo) / (hi - lo)
        return (1 - smooth) * f / factor + smooth * f, 1.0
    first = max(math.floor(d * math.log(length / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    last = min(math.ceil(d * math.log(length / (2 * math.pi)) / (2 * math.log(base))), d - 1)
    t = min(max((j - first) / max(last - first, 0.001), 0.0), 1.0)
    return f / factor * t + f * (1 - t), 1 + 0.1 * math.log(factor)


def _exact_turn(x, position, case):
    y = x.double().clone()
    half = case["part"] // 2
    for j in range(half):
        f, factor = _exact_frequency(case, j)
        a, b = (j, j + half) if case["layout"] == "half" else (2 * j, 2 * j + 1)
        c, s = (g(position.double() * f)[:, None] * factor for g in (torch.cos, torch.sin))
        y[..., a] = x[..., a].double() * c - x[..., b].double() * s
        y[..., b] = x[..., b].double() * c + x[..., a].double() * s
    return y


def exact(case, seed):
    x = _inputs(case, seed)
    H, G, D, ps, kind = case["kv_heads"], case["group"], case["dim"], case["page"], case["kind"]
    lengths, new = _lengths(case), _new(case)
    if kind == "four_append":
        after = x["lengths"].double() + torch.tensor(new, device="cuda").double()
        return {"k": _exact_values(x["new_k"]), "v": _exact_values(x["new_v"]), "lengths": after}
    if kind == "rotate":
        keys, values = x["k"].double(), x["v"].double()
        after = {name: x[name].double().clone() for name in ("lengths", "seen", "scores", "positions") if name in x}
        first = x["seen"] if "seen" in x else x["lengths"]
        position = torch.cat([int(first[b]) + torch.arange(m) for b, m in enumerate(new)]).cuda()
        turned = _exact_turn(x["new_k"], position, case)
        at = 0
        for b, (n, m) in enumerate(zip(lengths, new)):
            if m == 0:
                continue
            row = x["table"][b].long()
            slot = torch.arange(n, n + m, device="cuda")
            keys[row[slot // ps], :, slot % ps] = turned[at:at + m]
            values[row[slot // ps], :, slot % ps] = x["new_v"][at:at + m].double()
            after["lengths"][b] += m
            if "seen" in x:
                after["seen"][b] += m
                after["scores"][b, :, n:n + m] = 0
                after["positions"][b, :, n:n + m] = position[at:at + m].double()
            at += m
        return {"q": _exact_turn(x["q"], position, case), "k": keys, "v": values, **after}
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(x["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    rows = [1] * case["batch"] if kind == "four_attend" else new
    at = 0
    for b, m in enumerate(rows):
        total = int(x["lengths"][b])
        if m and total:
            used = x["table"][b, :(total + ps - 1) // ps].long()
            for h in range(H):
                if _four(case):
                    kb, vb = (_widen(x[name][used, h], x[name + "_scales"][used, h]).double() for name in ("k", "v"))
                else:
                    kb, vb = x["k"][used, h].double(), x["v"][used, h].double()
                kb, vb = kb.reshape(-1, D)[:total], vb.reshape(-1, D)[:total]
                kt = kb.T.contiguous()
                for g in range(h * G, (h + 1) * G):
                    for lo in range(0, m, 4096):
                        hi = min(m, lo + 4096)
                        seen = total - m + hi
                        s = (x["q"][at + lo:at + hi, g].double() @ kt[:, :seen]) / math.sqrt(D)
                        s += torch.full_like(s, -math.inf).triu_(seen - (hi - lo) + 1)
                        lse[at + lo:at + hi, g] = torch.logsumexp(s, -1)
                        out[at + lo:at + hi, g] = torch.softmax(s, -1) @ vb[:seen]
        at += m
    return {"out": out, "lse": lse}
