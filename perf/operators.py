"""The work that the paged cache's operators are measured on: what a program
that decodes from a key-value cache in pages has them do, through
`prismkv_amd.PagedCache`.

* append   new rows of keys and values into the pages of their sequences: one
           token each (a decode step), or prompts, packed without padding;
* attend   one new query token of every sequence over its pages, optionally
           adding each slot's attention weight to its score;
* step     `cache(q, k, v)`: the two as a decode step calls them;
* evict    cut every sequence to a budget: per KV head the slots of the highest
           scores stay, with the newest tokens and the first ones, and the
           kept rows behind the budget move into the places that became free.

A cache holds k and v pages [pages, kv_heads, page_size, head_dim], a page
table [sequences, max_pages], the lengths and, when it is scored, the number
of tokens seen, and each slot's score and original position [sequences,
kv_heads, slots].  Calls write their results into a fork of the cache (its own
lengths, scores and positions over the same pages), as a program does that may
take a step back, so that a pass can be repeated: the rows that append writes
and evict moves are then the same rows again.

The default geometry is this package's: 8 KV heads x 4 query heads, head_dim
128, bf16.  Keys and values are N(0, 1), queries N(0, 2): some slots then
stand out among the weights, as they do in a model.  Scores of a cache to be
cut are log-normal, some exactly zero (slots that no step has weighed yet).
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, batch, longest, mix="even", kv_heads=8, group=4, dim=128, dtype="bf16", page=64, **more):
    return dict(kind=kind, batch=batch, longest=longest, mix=mix, kv_heads=kv_heads, group=group, dim=dim,
                dtype=dtype, page=page, **more)


def listed():
    return [
        # the smallest request: one short prompt; launch and host latency count
        dict(_case("attend", 1, 75, page=16), name="attend_short"),
        # the kernel-check geometry (64K history, 256-row tail), every row read
        dict(_case("attend", 1, 65792), name="attend_64k"),
        # a server's batch of long requests: the largest
        dict(_case("attend", 32, 8192, "near", page=16), name="attend_batch"),
        # other heads and type, ragged (one sequence still empty), pages that end inside any tile
        dict(_case("attend", 7, 5003, "ragged", kv_heads=4, group=6, dim=64, dtype="fp16", page=24),
             name="attend_fp16_d64"),
        # full-precision rows of wide heads
        dict(_case("attend", 4, 4097, "near", kv_heads=2, group=8, dim=256, dtype="fp32", page=32),
             name="attend_fp32_d256"),
        # a long request whose slots are weighed for a later cut
        dict(_case("attend", 1, 32768, scored=True), name="attend_scored_32k"),
        # the decode step of a batch with a bounded cache: write, attend, weigh
        dict(_case("step", 16, 4099, "near", scored=True), name="step_batch"),
        # one token each of a large batch: latency again
        dict(_case("append", 128, 1000, "ragged", tokens=0, scored=True), name="append_tokens"),
        # the prompts of a batch, packed
        dict(_case("append", 4, 500, "ragged", tokens=20011, scored=True), name="append_prompts"),
        # steady state: every 64 steps a full cache goes back to its budget
        dict(_case("evict", 8, 2112, keep=2048, recent=256, sinks=4, scored=True), name="evict_block"),
        # a long prompt cut to a quarter before its first step
        dict(_case("evict", 1, 65536, keep=16384, recent=1024, sinks=4, scored=True), name="evict_prompt"),
        # ragged sequences, some under their budget, other heads and type
        dict(_case("evict", 16, 9001, "ragged", kv_heads=4, group=6, dim=64, dtype="fp16", page=24, keep=1000, recent=33,
                   sinks=0, scored=True, each=True), name="evict_ragged"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "scored", "step", "append", "append", "evict", "evict"])
    dim, dtype = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    page, mix = rng.choice([16, 16, 32, 64, 64, 128, 24, 17]), rng.choice(["even", "near", "ragged"])
    # the rows of all sequences together stay under those of the largest listed case
    row = kv_heads * dim * TYPES[dtype].itemsize * 2
    most = 700_000_000 // row
    batch = _between(rng, 1, 64)
    shape = dict(kv_heads=kv_heads, group=group, dim=dim, dtype=dtype, page=page)
    if kind in ("attend", "scored"):
        longest = _between(rng, 1, max(1, min(65536, most // batch)))
        return _case("attend", batch, longest, mix, **shape, **(dict(scored=True) if kind == "scored" else {}))
    if kind == "step":
        longest = _between(rng, 1, max(1, min(16384, most // batch)))
        return _case("step", batch, longest, mix, **shape, scored=True)
    if kind == "append":
        tokens = rng.choice([0, _between(rng, batch, max(batch, min(30000, most // 8)))])
        return _case("append", batch, _between(rng, 1, 2000), mix, **shape, tokens=tokens, scored=rng.random() < 0.7)
    longest = _between(rng, 40, max(40, min(65536, most // (2 * batch))))
    keep = max(16, int(longest * rng.uniform(0.1, 1.0)))
    return _case("evict", batch, longest, mix, **shape, keep=keep, recent=rng.randint(0, keep // 2),
                 sinks=rng.choice([0, 4]), scored=True, each=rng.random() < 0.3)


# ------------------------------------------------------------------ sizes of a case

def _lengths(case):
    """Tokens of every sequence before the call."""
    batch, longest, mix = case["batch"], case["longest"], case["mix"]
    rng = random.Random(batch * 1000003 + longest)
    if mix == "even":
        return [longest] * batch
    if mix == "near":
        return [longest] + [rng.randint((longest + 1) // 2, longest) for _ in range(batch - 1)]
    out = [longest] + [_between(rng, 1, longest) for _ in range(batch - 1)]
    if batch > 3:
        out[2] = 0
    return out


def _new(case):
    """New rows of every sequence: one each, or a prompt cut at random places."""
    batch, tokens = case["batch"], case.get("tokens", 0)
    if case["kind"] not in ("append", "step"):
        return [0] * batch
    if not tokens:
        return [1] * batch
    rng = random.Random(tokens)
    cuts = sorted(rng.randint(0, tokens) for _ in range(batch - 1))
    return [hi - lo for lo, hi in zip([0] + cuts, cuts + [tokens])]


def _keeps(case):
    """The budget of every sequence."""
    if not case.get("each"):
        return [case["keep"]] * case["batch"]
    rng = random.Random(case["keep"])
    return [rng.randint(max(1, case["keep"] // 2), case["keep"]) for _ in range(case["batch"])]


def work(case):
    es, H, G, D = TYPES[case["dtype"]].itemsize, case["kv_heads"], case["group"], case["dim"]
    lengths, new = _lengths(case), _new(case)
    bytes_, flops = 0, 0
    if case["kind"] in ("append", "step"):
        bytes_ += sum(new) * H * (4 * D * es + (8 if case.get("scored") else 0))
    if case["kind"] in ("attend", "step"):
        rows = sum(lengths) + sum(new)
        bytes_ += rows * H * (2 * D * es + (8 if case.get("scored") else 0)) + 2 * case["batch"] * H * G * D * es
        flops += 4 * rows * H * G * D
    if case["kind"] == "evict":
        for n, keep in zip(lengths, _keeps(case)):
            keep = min(n, keep)
            recent = min(case["recent"], n - keep)  # the newest lie behind the budget
            others = n - recent
            moved = recent + (n - keep - recent) * max(keep - recent, 0) / max(others, 1) if n > keep else 0
            # scores and positions read, those that stay written, the moved rows read and written
            bytes_ += H * (8 * n + 8 * keep + moved * 4 * D * es)
    return {"bytes": int(bytes_), "flops": int(flops)}


# ------------------------------------------------------------------ inputs (plain torch)

def _inputs(case, seed):
    """The cache's tensors and the call's, from the seed alone."""
    dev, dtype = "cuda", TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 1009 + 7)
    B, H, G, D, ps = case["batch"], case["kv_heads"], case["group"], case["dim"], case["page"]
    lengths, new = _lengths(case), _new(case)
    width = max(1, max((n + m + ps - 1) // ps for n, m in zip(lengths, new)))
    own_pages = [(n + m + ps - 1) // ps for n, m in zip(lengths, new)]
    pages = sum(own_pages) + 3
    order = torch.randperm(pages, generator=gen, device=dev).int().cpu()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(own_pages):
        table[b, :count] = order[at:at + count]
        at += count
    x = dict(k=torch.empty(pages, H, ps, D, dtype=dtype, device=dev),
             v=torch.empty(pages, H, ps, D, dtype=dtype, device=dev), table=table.to(dev),
             lengths=torch.tensor(lengths, dtype=torch.int32, device=dev))
    for name in ("k", "v"):
        for lo in range(0, pages, 256):
            part = x[name][lo:lo + 256]
            part.copy_(torch.randn(part.shape, generator=gen, device=dev))
    slots = width * ps
    if case.get("scored"):
        newest = case.get("recent", 0)
        x["scores"] = torch.exp(1.5 * torch.randn(B, H, slots, generator=gen, device=dev) - 2)
        x["scores"][torch.rand(B, H, slots, generator=gen, device=dev) < 0.1] = 0
        # slots hold distinct positions: older tokens in the order that earlier cuts left, the newest last
        x["positions"] = torch.zeros(B, H, slots, dtype=torch.int32, device=dev)
        seen = []
        for b, n in enumerate(lengths):
            tail = min(newest, n)
            total = 2 * n
            seen.append(total)
            if n:
                pick = torch.rand(H, total - tail, generator=gen, device=dev).argsort(dim=1)[:, :n - tail]
                x["positions"][b, :, :n - tail] = pick.int()
                x["positions"][b, :, n - tail:n] = torch.arange(total - tail, total, device=dev, dtype=torch.int32)
        x["seen"] = torch.tensor(seen, dtype=torch.int32, device=dev)
    if case["kind"] in ("attend", "step"):
        x["q"] = (2 * torch.randn(B, H * G, D, generator=gen, device=dev)).to(dtype)
    if case["kind"] in ("append", "step"):
        x["new_k"] = torch.randn(sum(new), H, D, generator=gen, device=dev).to(dtype)
        x["new_v"] = torch.randn(sum(new), H, D, generator=gen, device=dev).to(dtype)
        ends = [0]
        for m in new:
            ends.append(ends[-1] + m)
        x["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    if case["kind"] == "evict":
        x["keep"] = torch.tensor(_keeps(case), dtype=torch.int32, device=dev)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, **x)
    # the fork's own tensors: what a call writes beside the pages
    state["next"] = {name: torch.zeros_like(x[name]) for name in ("lengths", "seen", "scores", "positions") if name in x}
    if own:
        from prismkv_amd import PagedCache
        meta = [{name: t[name] for name in ("seen", "scores", "positions") if name in t} for t in (x, state["next"])]
        state["cache"] = PagedCache.from_tensors(x["k"], x["v"], x["table"], x["lengths"], **meta[0])
        state["fork"] = PagedCache.from_tensors(x["k"], x["v"], x["table"], state["next"]["lengths"], **meta[1])
        if case["kind"] == "evict":
            state["budget"] = x["keep"] if case.get("each") else case["keep"]
    return state


# ------------------------------------------------------------------ the plain form

def _rows(pages, table):
    """[sequences, kv_heads, slots, head_dim] in 32 bits, by the page table."""
    x = pages[table.clamp(min=0).long()]
    B, P, H, ps, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, P * ps, D).float()


def _plain_append(s, into):
    ps = s["k"].shape[2]
    offsets, lengths = s["offsets"].long(), s["lengths"].long()
    rows = torch.arange(s["new_k"].shape[0], device="cuda")
    b = torch.searchsorted(offsets, rows, right=True) - 1
    step = rows - offsets[b]
    slot = lengths[b] + step
    page = s["table"][b, slot // ps].long()
    s["k"][page, :, slot % ps] = s["new_k"]
    s["v"][page, :, slot % ps] = s["new_v"]
    into["lengths"].copy_(lengths + offsets[1:] - offsets[:-1])
    if "seen" in s:
        into["seen"].copy_(s["seen"] + (offsets[1:] - offsets[:-1]))
        for scores in (s["scores"], into["scores"]):
            scores[b, :, slot] = 0.0
        for positions in (s["positions"], into["positions"]):
            positions[b, :, slot] = (s["seen"][b] + step).int()[:, None].expand(-1, positions.shape[1])


def _plain_attend(s, lengths, scores, into):
    q = s["q"].float()
    k, v = _rows(s["k"], s["table"]), _rows(s["v"], s["table"])
    B, H, slots, D = k.shape
    q = q.reshape(B, H, -1, D) * (1.0 / math.sqrt(D))
    valid = (torch.arange(slots, device="cuda")[None] < lengths[:, None])[:, None, None]
    logits = (q @ k.transpose(-1, -2)).masked_fill(~valid, -math.inf)
    peak = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(logits - peak)
    z = p.sum(-1, keepdim=True)
    p = p / torch.where(z > 0, z, 1.0)
    out = (p @ v).reshape(B, -1, D).to(s["q"].dtype)
    if scores is not None:
        weighed = scores + p.sum(2)
        into.copy_(torch.where(valid[:, :, 0], weighed, into))
    return out


def _plain_evict(s, into):
    case = s["case"]
    ps = s["k"].shape[2]
    B, H, slots = s["scores"].shape
    lengths, keep = s["lengths"].long(), s["keep"].long()
    after = torch.minimum(lengths, keep)
    slot = torch.arange(slots, device="cuda").expand(B, H, slots)
    live = slot < lengths[:, None, None]
    held = s["positions"] >= (s["seen"] - case["recent"])[:, None, None]
    held |= s["positions"] < case["sinks"]
    rank = torch.where(live, torch.where(held, math.inf, s["scores"]), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(B, H, slots, dtype=torch.bool, device="cuda")
    stays.scatter_(2, order, slot < after[:, None, None])
    front = slot < after[:, None, None]
    hole, source = front & ~stays, stays & ~front
    into["lengths"].copy_(after)
    into["seen"].copy_(s["seen"])
    for name in ("scores", "positions"):
        into[name].copy_(torch.where(front, s[name], into[name]))
    to, of = hole.nonzero(), source.nonzero()  # the i-th of a row's sources goes to its i-th hole
    b, h, dst, src = to[:, 0], to[:, 1], to[:, 2], of[:, 2]
    for name in ("scores", "positions"):
        into[name][b, h, dst] = s[name][b, h, src]
    for x in (s["k"], s["v"]):
        x[s["table"][b, dst // ps].long(), h, dst % ps] = x[s["table"][b, src // ps].long(), h, src % ps]


def run(state):
    case, into = state["case"], state["next"]
    kind, scored = case["kind"], bool(case.get("scored"))
    out = None
    if own:
        cache, fork = state["cache"], state["fork"]
        if kind == "append":
            cache.append(state["new_k"], state["new_v"], state["offsets"] if case["tokens"] else None, into=fork)
        elif kind == "attend":
            out = cache.attend(state["q"], accumulate=scored, into=fork)
        elif kind == "step":
            out = cache(state["q"], state["new_k"], state["new_v"], accumulate=scored, into=fork)
        else:
            cache.evict(state["budget"], recent=case["recent"], sinks=case["sinks"], into=fork)
    elif kind == "append":
        _plain_append(state, into)
    elif kind == "attend":
        out = _plain_attend(state, state["lengths"], state.get("scores"), into.get("scores"))
    elif kind == "step":
        _plain_append(state, into)
        out = _plain_attend(state, into["lengths"], state["scores"], into["scores"])
    else:
        _plain_evict(state, into)
    result = {} if out is None else {"out": out}
    if kind != "attend":
        result.update(into, k=state["k"], v=state["v"])
    elif scored:
        result["scores"] = into["scores"]
    return result


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    x = _inputs(case, seed)
    H, G, D, ps = case["kv_heads"], case["group"], case["dim"], case["page"]
    lengths, new, kind = _lengths(case), _new(case), case["kind"]
    keys, values = x["k"].double(), x["v"].double()
    after = {name: torch.zeros_like(x[name]).double() for name in ("lengths", "seen", "scores", "positions") if name in x}
    result = {}
    at = 0
    outs = []
    for b, n in enumerate(lengths):
        pages = x["table"][b].tolist()
        if kind in ("append", "step"):
            for i in range(new[b]) if new[b] < 4 else ():
                keys[pages[(n + i) // ps], :, (n + i) % ps] = x["new_k"][at + i].double()
                values[pages[(n + i) // ps], :, (n + i) % ps] = x["new_v"][at + i].double()
            if new[b] >= 4:  # page by page
                for p in range(n // ps, (n + new[b] - 1) // ps + 1):
                    lo, hi = max(n, p * ps), min(n + new[b], (p + 1) * ps)
                    part = slice(at + lo - n, at + hi - n)
                    keys[pages[p], :, lo - p * ps:hi - p * ps] = x["new_k"][part].double().permute(1, 0, 2)
                    values[pages[p], :, lo - p * ps:hi - p * ps] = x["new_v"][part].double().permute(1, 0, 2)
            at += new[b]
            after["lengths"][b] = n + new[b]
            if "seen" in x:
                first = int(x["seen"][b])
                after["seen"][b] = first + new[b]
                after["positions"][b, :, n:n + new[b]] = torch.arange(first, first + new[b], device="cuda").double()
                x["scores"][b, :, n:n + new[b]] = 0
            n += new[b]
        if kind in ("attend", "step"):
            if n == 0:
                outs.append(torch.zeros(H * G, D, dtype=torch.float64, device="cuda"))
                continue
            used = pages[:(n + ps - 1) // ps]
            heads = []
            for h in range(H):
                kb = keys[used, h].reshape(-1, D)[:n]
                vb = values[used, h].reshape(-1, D)[:n]
                p = torch.softmax((kb @ x["q"][b, h * G:(h + 1) * G].double().T.contiguous()) / math.sqrt(D), dim=0)
                heads.append(p.T.contiguous() @ vb)
                if case.get("scored"):
                    after["scores"][b, h, :n] = x["scores"][b, h, :n].double() + p.sum(1)
            outs.append(torch.cat(heads))
        if kind == "evict":
            m = min(n, _keeps(case)[b])
            after["lengths"][b], after["seen"][b] = m, x["seen"][b]
            for h in range(H):
                score, position = x["scores"][b, h, :n].tolist(), x["positions"][b, h, :n].tolist()
                edge = int(x["seen"][b]) - case["recent"]
                ranked = sorted(range(n), key=lambda t: (not (position[t] >= edge or position[t] < case["sinks"]),
                                                         0.0 if position[t] >= edge or position[t] < case["sinks"]
                                                         else -score[t], t))
                kept = set(ranked[:m])
                src = torch.tensor([t for t in range(m, n) if t in kept], dtype=torch.long, device="cuda")
                dst = torch.tensor([t for t in range(m) if t not in kept], dtype=torch.long, device="cuda")
                slot = torch.arange(m, device="cuda")
                slot[dst] = src
                after["scores"][b, h, :m] = x["scores"][b, h, slot].double()
                after["positions"][b, h, :m] = x["positions"][b, h, slot].double()
                row = x["table"][b].long()
                for rows in (keys, values):
                    rows[row[dst // ps], h, dst % ps] = rows[row[src // ps], h, src % ps].clone()
    if outs:
        result["out"] = torch.stack(outs)
    if kind != "attend":
        result.update(after, k=keys, v=values)
    elif case.get("scored"):
        result["scores"] = after["scores"]
    return result
