"""Caches in pages of any type and storage, for the tests of what serves them."""
import math

import torch

from oracle import paged
from prismkv_amd import PagedCache

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(lengths, kv_heads=2, dim=128, page=16, dtype=BF16, storage=None, room=0, scored=False, seed=0, spare=2, fill=math.nan,
         device="cuda", edit=None):
    """A cache over shuffled pages whose slots behind the lengths (and spare pages) hold
    `fill`, and host copies of its tensors; k and v are there as the values that the
    pages hold.  `edit(k, v, table)` changes the rows before they are held."""
    gen = torch.Generator().manual_seed(seed)
    room = room if isinstance(room, (list, tuple)) else [room] * len(lengths)
    own = [-(-(n + r) // page) for n, r in zip(lengths, room)]
    width, pages = max(1, max(own)), sum(own) + spare
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=gen).to(dtype) for _ in range(2))
    live = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, (n, count) in enumerate(zip(lengths, own)):
        table[b, :count] = order[at:at + count]
        at += count
        for p in range(count):
            live[table[b, p], :max(0, min(page, n - p * page))] = True
    if edit is not None:
        edit(k, v, table)
    for x in (k, v):
        x.permute(0, 2, 1, 3)[~live] = fill
    host = dict(k=k, v=v, table=table, lengths=torch.tensor(lengths, dtype=torch.int32))
    given = {}
    if scored:
        slots = width * page
        host["scores"] = torch.rand(len(lengths), kv_heads, slots, generator=gen)
        host["positions"] = torch.stack([torch.stack([torch.randperm(slots, generator=gen) for _ in range(kv_heads)])
                                         for _ in lengths]).int()
        host["seen"] = torch.full((len(lengths),), slots, dtype=torch.int32)
        given.update({name: host[name].to(device) for name in ("seen", "scores", "positions")})
    if storage:
        pages_of = {}
        for name in ("k", "v"):
            codes, scales = paged.hold(host[name])
            host[name] = paged.value(codes, scales)
            pages_of[name] = paged.pack(codes).to(device)
            given[name + "_scales"] = scales.to(device)
        given["dtype"] = dtype
        cache = PagedCache.from_tensors(pages_of["k"], pages_of["v"], table.to(device), host["lengths"].to(device), **given)
    else:
        cache = PagedCache.from_tensors(k.to(device), v.to(device), table.to(device), host["lengths"].to(device), **given)
    return cache, host


def ends(new):
    total = [0]
    for m in new:
        total.append(total[-1] + m)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def rows_like(cache, count, heads, seed=1, sigma=1.5):
    gen = torch.Generator().manual_seed(seed)
    return (sigma * torch.randn(count, heads, cache._shape[2], generator=gen)).to(cache.dtype)


def check_prompt(q, host, lengths, new, out, lse=None, scale=None, skip=()):
    """Every sequence's rows against the definition, over the slots `lengths`."""
    at = 0
    out, lse = out.cpu(), None if lse is None else lse.cpu()
    for b, (n, m) in enumerate(zip(lengths, new)):
        part = slice(at, at + m)
        at += m
        if m == 0 or b in skip:
            continue
        k, v = (paged.rows(host[name], host["table"][b], n) for name in ("k", "v"))
        (want, l), (bound, l_bound) = paged.prompt(q[part], k, v, m, scale=scale)
        err = (out[part].double() - want).abs()
        assert (err <= bound).all(), (b, float((err / bound.clamp_min(1e-300)).max()))
        if lse is not None:
            same = torch.isinf(l) & (lse[part].double() == l)
            assert (((lse[part].double() - l).abs() <= l_bound) | same).all(), b
