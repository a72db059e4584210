"""The paged cache on the device against its 64-bit definition
(oracle/paged.py): append and evict exactly, attend within bounds derived
there."""
import math

import pytest
import torch

from oracle import paged
from prismkv_amd import PagedCache
from tests.gpu_util import log

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(lengths, kv_heads=2, dim=128, page=16, dtype=BF16, room=0, scored=False, seed=0, spare=2, fill=math.nan):
    """A cache over shuffled pages whose slots behind the lengths (and spare
    pages) hold `fill`, and host copies of its tensors."""
    gen = torch.Generator().manual_seed(seed)
    own = [-(-(n + room) // page) for n in lengths]
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
    for x in (k, v):
        x.permute(0, 2, 1, 3)[~live] = fill
    host = dict(k=k, v=v, table=table, lengths=torch.tensor(lengths, dtype=torch.int32))
    if scored:
        slots = width * page
        host["scores"] = torch.rand(len(lengths), kv_heads, slots, generator=gen)
        host["positions"] = torch.stack([torch.stack([torch.randperm(slots, generator=gen) for _ in range(kv_heads)])
                                         for _ in lengths]).int()
        host["seen"] = torch.full((len(lengths),), slots, dtype=torch.int32)
    dev = {name: x.cuda() for name, x in host.items()}
    cache = PagedCache.from_tensors(dev["k"], dev["v"], dev["table"], dev["lengths"],
                                    **{n: dev[n] for n in ("seen", "scores", "positions") if n in dev})
    return cache, host


def queries(cache, group, seed=1, sigma=1.5):
    gen = torch.Generator().manual_seed(seed)
    sequences, kv_heads, dim = cache.table.shape[0], cache.k.shape[1], cache.k.shape[3]
    return (sigma * torch.randn(sequences, kv_heads * group, dim, generator=gen)).to(cache.k.dtype)


def bits(x):
    """A tensor to be compared bit for bit (NaN equal to itself)."""
    return x.contiguous().view({2: torch.int16, 4: torch.int32}[x.element_size()]).cpu()


def check_attend(q, host, lengths, out, weights=None, lse=None, scale=None):
    out = out.cpu()
    for b, ((want, w, l), (tol, w_tol, l_tol)) in enumerate(
            paged.attend(q, host["k"], host["v"], host["table"], lengths, scale)):
        err = (out[b].double() - want).abs()
        assert (err <= tol).all(), (b, float((err / tol.clamp_min(1e-300)).max()))
        if weights is not None:
            err = (weights[b, :, :w.shape[1]].double() - w).abs()
            assert (err <= w_tol).all(), (b, float((err / w_tol.clamp_min(1e-300)).max()))
        if lse is not None:
            same = torch.isinf(l) & (lse[b].double() == l)
            assert (((lse[b].double() - l).abs() <= l_tol) | same).all(), b


ATTEND = [
    # lengths, kv_heads, group, dim, page, dtype
    ([1], 1, 1, 128, 16, BF16),
    ([75], 8, 4, 128, 16, BF16),
    ([0, 1, 31, 32, 33], 2, 4, 128, 16, BF16),
    ([129, 5, 0, 640], 2, 4, 64, 16, BF16),
    ([300, 77], 2, 4, 256, 32, BF16),
    ([1000], 1, 3, 128, 17, BF16),
    ([513, 100], 2, 16, 128, 64, BF16),
    ([200, 3], 1, 17, 128, 1, BF16),
    ([150], 1, 40, 64, 24, BF16),
    ([129, 5, 0, 640], 4, 6, 64, 24, FP16),
    ([1000, 31], 2, 5, 128, 16, FP16),
    ([300, 77], 1, 16, 256, 7, FP16),
    ([129, 5, 0, 640], 2, 4, 64, 16, FP32),
    ([1000, 31], 2, 7, 128, 24, FP32),
    ([300, 17], 1, 16, 256, 32, FP32),
    ([40 + 7 * b % 90 for b in range(70)], 1, 2, 64, 16, BF16),       # more sequences than lanes
    ([130] + [0] * 129 + [400], 2, 4, 64, 128, FP16),
    ([5000, 1], 1, 4, 128, 256, BF16),
]


@pytest.mark.parametrize("lengths,kv_heads,group,dim,page,dtype", ATTEND)
def test_attend(lengths, kv_heads, group, dim, page, dtype):
    log("attend", lengths[:5], kv_heads, group, dim, page, dtype)
    cache, host = make(lengths, kv_heads, dim, page, dtype, scored=True)
    q = queries(cache, group)
    lse = torch.zeros(q.shape[:2], device="cuda")
    fork = cache.fork()
    fork.scores.fill_(-7.0)
    cache.scores.zero_()
    out = cache.attend(q.cuda(), accumulate=True, lse=lse, into=fork)
    weights = fork.scores.cpu()
    check_attend(q, host, lengths, out, weights, lse.cpu())
    for b, n in enumerate(lengths):  # behind the length nothing is written
        assert (weights[b, :, n:] == -7).all()
    assert not cache.scores.any()
    # without weights the same output, bit for bit, on every call
    for _ in range(3):
        assert torch.equal(bits(cache.attend(q.cuda())), bits(out))
    cache.check_errors()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attend_scale_and_accumulation(dtype):
    lengths = [90, 200]
    cache, host = make(lengths, 2, 128, 16, dtype, scored=True)
    q = queries(cache, 4, sigma=0.5)
    before = host["scores"]
    for scale in (0.5, -0.25, 0.0):
        cache.scores.copy_(before)
        out = cache.attend(q.cuda(), scale=scale, accumulate=True)
        check_attend(q, host, lengths, out, scale=scale)
        for b, ((_, w, _), (_, tol, _)) in enumerate(paged.attend(q, host["k"], host["v"], host["table"], lengths, scale)):
            n = lengths[b]
            want = before[b, :, :n].double() + w
            err = (cache.scores[b, :, :n].cpu().double() - want).abs()
            assert (err <= tol + want * 2.0 ** -24).all()
            assert torch.equal(cache.scores[b, :, n:].cpu(), before[b, :, n:])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attend_peaked_and_wide_scores(dtype):
    """Scores far apart (one slot takes all) and all equal; values of large size."""
    lengths = [257, 300]
    cache, host = make(lengths, 1, 64, 16, dtype)
    q = queries(cache, 4, sigma=30.0)
    q[1] = 0
    out = cache.attend(q.cuda())
    check_attend(q, host, lengths, out)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("page", [16, 24])
def test_attend_scores_of_large_size(dtype, page):
    """Scores far above 2^24, where the rounding of score times scale is itself
    many units: the largest one's slot still has all the weight, once."""
    lengths, dim, group = [250, 65], 64, 3
    cache, host = make(lengths, 1, dim, page, dtype, scored=True)
    gen = torch.Generator().manual_seed(3)
    sign = torch.where(torch.rand(dim, generator=gen) < 0.5, -1.0, 1.0)
    first, last = [], []  # the slots of the smallest and largest score
    for b, n in enumerate(lengths):
        size = 1 + torch.randperm(n, generator=gen)  # (integers below 256: exact in every type)
        for t in range(n):
            host["k"][host["table"][b, t // page], 0, t % page] = (sign * size[t]).to(dtype)
        first.append(int(size.argmin()))
        last.append(int(size.argmax()))
    cache.k.copy_(host["k"])
    q = sign.expand(2, group, dim).contiguous().to(dtype)  # scores 64 * size, exact in fp32
    eps = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}[dtype]
    lse = torch.zeros(2, group, device="cuda")
    for power in (3, 9, 12, 15, 17, 20, 22, 27, 31, 60, 100):
        for factor in (0.1234, 0.777, 1.3, -0.9173):
            # (neighbouring scores lie 64 * 8 * 0.12 apart at least: e^-63 to 1)
            scale = factor * 2.0 ** power
            cache.scores.zero_()
            out = cache.attend(q.cuda(), scale=scale, accumulate=True, lse=lse).cpu().double()
            for b, n in enumerate(lengths):
                at = last[b] if scale > 0 else first[b]
                want = host["v"][host["table"][b, at // page], 0, at % page].double()
                # the rounding to the type, and four in 32 bits (two products, their sum, the quotient)
                assert ((out[b] - want).abs() <= want.abs() * (eps + 2.0 ** -21)).all(), (scale, b)
                weights = cache.scores[b, 0, :n].cpu().double()
                assert abs(float(weights[at]) - group) <= group * 2.0 ** -21, (scale, b)
                weights[at] = 0
                assert (weights <= group * 2.0 ** -60).all(), (scale, b)
                top = 64 * (n if scale > 0 else 1) * scale
                # five roundings: the scale's, the product's, the sum's, and with ln 2 two
                assert ((lse[b].cpu().double() - top).abs() <= abs(top) * 2.0 ** -21).all(), (scale, b)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attend_infinities(dtype):
    """An infinite value is the output's where its slot has weight; -infinite
    scores have none; NaN reaches the outputs of its own sequence only."""
    lengths = [70, 70, 70, 70]
    cache, host = make(lengths, 2, 64, 16, dtype)
    q = queries(cache, 3, sigma=0.3)
    clean = cache.attend(q.cuda()).cpu()
    at = [(int(host["table"][b, t // 16]), t % 16) for b, t in ((0, 69), (1, 3), (2, 17), (3, 40))]
    cache.v[at[0][0], 0, at[0][1], 5] = math.inf
    cache.v[at[1][0], 1, at[1][1], 7] = -math.inf
    cache.v[at[2][0], 0, at[2][1], 9] = math.nan
    out = cache.attend(q.cuda()).cpu()
    assert (out[0, :3, 5] == math.inf).all() and (out[1, 3:, 7] == -math.inf).all() and out[2, :3, 9].isnan().all()
    for b, heads, d in ((0, slice(0, 3), 5), (1, slice(3, 6), 7), (2, slice(0, 3), 9)):
        same = torch.ones_like(out[b], dtype=torch.bool)
        same[heads, d] = False
        assert torch.equal(bits(out[b])[same], bits(clean[b])[same])
    assert torch.equal(bits(out[3]), bits(clean[3]))
    # a key that makes a score -inf for head 0 of sequence 3
    q[3, 0, 0] = 1
    cache.k[at[3][0], 0, at[3][1], 0] = -math.inf
    out = cache.attend(q.cuda()).cpu()
    assert out[3, 0].isfinite().all()
    # NaN keys: the sequence's heads of that KV head, no other
    cache.k[at[3][0], 0, at[3][1], 0] = math.nan
    out = cache.attend(q.cuda()).cpu()
    assert out[3, :3].isnan().all() and torch.equal(bits(out[3, 3:]), bits(clean[3, 3:]))


def test_attend_all_slots_of_no_weight():
    cache, _ = make([40], 1, 64, 16, FP32)
    cache.k[:, :, :, 0] = -math.inf
    q = torch.ones(1, 2, 64, device="cuda")
    lse = torch.zeros(1, 2, device="cuda")
    out = cache.attend(q, lse=lse)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP32, 64)])
def test_strides(dtype, dim):
    """Pages as views: slots before heads, K and V of one tensor, rows with gaps."""
    lengths, page, heads = [100, 37], 16, 3
    cache, host = make(lengths, heads, dim, page, dtype, room=8)
    pages = host["k"].shape[0]
    q = queries(cache, 4)
    new = torch.randn(2, 2, heads, dim).to(dtype)
    plain = cache.attend(q.cuda())
    wide = torch.zeros(pages, page, 2, heads, dim + 16, dtype=dtype, device="cuda")
    k, v = (wide[:, :, i, :, :dim].permute(0, 2, 1, 3) for i in (0, 1))
    k.copy_(cache.k)
    v.copy_(cache.v)
    other = PagedCache.from_tensors(k, v, cache.table, cache.lengths.clone())
    assert torch.equal(bits(other.attend(q.cuda())), bits(plain))
    # rows of a wider projection: [rows, 2, heads, dim] -> k and v
    rows = new.cuda()
    other.append(rows[:, 0], rows[:, 1])
    cache.append(rows[:, 0].contiguous(), rows[:, 1].contiguous())
    assert torch.equal(bits(other.attend(q.cuda())), bits(cache.attend(q.cuda())))
    assert not wide[..., dim:].any()
    assert torch.equal(other.lengths, cache.lengths)


APPEND = [
    # lengths before, new rows (None: one each), kv_heads, dim, page, dtype
    ([0, 15, 16, 100], None, 8, 128, 16, BF16),
    ([7] * 130, None, 2, 64, 24, FP16),
    ([0, 15, 3, 100], [40, 0, 1, 17], 4, 256, 16, FP32),
    ([0, 0, 5, 5, 0], [0, 0, 33, 0, 0], 3, 64, 7, BF16),
    ([2, 1], [0, 0], 1, 128, 16, BF16),
    ([1], [1000], 8, 128, 64, FP16),
]


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("lengths,new,kv_heads,dim,page,dtype", APPEND)
def test_append(lengths, new, kv_heads, dim, page, dtype, scored):
    counts = [1] * len(lengths) if new is None else new
    log("append", lengths[:5], counts[:5], kv_heads, dim, page, dtype)
    cache, host = make(lengths, kv_heads, dim, page, dtype, room=max(counts), scored=scored, fill=3.0)
    k, v = (torch.randn(sum(counts), kv_heads, dim).to(dtype) for _ in range(2))
    ends = [sum(counts[:i]) for i in range(len(counts) + 1)]
    offsets = None if new is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    fork = cache.fork()
    cache.append(k.cuda(), v.cuda(), offsets, into=fork)
    assert torch.equal(cache.lengths.cpu(), host["lengths"])  # a step that can be taken back
    cache.append(k.cuda(), v.cuda(), offsets)
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            page_id, slot = int(host["table"][b, (n + i) // page]), (n + i) % page
            host["k"][page_id, :, slot] = k[ends[b] + i]
            host["v"][page_id, :, slot] = v[ends[b] + i]
        if scored:
            host["scores"][b, :, n:n + counts[b]] = 0
            host["positions"][b, :, n:n + counts[b]] = host["seen"][b] + torch.arange(counts[b])
    after = host["lengths"] + torch.tensor(counts, dtype=torch.int32)
    for got in (cache, fork):
        assert torch.equal(bits(got.k), bits(host["k"])) and torch.equal(bits(got.v), bits(host["v"]))
        assert torch.equal(got.lengths.cpu(), after)
        if scored:
            assert torch.equal(got.scores.cpu(), host["scores"]) and torch.equal(got.positions.cpu(), host["positions"])
            assert torch.equal(got.seen.cpu(), host["seen"] + torch.tensor(counts, dtype=torch.int32))
    cache.check_errors()


def check_evict(host, lengths, keeps, cache, into, recent=0, sinks=0):
    """Applies the definition to the host copies and compares everything."""
    page = host["k"].shape[2]
    for b, n in enumerate(lengths):
        for h in range(host["k"].shape[1]):
            scores, positions = host["scores"][b, h], host["positions"][b, h]
            for src, dst in paged.evict(scores.tolist(), positions.tolist(), n, keeps[b], int(host["seen"][b]), recent,
                                        sinks):
                scores[dst], positions[dst] = scores[src].clone(), positions[src].clone()
                for x in (host["k"], host["v"]):
                    x[host["table"][b, dst // page], h, dst % page] = \
                        x[host["table"][b, src // page], h, src % page].clone()
        m = min(n, keeps[b])
        assert int(into.lengths[b]) == m
        assert torch.equal(bits(into.scores[b, :, :m]), bits(host["scores"][b, :, :m])), b
        assert torch.equal(into.positions[b, :, :m].cpu(), host["positions"][b, :, :m]), b
    assert torch.equal(bits(cache.k), bits(host["k"])) and torch.equal(bits(cache.v), bits(host["v"]))
    assert torch.equal(into.seen.cpu(), host["seen"])


EVICT = [
    # lengths, keep, recent, sinks, kv_heads, dim, page, dtype
    ([20], 10, 0, 0, 1, 128, 16, BF16),
    ([65, 64, 63, 0, 1], 64, 8, 2, 2, 128, 16, BF16),
    ([300, 40, 700], 100, 33, 4, 3, 64, 24, FP16),
    ([100, 50], 0, 0, 0, 2, 64, 16, FP32),
    ([100, 50], 1, 1, 0, 2, 64, 17, FP32),
    ([100, 50], 99, 0, 0, 2, 256, 1, BF16),
    ([90], 20, 70, 40, 2, 128, 16, BF16),     # more protected than the budget: the lower slots
    ([500, 500], [500, 123], 5, 0, 2, 128, 16, BF16),
    ([2500, 1030], [1025, 4], 0, 0, 1, 64, 64, FP16),
]


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("lengths,keep,recent,sinks,kv_heads,dim,page,dtype", EVICT)
def test_evict(lengths, keep, recent, sinks, kv_heads, dim, page, dtype, apart):
    log("evict", lengths, keep, recent, sinks, kv_heads, dim, page, dtype)
    cache, host = make(lengths, kv_heads, dim, page, dtype, scored=True)
    keeps = keep if isinstance(keep, list) else [keep] * len(lengths)
    budget = torch.tensor(keep, dtype=torch.int32, device="cuda") if isinstance(keep, list) else keep
    into = cache
    if apart:
        into = cache.fork()
        into.scores.fill_(-1)
        into.positions.fill_(-1)
        into.lengths.fill_(-1)
    cache.evict(budget, recent=recent, sinks=sinks, into=into)
    if apart:  # the cache's own bookkeeping stays as it was
        for name in ("scores", "positions", "lengths", "seen"):
            assert torch.equal(bits(getattr(cache, name)), bits(host[name]))
    check_evict(host, lengths, keeps, cache, into, recent, sinks)
    cache.check_errors()


@pytest.mark.parametrize("values", ["ties", "zeros", "special", "falling", "rising", "close"])
def test_evict_scores(values):
    """Ties, all equal, NaN / infinities / both zeros, sorted and nearly equal scores."""
    n, keep = 1500, 700
    cache, host = make([n, n - 1], 2, 64, 16, BF16, scored=True)
    gen = torch.Generator().manual_seed(3)
    s = host["scores"]
    if values == "ties":
        s.copy_(torch.randint(0, 4, s.shape, generator=gen).float())
    elif values == "zeros":
        s.zero_()
    elif values == "special":
        pick = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1.5, 2.0, -math.nan])
        s.copy_(pick[torch.randint(0, 9, s.shape, generator=gen)])
    elif values == "close":
        s.copy_(1.0 + 2.0 ** -23 * torch.randint(0, 300, s.shape, generator=gen))
    else:
        s.copy_(torch.arange(s.shape[-1]).float().expand_as(s) * (-1 if values == "falling" else 1))
    cache.scores.copy_(s)
    cache.evict(keep, recent=20)
    check_evict(host, [n, n - 1], [keep, keep], cache, cache, 20, 0)


@pytest.mark.parametrize("lengths,keep,ties", [([70001], 30000, False), ([70001], 69990, False), ([70001], 5, True),
                                               ([16385, 9000, 0, 20000], 9000, True), ([40000, 300], 16384, True),
                                               ([16384, 16383], 8191, True), ([24576], 8192, False),
                                               ([20000] + [50] * 40, 700, False)])
@pytest.mark.parametrize("apart", [False, True])
def test_evict_long(lengths, keep, ties, apart):
    """Rows of several parts, and of one at its largest, with and without ties over their ends."""
    cache, host = make(lengths, 2, 64, 256, FP16, scored=True)
    if ties:
        host["scores"].mul_(16).floor_()
        cache.scores.copy_(host["scores"])
    into = cache.fork() if apart else cache
    cache.evict(keep, recent=3, sinks=2, into=into)
    check_evict(host, lengths, [keep] * len(lengths), cache, into, 3, 2)


def test_evict_longest():
    """Parts of more than one pass over their workgroup's registers (past 2^20
    slots), the result checked by torch's stable sort."""
    n, keep, page = 1300003, 600000, 4096
    gen = torch.Generator(device="cuda").manual_seed(0)
    pages = -(-n // page)
    k = torch.randn(pages, 1, page, 64, generator=gen, device="cuda").half()
    scores = torch.randint(0, 100000, (1, 1, pages * page), generator=gen, device="cuda").float()
    positions = torch.arange(pages * page, device="cuda").int().view(1, 1, -1).contiguous()
    table = torch.randperm(pages, generator=gen, device="cuda").int()[None]
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    cache = PagedCache.from_tensors(k, k.clone(), table, i32(n), seen=i32(n), scores=scores, positions=positions)
    before, flat = scores.clone(), k[table[0].long()].view(-1, 64).clone()
    cache.evict(keep, recent=10)
    rank = before[0, 0, :n].clone()
    rank[-10:] = math.inf
    kept = torch.zeros(n, dtype=torch.bool, device="cuda")
    kept[torch.sort(rank, descending=True, stable=True).indices[:keep]] = True
    slot = torch.arange(keep, device="cuda")
    slot[~kept[:keep]] = kept[keep:].nonzero()[:, 0] + keep
    assert int(cache.lengths) == keep
    assert torch.equal(cache.positions[0, 0, :keep], slot.int())
    assert torch.equal(cache.scores[0, 0, :keep], before[0, 0, slot])
    for x in (cache.k, cache.v):
        assert torch.equal(bits(x[table[0].long()].view(-1, 64)[:keep]), bits(flat[slot]))


def test_run_of_operators():
    """Prompts, steps that weigh the slots, a cut, and steps again: every
    output and score against the definition applied to the state so far."""
    torch.manual_seed(5)
    heads, dim, page, group = 2, 128, 16, 4
    cache = PagedCache(3, 24, 10, page_size=page, kv_heads=heads, head_dim=dim, scored=True)
    prompts = [100, 0, 37]
    cache.reserve(prompts)
    offsets = torch.tensor([0, 100, 100, 137], dtype=torch.int32, device="cuda")
    cache.append(torch.randn(137, heads, dim).bfloat16().cuda(), torch.randn(137, heads, dim).bfloat16().cuda(), offsets)
    lengths, seen = list(prompts), list(prompts)
    for step in range(12):
        cache.reserve([n + 1 for n in lengths])
        before = cache.scores.cpu()
        q = torch.randn(3, heads * group, dim).bfloat16()
        k, v = (torch.randn(3, heads, dim).bfloat16().cuda() for _ in range(2))
        out = cache(q.cuda(), k, v, accumulate=True)
        lengths, seen = [n + 1 for n in lengths], [n + 1 for n in seen]
        assert cache.lengths.tolist() == lengths and cache.seen.tolist() == seen
        host = dict(k=cache.k.cpu(), v=cache.v.cpu(), table=cache.table.cpu())
        for b, ((want, w, _), (tol, w_tol, _)) in enumerate(
                paged.attend(q, host["k"], host["v"], host["table"], lengths)):
            assert ((out[b].cpu().double() - want).abs() <= tol).all()
            old = before[b, :, :lengths[b]].double()
            old[:, -1] = 0  # the new slot
            err = (cache.scores[b, :, :lengths[b]].cpu().double() - old - w).abs()
            assert (err <= w_tol + (old + w) * 2.0 ** -24).all()
        if step in (4, 9):
            state = {name: getattr(cache, name).cpu() for name in ("k", "v", "table", "scores", "positions", "seen")}
            cache.evict(40, recent=8, sinks=2)
            check_evict(state, lengths, [40] * 3, cache, cache, 8, 2)
            lengths = [min(n, 40) for n in lengths]
            for b in range(3):
                cache.release(b, 48)
    for b, n in enumerate(lengths):  # the newest tokens and the first ones are held
        for h in range(heads):
            held = set(cache.positions[b, h, :n].tolist())
            assert len(held) == n and set(range(seen[b] - min(8, n), seen[b])) <= held
            assert set(range(min(2, seen[b]))) <= held


def test_graph_replays():
    """A captured decode step (append + weighed attend) and a captured cut,
    replayed with eager work between, equal the eager calls."""
    lengths = [50, 90]
    eager, host = make(lengths, 2, 128, 16, BF16, room=40, scored=True, fill=0.0)
    torch.manual_seed(1)
    qs = torch.randn(6, 2, 8, 128).bfloat16().cuda()
    ks, vs = (torch.randn(6, 2, 2, 128).bfloat16().cuda() for _ in range(2))
    captured, _ = make(lengths, 2, 128, 16, BF16, room=40, scored=True, fill=0.0)
    q, k, v = (x[0].clone() for x in (qs, ks, vs))
    warm = captured.fork()
    captured(q, k, v, accumulate=True, into=warm)  # makes the workspaces; the state is a fork's
    captured.evict(10, into=captured.fork())
    for name in ("k", "v", "scores", "positions"):
        getattr(captured, name).copy_(host[name])
    step, cut = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(step):
        out = captured(q, k, v, accumulate=True)
    with torch.cuda.graph(cut):
        captured.evict(48, recent=4)
    for i in range(6):
        for dst, src in ((q, qs), (k, ks), (v, vs)):
            dst.copy_(src[i])
        step.replay()
        want = eager(qs[i], ks[i], vs[i], accumulate=True)
        assert torch.equal(bits(out), bits(want))
        if i in (1, 3):
            cut.replay()
            eager.evict(48, recent=4)
        torch.cuda.synchronize()
        for name in ("lengths", "seen", "scores", "positions"):
            assert torch.equal(bits(getattr(captured, name)), bits(getattr(eager, name))), (i, name)
    fresh, _ = make([5], 1, 64, 16, BF16)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.attend(torch.zeros(1, 1, 64, dtype=BF16, device="cuda"))


def test_streams():
    """Two instances on two streams at once; each result as on its own."""
    a, _ = make([5000], 2, 128, 16, BF16, seed=1)
    b, _ = make([4000, 100], 2, 128, 16, BF16, seed=2)
    qa, qb = queries(a, 4).cuda(), queries(b, 4).cuda()
    want = bits(a.attend(qa)), bits(b.attend(qb))
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(sa):
            x = a.attend(qa)
        with torch.cuda.stream(sb):
            y = b.attend(qb)
        outs.append((x, y))
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(bits(x), want[0]) and torch.equal(bits(y), want[1])


def test_far_pages():
    """Pages that lie past 2^32 bytes."""
    pages, page, heads, dim = 35000, 64, 8, 128  # 4.3 GiB of keys
    lengths = [150]
    big_k = torch.empty(pages, heads, page, dim, dtype=BF16, device="cuda")
    big_v = torch.empty_like(big_k)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(0)
    host = dict(k=torch.randn(3, heads, page, dim, generator=gen).bfloat16(),
                v=torch.randn(3, heads, page, dim, generator=gen).bfloat16(), table=torch.tensor([[0, 1, 2]]))
    for x, name in ((big_k, "k"), (big_v, "v")):
        x[table[0].long()] = host[name].cuda()
    cache = PagedCache.from_tensors(big_k, big_v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    q = queries(cache, 4)
    check_attend(q, host, lengths, cache.attend(q.cuda()))
    rows = torch.randn(1, heads, dim).bfloat16().cuda()
    cache.append(rows, rows)
    assert torch.equal(bits(big_k[pages - 2, :, 150 - 128]), bits(rows[0]))


def test_slots_without_pages_are_reported():
    cache, host = make([40, 20], 2, 64, 16, BF16, scored=True)
    q = queries(cache, 4).cuda()
    cache.attend(q)
    for bad in (-1, 10 ** 6):
        cache.table[0, 1] = bad
        cache.attend(q)  # reads page 0 in its place
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="has no page"):
            cache.attend(q)
        cache.table[0, 1] = host["table"][0, 1].cuda()
        cache.attend(q)  # (the report was cleared)
        torch.cuda.synchronize()
        cache.check_errors()
    # moves from a slot without a page are left out
    cache.scores.copy_(torch.arange(cache.slots).float().expand_as(host["scores"]))
    cache.table[0, 2] = -1
    before = bits(cache.k)
    cache.evict(8)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="has no page"):
        cache.check_errors()
    assert torch.equal(bits(cache.k)[host["table"][0].long()], before[host["table"][0].long()])
    # rows behind the table's end are dropped and reported; nothing else is written
    k = torch.ones(2, 2, 64, dtype=BF16, device="cuda")
    full, host = make([48, 20], 2, 64, 16, BF16, fill=2.0)
    full.append(k, k)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="has no page"):
        full.check_errors()
    assert full.lengths.tolist() == [48, 21]
    host["k"][host["table"][1, 1], :, 4] = 1
    assert torch.equal(bits(full.k), bits(host["k"]))
    full.check_errors()


@pytest.mark.parametrize("bad", [[0, 2, 4], [0, 4, 3], [1, 2, 3], [0, 3, 2], [-1, 2, 3]])
def test_offsets_that_do_not_fit_are_reported(bad):
    for apart in (False, True):
        cache, _ = make([20, 3], 2, 64, 16, BF16, room=8, scored=True)
        rows = torch.zeros(3, 2, 64, dtype=BF16, device="cuda")
        cache.append(rows, rows, torch.tensor(bad, dtype=torch.int32, device="cuda"), into=cache.fork() if apart else None)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="offsets"):
            cache.check_errors()


def test_many_sequences():
    """More sequences than one load of the lengths finds, short and empty ones
    between a long one's."""
    lengths = [(7 * b) % 40 for b in range(700)]
    lengths[3], lengths[411], lengths[699] = 3000, 900, 0
    cache, host = make(lengths, 1, 64, 32, BF16, scored=True)
    q = queries(cache, 2)
    out = cache.attend(q.cuda(), accumulate=True, into=cache.fork())
    pick = list(range(0, 20)) + list(range(400, 420)) + list(range(690, 700))
    few = dict(host, table=host["table"][pick])
    check_attend(q[pick], few, [lengths[b] for b in pick], out[pick])


@pytest.mark.parametrize("kv_heads,group,dim,page,dtype", [(1, 17, 64, 16, BF16), (2, 4, 128, 16, FP16), (1, 3, 256, 24, BF16),
                                                           (2, 16, 128, 7, FP32), (3, 1, 256, 32, FP32)])
def test_many_short_sequences(kv_heads, group, dim, page, dtype):
    """A wave for each pair: up to 512 tokens, 512 pairs or more; as soon as one
    sequence is longer, workgroups again, with the same bounds."""
    lengths = [(37 * b) % 513 for b in range(520 // kv_heads)]
    lengths[-1], lengths[100] = 512, 0
    cache, host = make(lengths, kv_heads, dim, page, dtype, room=1, scored=True)
    q = queries(cache, group)
    pick = [0, 1, 2, 99, 100, 101, 120, len(lengths) - 1]
    few = dict(host, table=host["table"][pick])
    for longest in (512, 513):
        fork = cache.fork()
        fork.scores.fill_(-7.0)
        cache.scores.zero_()
        lse = torch.zeros(q.shape[:2], device="cuda")
        if longest == 513:  # (one more token: a row of zeros)
            at = host["table"][-1, 512 // page]
            for x in (cache.k, cache.v, few["k"], few["v"]):
                x[at, :, 512 % page] = 0
            cache.lengths[-1] = 513
            lengths[-1] = 513
        out = cache.attend(q.cuda(), accumulate=True, lse=lse, into=fork)
        check_attend(q[pick], few, [lengths[b] for b in pick], out[pick], fork.scores[pick].cpu(), lse[pick].cpu())
        for b in pick:
            assert (fork.scores[b, :, lengths[b]:] == -7).all()
        assert torch.equal(bits(cache.attend(q.cuda())), bits(out))
    cache.check_errors()


@pytest.mark.parametrize("dim,group,dtype", [(128, 16, BF16), (256, 16, FP16), (128, 16, FP32), (64, 40, BF16)])
def test_wide_calls_in_a_graph(dim, group, dtype):
    """The calls that take most LDS and a second launch, captured."""
    lengths = [9000, 300]
    cache, host = make(lengths, 1, dim, 64, dtype, scored=True, fill=0.0)
    q = queries(cache, group).cuda()
    fork = cache.fork()
    want = cache.attend(q, accumulate=True, into=fork)
    scores = fork.scores.clone()
    check_attend(q.cpu(), host, lengths, want)
    after = cache.fork()
    cache.evict(7000, recent=5, into=after)
    positions = after.positions[:, :, :300].clone()
    cache.k.copy_(host["k"])
    cache.v.copy_(host["v"])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = cache.attend(q, accumulate=True, into=fork)
        cache.evict(7000, recent=5, into=after)
    for _ in range(3):
        for x in (fork.scores, after.positions, after.lengths):
            x.zero_()
        cache.k.copy_(host["k"])
        cache.v.copy_(host["v"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(want)) and after.lengths.tolist() == [7000, 300]
        for b, n in enumerate(lengths):
            assert torch.equal(fork.scores[b, :, :n], scores[b, :, :n])
        assert torch.equal(after.positions[:, :, :300], positions)


def test_reserve_and_release():
    cache = PagedCache(2, 6, 4, page_size=16, kv_heads=1, head_dim=64)
    cache.reserve([17, 1])
    assert (cache.table >= 0).sum(1).tolist() == [2, 1]
    with pytest.raises(RuntimeError, match="pages wanted"):
        cache.reserve([64, 64])
    assert (cache.table >= 0).sum(1).tolist() == [2, 1]
    cache.reserve([64, 20])
    used = cache.table[cache.table >= 0].tolist()
    assert len(used) == len(set(used)) == 6
    cache.release(0, 20)
    assert (cache.table >= 0).sum(1).tolist() == [2, 2]
    cache.reserve([0, 64])
    assert (cache.table >= 0).sum(1).tolist() == [2, 4]
    with pytest.raises(ValueError, match="token counts"):
        cache.reserve(65)
    with pytest.raises(RuntimeError, match="kept by the caller"):
        cache.fork().reserve(1)


def test_refusals():
    cache, _ = make([20, 3], 2, 128, 16, BF16)
    k = torch.zeros(2, 2, 128, dtype=BF16, device="cuda")
    q = torch.zeros(2, 8, 128, dtype=BF16, device="cuda")
    bad_q = [q[:1], q[:, :7], q[..., :64], q.float(), q.cpu(), torch.zeros(2, 8, 256, dtype=BF16, device="cuda")[..., ::2],
             torch.zeros(2 * 8 * 128 + 1, dtype=BF16, device="cuda")[1:].view(2, 8, 128)]
    for x in bad_q:
        with pytest.raises(ValueError):
            cache.attend(x)
    with pytest.raises(ValueError, match="scored"):
        cache.attend(q, accumulate=True)
    with pytest.raises(ValueError, match="scored"):
        cache.evict(4)
    for scale in (math.nan, math.inf):
        with pytest.raises(ValueError, match="finite"):
            cache.attend(q, scale=scale)
    with pytest.raises(ValueError, match="lse"):
        cache.attend(q, lse=torch.zeros(2, 4, device="cuda"))
    for kk, vv in ((k[:1], k[:1]), (k.float(), k.float()), (k, k[:1]), (k.cpu(), k.cpu()), (k[:, :1], k[:, :1])):
        with pytest.raises(ValueError):
            cache.append(kk, vv)
    with pytest.raises(ValueError, match="offsets"):
        cache.append(k, k, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        cache(q[:, :7], k, k)
    assert cache.lengths.tolist() == [20, 3]  # nothing appended for the refused query
    other, _ = make([20, 3], 2, 128, 16, BF16)
    with pytest.raises(ValueError, match="fork"):
        cache.append(k, k, into=other)
    with pytest.raises(NotImplementedError):
        PagedCache.from_tensors(k.view(1, 2, 2, 128)[..., :96], k.view(1, 2, 2, 128)[..., :96], cache.table, cache.lengths)
    with pytest.raises(NotImplementedError):
        PagedCache(1, 4, 4, dtype=torch.float64)
    with pytest.raises(ValueError, match="equal strides"):
        PagedCache.from_tensors(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2), cache.table, cache.lengths)
    with pytest.raises(ValueError, match="together"):
        PagedCache.from_tensors(cache.k, cache.v, cache.table, cache.lengths, seen=cache.lengths)
    scored, _ = make([20, 3], 2, 128, 16, BF16, scored=True)
    for bad in (-1, 2 ** 31, torch.zeros(3, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            scored.evict(bad)
    with pytest.raises(ValueError):
        scored.evict(4, recent=-1)
