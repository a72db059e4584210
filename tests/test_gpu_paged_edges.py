"""The paged cache where its operators are easily wrong: outputs that cancel,
infinite values of little weight, wide page tables, shared buffers, the
largest calls.  Bounds are derived beside each test."""
import math

import pytest
import torch

from prismkv_amd import PagedCache
from tests.gpu_util import log
from tests.test_gpu_paged import BF16, FP16, FP32, bits

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_outputs_that_cancel(dtype):
    """Sums of p v that are near 0 beside their terms, where the output's own
    rounding hides nothing: p is used with 32 bits in every type.

    Four tokens a sequence, one query head to a KV head.  A score is one product
    (the other dims of q are 0), exact in fp32, and the largest is 0.  A weight's
    exponent has two roundings, the scale's and its own: with the exponential's,
    2^-23, p is off by less than 2 * 2^-23 + 2^-23 < 2^-21 of itself where |s| <= 2, and
    by 2^-19 for the token of 6.24, whose term is 2^-8 of the others at most.  As
    the terms' sum is near 0 the denominator's error does not count.  p as terms of
    the type is exact (three of bf16; fp32 itself) or off by 2^-22 (two of fp16).
    The products are exact in fp32 and the first terms' sum takes four roundings,
    of 2^-23 each where the matrix cores should truncate; the other terms add to
    what that left, 2^-7 of it.  All together: (0.5 + 0.01 + 0.25 + 0.52) 2^-20 of
    sum p |v|, held to 2^-19, and the output's own rounding."""
    gen = torch.Generator().manual_seed(11)
    sequences, heads, dim = 64, 4, 64
    step = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}[dtype]
    # scores 0, two in [-2, 0], -6.24: one product each
    s = torch.zeros(sequences, heads, 4, dtype=torch.float64)
    s[:, :, 1:3] = -2 * torch.rand(sequences, heads, 2, generator=gen, dtype=torch.float64)
    s[:, :, 3] = -6.24
    k = torch.zeros(sequences, heads, 16, dim)
    k[:, :, :4, 0] = s.float()
    k = k.to(dtype)
    q = torch.zeros(sequences, heads, dim, dtype=dtype)
    q[:, :, 0] = 1
    p = torch.exp(k[:, :, :4, 0].double())
    p /= p.sum(-1, keepdim=True)
    # values: two at random, then what cancels, rounded, and once more for the rest
    v = torch.zeros(sequences, heads, 16, dim, dtype=dtype)
    v[:, :, :2] = torch.randn(sequences, heads, 2, dim, generator=gen).to(dtype)
    for t in (2, 3):
        rest = (p[..., None] * v[:, :, :4].double()).sum(2)
        v[:, :, t] = (-rest / p[:, :, t, None]).to(dtype)
    want = (p[..., None] * v[:, :, :4].double()).sum(2)
    spread = (p[..., None] * v[:, :, :4].double().abs()).sum(2)
    assert (want.abs() * step < 2.0 ** -22 * spread).all()  # (they do cancel)
    cache = PagedCache.from_tensors(k.cuda(), v.cuda(), torch.arange(sequences, dtype=torch.int32, device="cuda")[:, None],
                                    i32(*[4] * sequences))
    out = cache.attend(q.cuda(), scale=1.0).cpu().double()
    smallest = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}[dtype]  # half the least subnormal
    error = (out - want).abs() / (spread * 2.0 ** -19 + want.abs() * step + smallest)
    log("largest error over its bound", dtype, float(error.max()))
    assert (error <= 1).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("page", [16, 24])
def test_infinite_values_of_little_weight(dtype, page):
    """An infinite value is the output's wherever its slot has weight in 32 bits
    (2^-126 of the largest and more), and changes no other dim.

    The other dims: weight 1 and one of 2^-10 at most, the bounds of
    test_outputs_that_cancel; fp16 terms no less than 2^-24 of 2^15 add
    2 * 2^-39 |v|."""
    powers = [10, 20, 29, 31, 36, 40, 45, 60, 100, 120]
    dim = 64
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.zeros(len(powers), 1, page, dim, dtype=dtype) for _ in range(2))
    k[:, 0, 1, 0] = -math.log(2) * torch.tensor(powers).to(dtype)
    v[:, 0, :2] = torch.randn(len(powers), 2, dim, generator=gen).to(dtype)
    p = torch.exp(k[:, 0, :2, 0].double())
    p /= p.sum(-1, keepdim=True)
    want = (p[..., None] * v[:, 0, :2].double()).sum(1)
    spread = (p[..., None] * v[:, 0, :2].double().abs()).sum(1)
    v[:, 0, 1, 5], v[:, 0, 1, 40] = math.inf, -math.inf
    q = torch.zeros(len(powers), 1, dim, dtype=dtype)
    q[..., 0] = 1
    cache = PagedCache.from_tensors(k.cuda(), v.cuda(), torch.arange(len(powers), dtype=torch.int32, device="cuda")[:, None],
                                    i32(*[2] * len(powers)))
    out = cache.attend(q.cuda(), scale=1.0).cpu()[:, 0].double()
    assert (out[:, 5] == math.inf).all(), out[:, 5]
    assert (out[:, 40] == -math.inf).all(), out[:, 40]
    step = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}[dtype]
    smallest = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}[dtype]
    other = [d for d in range(dim) if d not in (5, 40)]
    v_max = v[:, 0, :2, other].double().abs().amax()
    bound = want.abs() * step + spread * 2.0 ** -19 + v_max * 2.0 ** -38 + smallest
    assert ((out - want).abs() <= bound)[:, other].all()


def test_a_report_outlives_resizing():
    """Rows dropped for want of a page are reported to the cache that takes
    this one's place."""
    for fork in (False, True):
        cache = PagedCache(2, 8, 4, page_size=16, kv_heads=2, head_dim=64, scored=True)
        cache.reserve([16, 0])
        rows = torch.ones(20, 2, 64, dtype=BF16, device="cuda")
        cache.append(rows, rows, i32(0, 16, 20), into=cache.fork() if fork else None)  # (the second sequence has no page)
        cache = cache.resized(6, 3)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="has no page"):
            cache.check_errors()
        cache.check_errors()


def test_resized():
    """The contents of sequences of different page counts, and what runs on them."""
    gen = torch.Generator().manual_seed(2)
    lengths = [37, 0, 64, 5]
    cache = PagedCache(4, 20, 8, page_size=16, kv_heads=2, head_dim=64, scored=True)
    cache.reserve([50, 20, 64, 5])  # (more than the lengths)
    rows = torch.randn(sum(lengths), 2, 64, generator=gen).bfloat16().cuda()
    ends = i32(0, 37, 37, 101, 106)
    cache.append(rows, -rows, ends)
    q = torch.randn(4, 4, 64, generator=gen).bfloat16().cuda()
    cache.attend(q, accumulate=True)
    cache.release(1)
    for pages, max_pages in ((9, 4), (30, 12)):
        new = cache.resized(pages, max_pages)
        assert new.k.shape[0] == pages and new.table.shape[1] == max_pages
        assert (new.table >= 0).sum(1).tolist() == [4, 0, 4, 1]
        used = new.table[new.table >= 0].tolist()
        assert len(set(used)) == 9
        for b, n in enumerate(lengths):
            at = torch.arange(n, device="cuda")
            place = [(c.table[b, at // 16].long(), at % 16) for c in (cache, new)]
            for x, y in ((cache.k, new.k), (cache.v, new.v)):
                assert torch.equal(bits(x[place[0][0], :, place[0][1]]), bits(y[place[1][0], :, place[1][1]]))
            assert torch.equal(new.scores[b, :, :n], cache.scores[b, :, :n])
            assert torch.equal(new.positions[b, :, :n], cache.positions[b, :, :n])
        assert torch.equal(new.lengths, cache.lengths) and torch.equal(new.seen, cache.seen)
        assert torch.equal(bits(new.attend(q)), bits(cache.attend(q)))
        new.evict(20, recent=3)
        old = cache.resized(20, 8)
        old.evict(20, recent=3)
        for b in range(4):
            m = min(lengths[b], 20)
            assert torch.equal(new.positions[b, :, :m], old.positions[b, :, :m])
        new.check_errors()
    with pytest.raises(ValueError, match="do not fit"):
        cache.resized(8, 4)


def test_more_caches_than_a_page_of_error_words():
    """Made and let go one after another with work queued: a report reaches its own cache only."""
    q = torch.zeros(1, 1, 64, dtype=BF16, device="cuda")
    for i in range(700):
        cache = PagedCache(1, 1, 1, page_size=16, kv_heads=1, head_dim=64)
        if i % 3:
            cache.reserve(1)
        cache.lengths.fill_(1)
        cache.attend(q)
        if i % 50 < 3:
            torch.cuda.synchronize()
            if i % 3:
                cache.check_errors()
            else:
                with pytest.raises(RuntimeError, match="has no page"):
                    cache.check_errors()


def test_buffers_that_overlap_are_refused():
    """Lengths, tokens seen, scores and positions are buffers of their own, and a
    cache that results go to has either all of this one's or none."""
    k = torch.zeros(4, 2, 16, 64, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    q = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")

    def state():
        return dict(lengths=i32(3, 4), seen=i32(3, 4), scores=torch.zeros(2, 2, 32, device="cuda"),
                    positions=torch.zeros(2, 2, 32, dtype=torch.int32, device="cuda"))

    def made(x):
        return PagedCache.from_tensors(k, v, table, x["lengths"], seen=x["seen"], scores=x["scores"], positions=x["positions"])

    own = state()
    with pytest.raises(ValueError, match="overlap"):
        made(dict(own, seen=own["lengths"]))
    with pytest.raises(ValueError, match="overlap"):
        made(dict(own, positions=own["scores"].view(torch.int32)))
    words = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        made(dict(own, lengths=words[:2], seen=words[1:]))
    cache = made(own)
    for name in own:
        with pytest.raises(ValueError, match="overlap"):
            cache.attend(q, into=made(dict(state(), **{name: own[name]})))
    longer = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        made(dict(own, lengths=longer[:2])).attend(q, into=made(dict(state(), seen=longer[1:])))
    cache.attend(q, into=made(own))      # all of them: the cache itself
    cache.attend(q, into=made(state()))  # none
    cache.attend(q, into=cache.fork())
    fork = cache.fork()
    fork.attend(q, into=fork.fork())
    unscored = [PagedCache.from_tensors(k, v, table, x) for x in (own["lengths"], own["lengths"], own["seen"])]
    unscored[0].attend(q, into=unscored[1])
    unscored[0].attend(q, into=unscored[2])


@pytest.mark.parametrize("default", [BF16, FP16, torch.float64])
def test_default_types_do_not_matter(default):
    """Scores are float32 whatever torch's default type is."""
    torch.set_default_dtype(default)
    try:
        cache = PagedCache(1, 4, 4, page_size=16, kv_heads=1, head_dim=64, scored=True)
        cache.reserve(20)
        new = cache.resized(2, 2)
    finally:
        torch.set_default_dtype(FP32)
    assert cache.scores.dtype == new.scores.dtype == FP32


def test_default_devices_do_not_matter(monkeypatch):
    """The error word lies in host memory whatever torch's default device is."""
    from prismkv_amd import paged as module
    monkeypatch.setattr(module._ErrorWord, "homes", {})  # (the first cache makes its page of words)
    with torch.device("cuda"):
        cache = PagedCache(2, 4, 4, page_size=16, kv_heads=1, head_dim=64, scored=True)
        cache.reserve([20, 3])
        new = cache.resized(3, 2)
        q = torch.zeros(2, 1, 64, dtype=BF16)
        assert not new.attend(q).any() and not new.fork().attend(q).any()
    new.check_errors()


def test_rows_beyond_one_launch():
    """More packed rows than one launch has threads for (2^27 rows of 8 a
    workgroup of 256 would take 2^32), on two sequences, in place and into a fork."""
    rows, page = (1 << 27) + 1000, 1 << 16
    gen = torch.Generator().manual_seed(0)
    few = 1 << 12
    pages = [rows // page, 2]
    shape = (sum(pages), 1, page, 64)
    k = torch.zeros(shape, dtype=BF16, device="cuda")
    v = torch.zeros(shape, dtype=BF16, device="cuda")
    table = torch.full((2, pages[0]), -1, dtype=torch.int32)
    table[0] = torch.arange(pages[0]).flip(0)
    table[1, :2] = torch.arange(pages[0], sum(pages))
    cache = PagedCache.from_tensors(k, v, table.cuda(), i32(0, 5))
    one = torch.randn(few, 64, generator=gen).bfloat16().cuda()
    new = torch.empty(rows, 1, 64, dtype=BF16, device="cuda")
    for at in range(0, rows, few):  # (block i of the rows: `one` turned by i)
        n = min(few, rows - at)
        new[at:at + n, 0] = one.roll(at // few, 0)[:n]
    first = pages[0] * page  # rows of the first sequence; the rest is the second's
    ends = i32(0, first, rows)
    fork = cache.fork()
    for to in (fork, cache):
        k.zero_()
        v.zero_()
        cache.append(new, new, ends, into=to)
        torch.cuda.synchronize()
        cache.check_errors()
        assert to.lengths.tolist() == [first, 5 + rows - first]
        for x in (k, v):
            for b in range(pages[0]):
                assert torch.equal(x[int(table[0, b]), 0], new[b * page:(b + 1) * page, 0])
            flat = x[pages[0]:].view(-1, 64)
            assert torch.equal(flat[5:5 + rows - first], new[first:, 0])
            assert not flat[:5].any() and not flat[5 + rows - first:].any()
    assert fork.lengths.tolist() == cache.lengths.tolist()
    del x, k, v, new, flat, cache, fork, to
    torch.cuda.empty_cache()


def test_lengths_past_the_table():
    """Read as the table's slots: a row is dropped and reported, the length stays there."""
    for far in (33, 2 ** 31 - 1):
        for offsets in (None, i32(0, 1, 2)):
            cache = PagedCache(2, 4, 2, page_size=16, kv_heads=1, head_dim=64)
            cache.reserve(32)
            cache.lengths.copy_(i32(far, 3))
            rows = torch.ones(2, 1, 64, dtype=BF16, device="cuda")
            cache.append(rows, rows, offsets)
            assert cache.lengths.tolist() == [32, 4]
            assert int(cache.k.count_nonzero()) == 64
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="has no page"):
                cache.check_errors()


def test_scales_that_32_bits_do_not_hold_are_refused():
    cache = PagedCache(1, 1, 1, page_size=16, kv_heads=1, head_dim=64)
    cache.reserve(1)
    cache.lengths.fill_(1)
    q = torch.zeros(1, 1, 64, dtype=BF16, device="cuda")
    for scale in (3e38, -3e38, 1e300):  # (times log2(e), as the kernels have it)
        with pytest.raises(ValueError, match="finite"):
            cache.attend(q, scale=scale)
    for scale in (2e38, 0.0, 1e-300):
        assert not cache.attend(q, scale=scale).any()


def test_a_step_that_is_refused_appends_nothing():
    """Also where it is the size of the call that cannot be attended to."""
    k = torch.zeros(1, 1, 1 << 20, 64, dtype=BF16, device="cuda")
    cache = PagedCache.from_tensors(k, torch.zeros_like(k), torch.zeros(1, 1 << 10, dtype=torch.int32, device="cuda"), i32(3))
    q = torch.zeros(1, 1024, 64, dtype=BF16, device="cuda")
    row = torch.ones(1, 1, 64, dtype=BF16, device="cuda")
    for call in (lambda: cache(q, row, row), lambda: cache.attend(q)):
        with pytest.raises(NotImplementedError, match="2\\^31"):
            call()
    assert cache.lengths.tolist() == [3] and not k.any()
    cache(q[:, :512].contiguous(), row, row)  # half as many query heads
    assert cache.lengths.tolist() == [4]


def test_a_step_without_its_workspace_is_not_captured():
    cache = PagedCache(1, 2, 2, page_size=16, kv_heads=1, head_dim=64)
    cache.reserve(20)
    q = torch.zeros(1, 2, 64, dtype=BF16, device="cuda")
    row = torch.ones(1, 1, 64, dtype=BF16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        filler = q + 1
        with pytest.raises(RuntimeError, match="before the capture"):
            cache(q, row, row)
    graph.replay()
    torch.cuda.synchronize()
    assert cache.lengths.tolist() == [0] and not cache.k.any() and filler.bool().all()


@pytest.mark.parametrize("width", [40, 2048])
def test_tables_wider_than_the_sequences(width):
    """Room for far longer sequences than there are: a step that weighs, cuts (by
    one launch, and by the launches of rows as long as the table) and steps again."""
    from oracle import paged
    from tests.test_gpu_paged import check_attend, check_evict, make, queries
    lengths, heads, page = [300, 0, 41], 2, 16
    narrow, host = make(lengths, heads, 64, page, BF16, room=20, scored=True)
    slots = width * page
    table = torch.full((3, width), -1, dtype=torch.int32)
    table[:, :host["table"].shape[1]] = host["table"]
    gen = torch.Generator().manual_seed(1)
    host.update(table=table, scores=torch.zeros(3, heads, slots), seen=torch.tensor(lengths, dtype=torch.int32),
                positions=torch.arange(slots, dtype=torch.int32).expand(3, heads, slots).clone())
    cache = PagedCache.from_tensors(narrow.k, narrow.v, table.cuda(), narrow.lengths, seen=host["seen"].cuda(),
                                    scores=host["scores"].cuda(), positions=host["positions"].cuda())
    for keep in (None, 120, 60, 4):
        q = queries(cache, 4, seed=keep or 0)
        k, v = (torch.randn(3, heads, 64, generator=gen).bfloat16() for _ in range(2))
        before = cache.scores.cpu()
        out = cache(q.cuda(), k.cuda(), v.cuda(), accumulate=True)
        lengths = [n + 1 for n in lengths]
        state = {n: getattr(cache, n).cpu() for n in ("k", "v", "table", "scores", "positions", "seen")}
        check_attend(q, state, lengths, out)
        for b, ((_, w, _), (_, tol, _)) in enumerate(paged.attend(q, state["k"], state["v"], table, lengths)):
            old = before[b, :, :lengths[b]].double()
            old[:, -1] = 0
            got = cache.scores[b, :, :lengths[b]].cpu().double()
            assert ((got - old - w).abs() <= tol + (old + w) * 2.0 ** -24).all()
        if keep:
            cache.evict(keep, recent=5, sinks=1)
            check_evict(state, lengths, [keep] * 3, cache, cache, 5, 1)
            lengths = [min(n, keep) for n in lengths]
    cache.check_errors()


def test_a_cut_into_a_fork_may_be_repeated_only():
    """The rows move in the pages that the original shares: the same cut, into another
    fork or in place, leaves the same; attending to the original would read moved rows."""
    from tests.test_gpu_paged import make, queries
    cache, host = make([300, 90], 2, 64, 16, BF16, scored=True)
    q = queries(cache, 2).cuda()
    first, second = cache.fork(), cache.fork()
    before = bits(cache.attend(q))
    cache.evict(50, recent=4, into=first)
    pages, out = bits(cache.k), bits(first.attend(q))
    assert cache.lengths.tolist() == [300, 90] and not torch.equal(bits(cache.attend(q)), before)
    cache.evict(50, recent=4, into=second)
    cache.evict(50, recent=4)
    assert torch.equal(bits(cache.k), pages)
    for other in (second, cache):
        assert torch.equal(bits(other.attend(q)), out)
        for name in ("lengths", "seen"):
            assert torch.equal(getattr(other, name), getattr(first, name))
        for name in ("scores", "positions"):
            assert torch.equal(getattr(other, name)[:, :, :50], getattr(first, name)[:, :, :50])


def plain_attend(q, k, v, n):
    """Softmax attention in 64 bits of q [..., G, D] over k, v [..., S, D], slots [0, n) of each."""
    s = (q.double() @ k.double().transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    s = s.masked_fill(torch.arange(k.shape[-2]) >= n[..., None, None], -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))  # (no slot: no weight)
    return p @ v.double(), p, (p @ v.double().abs())


@pytest.mark.parametrize("many", ["sequences", "heads"])
def test_the_most_sequences_and_heads(many):
    """65535 of each: append, a weighed step and a cut, against all of them in 64
    bits.  The sums of 64 |q k| stay below 8, scores are off by (64 + 8) 2^-24 of an
    eighth of that, less than 2^-17.8, weights and outputs by twice that and the
    exponential's 2^-20: 2^-16, and fp32's rounding."""
    count, page, dim, group = 65535, 4, 64, 2
    B, H = (count, 1) if many == "sequences" else (1, count)
    gen = torch.Generator().manual_seed(7)
    cache = PagedCache(B, B, 1, page_size=page, kv_heads=H, head_dim=dim, dtype=FP32, scored=True)
    cache.reserve(page)
    new = torch.randint(0, 4, (B,), generator=gen) if B > 1 else torch.tensor([3])
    rows = int(new.sum())
    k, v = (torch.rand(rows, H, dim, generator=gen) - 0.5 for _ in range(2))
    ends = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).int().cuda()
    cache.append(k.cuda(), v.cuda(), ends)
    assert torch.equal(cache.lengths.cpu(), new.int())
    q = torch.rand(B, H * group, dim, generator=gen) - 0.5
    one = torch.rand(2, B, H, dim, generator=gen) - 0.5
    out = cache(q.cuda(), one[0].cuda(), one[1].cuda(), accumulate=True).cpu()
    n = new + 1
    # [B, H, page, dim] of what was written
    full = torch.zeros(2, B, H, page, dim)
    b = torch.repeat_interleave(torch.arange(B), new)
    slot = torch.arange(rows) - torch.repeat_interleave(new.cumsum(0) - new, new)
    full[0][b, :, slot], full[1][b, :, slot] = k, v
    full[0][torch.arange(B), :, new], full[1][torch.arange(B), :, new] = one[0], one[1]
    order = cache.table[:, 0].long()
    used = torch.arange(page) < n[:, None]
    for x, y in ((cache.k, full[0]), (cache.v, full[1])):
        assert torch.equal(x[order].cpu().transpose(1, 2)[used], y.transpose(1, 2)[used])
    want, p, spread = plain_attend(q.view(B, H, group, dim), full[0], full[1], n[:, None].expand(B, H))
    assert ((out.view(want.shape).double() - want).abs() <= spread * 2.0 ** -16 + want.abs() * 2.0 ** -24).all()
    weights = p.sum(2)
    got = cache.scores.cpu()
    assert ((got.double() - weights).abs() <= weights * 2.0 ** -16)[used[:, None].expand_as(got)].all()
    # two slots stay: the newest and the heaviest other
    before = {name: getattr(cache, name).cpu() for name in ("k", "v", "positions", "scores")}
    cache.evict(2, recent=1)
    assert torch.equal(cache.lengths.cpu(), n.clamp(max=2).int())
    rank = before["scores"].masked_fill(~used[:, None], -1.0)
    newest = torch.arange(page) == (n - 1)[:, None]
    rank = rank.masked_fill(newest[:, None], 1e9)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :2].sort(-1).values
    held = cache.positions.cpu()[..., :2].sort(-1).values
    live = (n >= 2)[:, None, None].expand_as(kept)
    assert torch.equal(held[live].long(), kept[live])
    cache.check_errors()
