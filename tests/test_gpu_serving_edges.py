"""Where the serving operators of the paged cache are easily wrong: bad pages and
offsets, strides, pages far apart, graphs, streams, cuts, and a run of all together."""
import math

import pytest
import torch

from oracle import paged
from prismkv_amd import PagedCache, Rotary
from tests.serving_util import BF16, FP16, FP32, check_prompt, ends, make, rows_like

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ reports and refusals

@pytest.mark.parametrize("storage", [None, "mxfp4"])
def test_a_missing_page_is_reported(storage):
    cache, _ = make([100, 40], 2, 128, 16, BF16, storage)
    cache.table[0, 2] = -1
    q = rows_like(cache, 20, 4).cuda()
    e = ends([10, 10])
    for call in (lambda: cache.attend_prompt(q, e), lambda: cache.read(ends([90, 1]), rows=91), lambda: cache.attend(q[:2])):
        call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="no page"):
            cache.check_errors()
        cache.check_errors()
    k, v = cache.read(ends([90, 1]), rows=91)
    torch.cuda.synchronize()
    missing = slice(32 - 10, 48 - 10)
    assert (k[missing] == 0).all() and (v[missing] == 0).all() and torch.isfinite(k).all()


def test_a_page_out_of_range_is_reported():
    cache, _ = make([100], 2, 128, 16, BF16, room=10)
    cache.table[0, 6] = 10 ** 6
    rotary = Rotary(128)
    x = rows_like(cache, 1, 2).cuda()
    cache.append(x, x, rotary=rotary)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="no page"):
        cache.check_errors()


@pytest.mark.parametrize("bad", [[0, 5, 11], [1, 5, 12], [0, 7, 5], [0, 20, 12], [0, -3, 12], [5, 5, 12]])
def test_offsets_that_do_not_cover_the_rows(bad):
    cache, _ = make([60, 70], 2, 64, 16, BF16)
    e = torch.tensor(bad, dtype=torch.int32, device="cuda")
    q = rows_like(cache, 12, 4).cuda()
    out = cache.attend_prompt(q, e)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="offsets of a prompt or a read"):
        cache.check_errors()
    assert out.shape == q.shape
    cache.read(e, rows=12)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="offsets of a prompt or a read"):
        cache.check_errors()
    x = rows_like(cache, 12, 2).cuda()
    room, _ = make([3, 4], 2, 64, 16, BF16, room=40)
    room.append(x, x, e, rotary=Rotary(64))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="offsets of an append"):
        room.check_errors()


def test_more_rows_than_a_sequence_holds():
    cache, host = make([3, 30], 1, 64, 16, BF16)
    q = rows_like(cache, 15, 2).cuda()
    lse = torch.empty(15, 2, device="cuda")
    out = cache.attend_prompt(q, ends([5, 10]), lse=lse)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="more rows than a sequence holds"):
        cache.check_errors()
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    check_prompt(q.cpu()[2:], host, [3, 30], [3, 10], out[2:], lse[2:])
    k, _ = cache.read(ends([5, 10]), rows=15)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="more rows than a sequence holds"):
        cache.check_errors()
    assert (k[:2] == 0).all() and torch.equal(k[2:5].cpu(), paged.rows(host["k"], host["table"][0], 3).transpose(0, 1))


def test_refused_calls():
    cache, _ = make([30, 40], 2, 128, 16, BF16, room=20)
    four, _ = make([30, 40], 2, 128, 16, BF16, "mxfp4", room=20)
    rotary = Rotary(128)
    q, k = rows_like(cache, 6, 4).cuda(), rows_like(cache, 6, 2).cuda()
    e = ends([2, 4])
    for c in (cache, four):
        before = c.lengths.tolist()
        for call in (lambda: c.attend_prompt(q), lambda: c.attend_prompt(q[:, :3].contiguous(), e),
                     lambda: c.attend_prompt(q.float(), e), lambda: c.attend_prompt(q[:, ::2], e),
                     lambda: c.attend_prompt(q.cpu(), e), lambda: c.attend_prompt(q, e.long()),
                     lambda: c.attend_prompt(q, e.cpu()), lambda: c.attend_prompt(q, e, scale=math.inf),
                     lambda: c.attend_prompt(q, e, lse=torch.empty(6, 2, device="cuda")),
                     lambda: c.append(k, k, e, q=q), lambda: c.append(k, k, e, rotary=Rotary(64)),
                     lambda: c.append(k, k, e, rotary=Rotary(128, device="cpu")), lambda: c.append(k, k, e, rotary=1),
                     lambda: c.append(k, k, e, q=q[:5], rotary=rotary), lambda: c.append(k, k, e, q=q.half(), rotary=rotary),
                     lambda: c.append(k, k, e, q=q.transpose(1, 2), rotary=rotary), lambda: c.read(e),
                     lambda: c.read(rows=5), lambda: c.read(e.long(), rows=6), lambda: c.read(e, rows=-1),
                     lambda: c.prompt(q, k[:5], k[:5], e), lambda: c.prompt(q.half(), k, k, e),
                     lambda: c(q[:2], k[:2], k[:2], rotary=Rotary(64))):
            with pytest.raises(ValueError):
                call()
        assert c.lengths.tolist() == before
    with pytest.raises(NotImplementedError):
        PagedCache(1, 1, 1, dtype=FP32, storage="mxfp4")
    with pytest.raises(ValueError):
        PagedCache(1, 1, 1, storage="int4")
    with pytest.raises(ValueError):
        cache.append(k, k, e, into=four)
    pages = dict(dtype=BF16, k_scales=four.k_scales, v_scales=four.v_scales)
    PagedCache.from_tensors(four.k, four.v, four.table, four.lengths, **pages)
    for bad in (dict(k_scales=None), dict(v_scales=four.v_scales[:, :, :, :2]), dict(v_scales=four.v_scales.int()),
                dict(k_scales=four.k_scales.transpose(0, 1).contiguous().transpose(0, 1)), dict(k_scales=four.k_scales.cpu())):
        with pytest.raises(ValueError):
            PagedCache.from_tensors(four.k, four.v, four.table, four.lengths, **{**pages, **bad})
    with pytest.raises(NotImplementedError):
        PagedCache.from_tensors(four.k, four.v, four.table, four.lengths, k_scales=four.k_scales, v_scales=four.v_scales)
    with pytest.raises(ValueError):  # another cache's scales
        other = PagedCache.from_tensors(four.k, four.v, four.table, four.lengths.clone(), dtype=BF16,
                                        k_scales=four.v_scales, v_scales=four.k_scales)
        four.append(k, k, e, into=other)


def test_nothing_to_do():
    for storage in (None, "mxfp4"):
        cache, _ = make([30, 0], 2, 128, 16, BF16, storage, room=4)
        none = torch.empty(0, 8, 128, dtype=BF16, device="cuda")
        assert cache.attend_prompt(none, ends([0, 0])).shape == (0, 8, 128)
        k, v = cache.read(ends([0, 0]), rows=0)
        assert k.shape == v.shape == (0, 2, 128)
        assert cache.append(none[:, :2], none[:, :2], ends([0, 0]), q=none, rotary=Rotary(128)).shape == (0, 8, 128)
        assert cache.lengths.tolist() == [30, 0]
        torch.cuda.synchronize()
        cache.check_errors()


# ------------------------------------------------------------------ strides and far pages

def spread(cache, host, far):
    """The cache over the same rows in pages of other strides: heads and pages exchanged,
    a gap behind each slot, the last page `far` bytes from the first."""
    def move(x, slot, align, far):
        pages, heads, page, row = x.shape
        es = x.element_size()
        slot_stride = (row * es + align + 15) // 16 * 16 // es if align >= 16 else row + align // es
        head_stride = page * slot_stride
        page_stride = max(heads * head_stride, far // es // (pages - 1) // 128 * 128)
        flat = torch.zeros((pages - 1) * page_stride + heads * head_stride, dtype=x.dtype, device="cuda")
        out = flat.as_strided(x.shape, (page_stride, head_stride, slot_stride, 1))
        out.copy_(x)
        return out
    more = {}
    if cache.storage:
        width = cache.k_scales.shape[3]
        more = dict(k_scales=move(cache.k_scales, 0, width, far // 16), v_scales=move(cache.v_scales, 0, width, far // 16),
                    dtype=cache.dtype)
    return PagedCache.from_tensors(move(cache.k, 0, 32, far), move(cache.v, 0, 32, far), cache.table,
                                   cache.lengths.clone(), **more)


@pytest.mark.parametrize("storage,dtype", [(None, BF16), (None, FP32), ("mxfp4", FP16), ("mxfp4", BF16)])
@pytest.mark.parametrize("far", [0, 9 << 30])
def test_other_strides_and_pages_gigabytes_apart(storage, dtype, far):
    lengths, new = [100, 61], [40, 33]
    cache, host = make(lengths, 2, 128, 16, dtype, storage, room=16)
    moved = spread(cache, host, far)
    q = rows_like(cache, 73, 8).cuda()
    e = ends(new)
    assert torch.equal(moved.attend_prompt(q, e), cache.attend_prompt(q, e))
    one = q[:2].contiguous()
    got = moved.attend(one).cpu()
    for b, ((want, _, _), (tol, _, _)) in enumerate(paged.attend(one.cpu(), host["k"], host["v"], host["table"], lengths)):
        assert ((got[b].double() - want).abs() <= tol).all()
    rotary = Rotary(128)
    k, v = (rows_like(cache, 9, 2, s).cuda() for s in (4, 5))
    for c in (cache, moved):
        c.append(k, v, ends([5, 4]), rotary=rotary)
    for a, b in zip(cache.read(ends([50, 50]), rows=100), moved.read(ends([50, 50]), rows=100)):
        assert torch.equal(a, b)
    moved.check_errors()


# ------------------------------------------------------------------ cuts

@pytest.mark.parametrize("storage", [None, "mxfp4"])
def test_long_histories_in_chunks(storage):
    # one sequence is cut into chunks beside others that are not, a longer table than any
    lengths, new = [9000, 130, 0, 2500, 64], [40, 100, 0, 1, 64]
    cache, host = make(lengths, 2, 64, 64, BF16, storage, room=[3000, 0, 0, 0, 0])
    q = rows_like(cache, sum(new), 6)
    lse = torch.empty(sum(new), 6, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends(new), lse=lse)
    check_prompt(q, host, lengths, new, out, lse)
    again = cache.attend_prompt(q.cuda(), ends(new))
    assert torch.equal(out, again)
    cache.check_errors()


def test_special_values_in_cut_sequences():
    n, m = 6000, 30

    def edit(k, v, table):
        v[table[0, 100 // 64], :, 100 % 64, 5] = math.inf   # in the first chunk: all rows see it
        v[table[0, 5990 // 64], :, 5990 % 64, 6] = -math.inf  # in the last: rows 20 ..

    cache, _ = make([n], 1, 64, 64, FP16, edit=edit)
    out = cache.attend_prompt(rows_like(cache, m, 4).cuda(), ends([m])).cpu()
    assert (out[:, :, 5] == math.inf).all()
    assert torch.isfinite(out[:20, :, 6]).all() and (out[20:, :, 6] == -math.inf).all()
    out[:, :, 5:7] = 0
    assert torch.isfinite(out).all()


def test_more_sequences_than_lanes_some_cut():
    lengths = [700 if b % 50 == 3 else 1 + b % 40 for b in range(150)]
    new = [1 + b % 3 if b % 7 else 0 for b in range(150)]
    new = [min(m, n) for m, n in zip(new, lengths)]
    cache, host = make(lengths, 1, 64, 16, FP32)
    q = rows_like(cache, sum(new), 2)
    out = cache.attend_prompt(q.cuda(), ends(new))
    check_prompt(q, host, lengths, new, out)


# ------------------------------------------------------------------ streams and graphs

def test_another_stream():
    cache, host = make([300, 200], 2, 128, 16, BF16)
    q = rows_like(cache, 150, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = cache.attend_prompt(q.cuda(), ends([100, 50]))
        k, v = cache.read(ends([100, 50]), rows=150)
    stream.synchronize()
    check_prompt(q, host, [300, 200], [100, 50], out)
    assert torch.equal(k[:100].cpu(), paged.rows(host["k"], host["table"][0], 300)[:, 200:].transpose(0, 1))


@pytest.mark.parametrize("storage", [None, "mxfp4"])
def test_graphs_of_two_sizes_and_eager_calls_between(storage):
    rotary = Rotary(128)
    cache, host = make([2000, 300], 2, 128, 16, BF16, storage, room=200)
    new = {48: [30, 18], 100: [1, 99]}
    x = {n: [rows_like(cache, n, h, s + n).cuda() for h, s in ((8, 1), (2, 2), (2, 3))] for n in new}
    e = {n: ends(m) for n, m in new.items()}
    forks = {n: cache.fork() for n in new}

    def run(n):
        out = cache.prompt(*x[n], e[n], rotary=rotary, into=forks[n])
        return (out, *forks[n].read(e[n], rows=n), forks[n].lengths)

    want = {n: [t.clone() for t in run(n)] for n in new}
    torch.cuda.synchronize()
    graphs = {}
    for n in new:
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n]):
            got = run(n)
        graphs[n].results = got
    big = rows_like(cache, 400, 8).cuda()  # (a larger workspace, beside those that the graphs use)
    for _ in range(3):
        for n in new:
            for t in graphs[n].results:
                t.zero_()
            graphs[n].replay()
            cache.attend_prompt(big, ends([200, 200]))
            torch.cuda.synchronize()
            for a, b in zip(graphs[n].results, want[n]):
                assert torch.equal(a, b)
    cache.check_errors()


def test_no_workspace_inside_a_capture():
    cache, _ = make([5000], 1, 64, 64, BF16)
    q = rows_like(cache, 40, 2).cuda()
    e = ends([40])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first call of a kind"):
        with torch.cuda.graph(graph):
            cache.attend_prompt(q, e)
    torch.cuda.synchronize()
    cache.attend_prompt(q, e)


# ------------------------------------------------------------------ all together

@pytest.mark.parametrize("storage", [None, "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_served_conversation(storage, dtype):
    """Prompts in chunks, steps, a cut, a turn behind it: every output against the
    definition over what the cache then holds, whose rows are the turned ones."""
    rotary = Rotary(64, base=5e5, rotary_dim=32, interleaved=True)
    cache = PagedCache(3, 60, 20, page_size=16, kv_heads=2, head_dim=64, dtype=dtype, storage=storage, scored=True)
    gen = torch.Generator().manual_seed(7)
    held = [[[], []] for _ in range(3)]  # per sequence the turned k and v rows, as held
    seen = [0, 0, 0]
    lengths = [0, 0, 0]

    def tokens(new):
        qkv = torch.randn(sum(new), 6 + 2 + 2, 64, generator=gen).to(dtype)
        return qkv, qkv.cuda()

    def held_now():
        k, v = cache.read(ends(lengths), rows=sum(lengths))
        return [x.cpu().split(lengths) for x in (k, v)]

    def check(q, new, out):
        k, v = held_now()
        at = 0
        for b, m in enumerate(new):
            if m:
                position = seen[b] - m + torch.arange(m)
                # (the queries' turn is checked by itself elsewhere: here the device's)
                (want, _), (bound, _) = paged.prompt(q[at:at + m], k[b].transpose(0, 1), v[b].transpose(0, 1), m)
                assert ((out[at:at + m].cpu().double() - want).abs() <= bound).all(), (b, position)
            at += m

    def turned(qkv, new):
        """The queries as the append turns them, from a cache of its own."""
        other = PagedCache(3, 3 * 13, 13, page_size=16, kv_heads=2, head_dim=64, dtype=dtype, scored=True)
        other.reserve(max(new))
        other.seen.copy_(torch.tensor([s - m for s, m in zip(seen, new)]))
        q = other.append(qkv[:, 6:8], qkv[:, 8:], ends(new), q=qkv[:, :6], rotary=rotary)
        return q.cpu()

    def prompt(new):
        _, on = tokens(new)
        for b, m in enumerate(new):
            lengths[b] += m
            seen[b] += m
        cache.reserve(lengths)
        out = cache.prompt(on[:, :6], on[:, 6:8], on[:, 8:], ends(new), rotary=rotary)
        check(turned(on, new), new, out)

    def step():
        _, on = tokens([1, 1, 1])
        for b in range(3):
            lengths[b] += 1
            seen[b] += 1
        cache.reserve(lengths)
        out = cache(on[:, :6], on[:, 6:8], on[:, 8:], rotary=rotary, accumulate=True)
        check(turned(on, [1, 1, 1]), [1, 1, 1], out)

    prompt([100, 7, 33])
    prompt([1, 150, 0])
    for _ in range(3):
        step()
    cache.evict(64, recent=16, sinks=2)
    lengths[:] = [min(n, 64) for n in lengths]
    assert cache.lengths.tolist() == lengths and cache.seen.tolist() == seen
    step()
    prompt([40, 3, 90])
    step()
    assert cache.lengths.tolist() == lengths
    cache.check_errors()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_the_bounded_session_in_four_bits(dtype):
    from prismkv_amd.hf import HFNative
    from tests.test_gpu_evict_session import decode
    from tests.test_gpu_hf import tiny_qwen3
    model = tiny_qwen3(1).to(dtype)
    with pytest.raises(ValueError):
        HFNative(model, {}, mode="evict", cache_storage="int4")
    session = HFNative(model, {}, mode="evict", cache_budget=96, cache_recent=16, cache_sinks=4, evict_every=8, observe=24,
                       cache_storage="mxfp4")
    forward, steps = session.forward, []

    def keep(module, q, k, v, mask, **kw):
        out = forward(module, q, k, v, mask, **kw)
        if q.shape[-2] == 1:
            op = session.ops[0]
            assert op.cache.storage == "mxfp4"
            rows = op.cache.read(torch.tensor([0, op.held], dtype=torch.int32, device="cuda"), rows=op.held)
            (want, _), (bound, _) = paged.prompt(q[0, :, 0][None].cpu(), *(x.cpu().transpose(0, 1) for x in rows), 1)
            steps.append(((out[0].reshape(1, -1, q.shape[-1]).cpu().double() - want).abs() <= bound).all())
            # the newest row is the held form of the token's
            codes, scales = paged.hold(k[0, :, -1].cpu())
            assert torch.equal(rows[0][-1].cpu().double(), paged.value(codes, scales))
        return out

    session.forward = keep
    ids = torch.randint(0, 256, (1, 240), generator=torch.Generator().manual_seed(2)).cuda()
    decode(model, session, ids, 200)
    session.close()
    assert len(steps) == 40 and all(steps)
