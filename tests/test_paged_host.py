"""CPU checks of the paged cache's C entries (refusals before anything is
enqueued) and of its 64-bit definition (oracle/paged.py)."""
import ctypes
import random

import pytest
import torch

from oracle import paged
from tests.test_abi import BIG, call_raw, lib  # noqa: F401

GOOD = dict(k=16, v=16, table=16, lengths=16, seen=16, scores=16, positions=16, err=16, pages=40,
            page_stride=8 * 16 * 128, head_stride=16 * 128, slot_stride=128, sequences=3, kv_heads=8, head_dim=128,
            page_size=16, max_pages=10, dtype=0)


def desc(**changed):
    from prismkv_amd._lib import PagedCacheDesc
    return ctypes.byref(PagedCacheDesc(**{**GOOD, **changed}))


def attend(lib, cache=None, into=None, q=16, lse=0, work=16, out=16, group=4, flags=1, scale=0.1, nbytes=BIG):
    return call_raw(lib, "prismkv_paged_attend", cache or desc(), into or cache or desc(), q, lse, work, out, group, flags,
                    scale, nbytes)


def append(lib, cache=None, into=None, k=16, v=16, offsets=16, rows=5, strides=(1024, 128, 1024, 128)):
    return call_raw(lib, "prismkv_paged_append", cache or desc(), into or cache or desc(), k, v, offsets, rows, *strides)


def evict(lib, cache=None, into=None, keeps=0, work=16, keep=5, recent=0, sinks=0, nbytes=BIG):
    return call_raw(lib, "prismkv_paged_evict", cache or desc(), into or cache or desc(), keeps, work, keep, recent, sinks,
                    nbytes)


SHAPE = ("sequences", "kv_heads", "head_dim", "page_size", "max_pages")
STRIDES = ("pages", "page_stride", "head_stride", "slot_stride")
BAD_SHAPES = [(0, 8, 128, 16, 10), (65536, 8, 128, 16, 10), (3, 0, 128, 16, 10), (3, 8, 96, 16, 10), (3, 8, 128, 0, 10),
              (3, 8, 128, 16, 0), (3, 8, 128, 1 << 20, 1 << 11), (3, 8, 128, 1 << 30, 1), (2, 8, 128, 1 << 30, 2)]
BAD_STRIDES = [(0, 16384, 2048, 128), (40, 8 * 16 * 128 + 1, 2048, 128), (40, 16384, 2048 + 4, 128),
               (40, 16384, 2048, 120), (40, -16384, 2048, 128), (1 << 31, 16384, 2048, 128), (40, 1 << 35, 2048, 128),
               (40, 1 << 62, 2048, 128), (40, 16384, 2048, 1 << 60)]


@pytest.mark.parametrize("call", [attend, append, evict])
def test_refused_caches(lib, call):  # noqa: F811
    for shape in BAD_SHAPES:
        assert call(lib, desc(**dict(zip(SHAPE, shape)))) == -1, shape
    for strides in BAD_STRIDES:
        assert call(lib, desc(**dict(zip(STRIDES, strides)))) == -1, strides
    for dtype in (-1, 3):
        assert call(lib, desc(dtype=dtype)) == -2
    for name in ("k", "v", "table", "lengths", "err"):
        assert call(lib, desc(**{name: 0})) == -1, name
    for name in ("seen", "scores", "positions"):  # all of a scored cache, or none
        assert call(lib, desc(**{name: 0})) == -1, name
    for name in ("k", "v"):
        assert call(lib, desc(**{name: 24})) == -1, name
    for name in ("table", "lengths", "seen", "scores", "positions", "err"):
        assert call(lib, desc(**{name: 18})) == -1, name
    # results go to a cache over the same pages and table
    for name in ("k", "v", "table", *STRIDES, *SHAPE, "dtype"):
        other = {"dtype": 1, "head_dim": 64, "slot_stride": 256, "head_stride": 4096}.get(name, 2 * GOOD[name])
        assert call(lib, desc(), desc(**{name: other})) == -1, name
    assert call(lib, desc(), desc(seen=0, scores=0, positions=0)) == -1
    name = "prismkv_paged_" + call.__name__
    assert call_raw(lib, name, *[0] * (len(getattr(lib.cdll, name).argtypes) - 1)) == -1  # no cache


def test_refused_arguments(lib):  # noqa: F811
    plain = desc(seen=0, scores=0, positions=0)
    assert attend(lib, plain, flags=1) == -1 and evict(lib, plain) == -1  # not scored
    for bad in (dict(q=0), dict(q=24), dict(work=0), dict(work=24), dict(out=0), dict(out=18), dict(lse=18),
                dict(group=0), dict(group=1025), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attend(lib, **bad) == -1, bad
    assert attend(lib, flags=4) == -2
    for bad in (dict(k=0), dict(v=0), dict(k=24), dict(offsets=18), dict(rows=-1), dict(rows=1 << 31),
                dict(offsets=0, rows=4)):  # (one row per sequence without offsets)
        assert append(lib, **bad) == -1, bad
    for i in range(4):
        for bad in (1028, 1 << 41, -(1 << 41), 1 << 62):
            assert append(lib, strides=[bad if j == i else 1024 for j in range(4)]) == -1
    for bad in (dict(keep=-1), dict(recent=-1), dict(sinks=-1), dict(work=0), dict(work=24), dict(keeps=18, keep=0),
                dict(keeps=16, keep=5)):  # (a budget for all and one for each)
        assert evict(lib, **bad) == -1, bad


def test_workspace_sizes(lib):  # noqa: F811
    need = lib.query("prismkv_paged_attend_work_bytes", 3, 8, 4, 128, 160, 1, 0)
    # the weighed logits of every query head and slot, at least
    assert need >= 3 * 32 * 160 * 4 + lib.query("prismkv_paged_attend_work_bytes", 3, 8, 4, 128, 160, 0, 0)
    assert attend(lib, nbytes=need - 1) == -1
    assert attend(lib, nbytes=need) not in (0, -1, -2)  # past every host check, refused by the runtime (no device)
    for bad in ((0, 8, 4, 128, 160, 0, 0), (3, 0, 4, 128, 160, 0, 0), (3, 8, 0, 128, 160, 0, 0), (3, 8, 4, 128, 0, 0, 0),
                (3, 8, 4, 128, 160, 0, 3)):
        assert lib.query("prismkv_paged_attend_work_bytes", *bad) == 0
    need = lib.query("prismkv_paged_evict_work_bytes", 3, 8, 160)
    assert need >= 24 * 160 * 4
    assert evict(lib, nbytes=need - 1) == -1 and evict(lib, nbytes=need) not in (0, -1, -2)
    assert lib.query("prismkv_paged_evict_work_bytes", 0, 8, 160) == 0
    assert append(lib) not in (0, -1, -2)


def test_host_only_tensors_are_refused():
    from prismkv_amd import PagedCache
    k = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        PagedCache.from_tensors(k, k, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="device tensor"):
        PagedCache(1, 4, 4, device="cpu")
    with pytest.raises(ValueError, match="sequences must be positive"):
        PagedCache(0, 4, 4)


def test_too_large_caches_are_refused():
    """By the constructor, before anything is allocated: 2^25 pages of 16 x 128 bf16 rows."""
    from prismkv_amd import PagedCache
    with pytest.raises(NotImplementedError, match="64 GiB"):
        PagedCache(1, 1 << 25, 1 << 10, page_size=16, kv_heads=1, device="cuda:0")
    with pytest.raises(NotImplementedError, match="slots"):
        PagedCache(1, 4, 1 << 27, page_size=16, kv_heads=1, device="cuda:0")


def test_definition_of_attend():
    """The oracle's rows, weights and log-sum against softmax on gathered rows."""
    torch.manual_seed(0)
    k, v = torch.randn(6, 2, 4, 64), torch.randn(6, 2, 4, 64)
    table = torch.tensor([[3, 5, 0], [1, -1, -1], [-1, -1, -1]], dtype=torch.int32)
    q = torch.randn(3, 4, 64)
    got = paged.attend(q, k, v, table, [9, 4, 0])
    flat = [torch.cat([x[p] for p in (3, 5, 0)], dim=1)[:, :9].double() for x in (k, v)]
    for head in range(4):
        s = flat[0][head // 2] @ q[0, head].double() / 8
        p = torch.softmax(s, 0)
        assert torch.allclose(got[0][0][0][head], p @ flat[1][head // 2], atol=1e-12)
        assert abs(got[0][0][2][head] - torch.logsumexp(s, 0)) < 1e-12
    assert torch.allclose(got[0][0][1].sum(1), torch.full((2,), 2.0, dtype=torch.float64))
    assert not got[2][0][0].any() and got[2][0][2].isinf().all()


def test_definition_of_evict():
    rng = random.Random(0)
    for _ in range(50):
        n, keep = rng.randint(0, 30), rng.randint(0, 30)
        scores = [float(rng.choice([0, 1, 2, 3])) for _ in range(n)]
        positions = rng.sample(range(40), n)
        moves = paged.evict(scores, positions, n, keep, 40, recent=rng.randint(0, 5), sinks=2)
        m = min(n, keep)
        assert all(d < m <= s for s, d in moves) and moves == sorted(moves)
        assert [d for _, d in moves] == sorted(d for _, d in moves)
        stay = (set(range(m)) - {d for _, d in moves}) | {s for s, _ in moves}
        left = set(range(n)) - stay
        assert len(stay) == m
        if not any(positions[t] >= 35 or positions[t] < 2 for t in range(n)) and left and stay:
            assert min(scores[t] for t in stay) >= max(scores[t] for t in left)


def test_evict_session_on_host():
    """Mode "evict" without encoders: its checks, and the prefill through the model's own attention."""
    from prismkv_amd.hf import DecodeGraph, HFNative
    from tests.test_hf_host import encoders, tiny_qwen3
    model = tiny_qwen3()
    for bad in (dict(cache_budget=0), dict(evict_every=0), dict(cache_recent=-1), dict(observe=-1),
                dict(cache_budget=10, cache_recent=8, cache_sinks=3)):
        with pytest.raises(ValueError, match="cache budget"):
            HFNative(model, {}, mode="evict", **bad)
    with pytest.raises(ValueError, match="sparse, all_read or evict"):
        HFNative(model, encoders(1), mode="dense")
    with pytest.raises(ValueError, match="missing"):
        HFNative(model, {}, mode="all_read")
    ids = torch.randint(0, 128, (1, 12))
    with torch.no_grad():
        dense = model(ids).logits
    session = HFNative(model, {}, mode="evict", observe=5)
    with pytest.raises(NotImplementedError, match="sparse mode"):
        DecodeGraph(session, None)
    with torch.no_grad():
        assert torch.equal(model(ids).logits, dense)
    assert session._observed[0].shape == (32, 5, 128)
    # chunks: the last queries of the whole prompt
    from transformers import DynamicCache
    whole = session._observed[0]
    cache = DynamicCache(config=model.config)
    session.begin_request()
    with torch.no_grad(), session.prefill():
        for lo, hi in ((0, 8), (8, 11), (11, 12)):
            model(ids[:, lo:hi], past_key_values=cache, use_cache=True)
    assert torch.allclose(session._observed[0], whole, atol=1e-5)
    session.close()
    assert model.config._attn_implementation == "sdpa" and not session._observed


@pytest.fixture
def words(monkeypatch):
    """_ErrorWord without a device: (made words' class, device, the synchronisations so far)."""
    import contextlib
    from prismkv_amd import paged as module
    zeros, synced = torch.zeros, []
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: synced.append(d))

    class Lib:
        def query(self, name, address):
            return address

    device = torch.device("cuda", 97)  # (no other test's)
    return lambda: module._ErrorWord(Lib(), device), synced


def test_error_words_are_used_again_only_behind_a_synchronisation(words):
    """A launch still queued when its cache goes may write the word: it is another
    cache's only after everything enqueued before has run."""
    make, synced = words
    retired = {}  # address -> synchronisations when it was given back
    held = []
    for i in range(3000):
        word = make()
        assert word.word.value == 0 and word.address not in [w.address for w in held]
        if word.address in retired:
            assert len(synced) > retired[word.address], i
        word.word.value = 4  # (a late report)
        held.append(word)
        if len(held) > 5:
            gone = held.pop(0)
            retired[gone.address] = len(synced)
            del gone
    assert len(set(retired)) < 1000  # (they are used again)
    assert len(synced) < 30


def test_error_words_of_several_threads(words):
    import threading
    make, _ = words
    problems = []

    def run():
        try:
            for _ in range(2000):
                word = make()
                word.word.value = token = threading.get_ident() % 2 ** 30 + 1
                if make().address == word.address or word.word.value != token:
                    problems.append("a word of two caches")
        except Exception as e:  # noqa: BLE001
            problems.append(repr(e))

    threads = [threading.Thread(target=run) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the addresses are made up: host checks only")
def test_overlapping_results_are_refused(lib):  # noqa: F811
    """Buffers of the second cache that are not all the first's lie apart from all of the first's."""
    size = dict(lengths=4 * 3, seen=4 * 3, scores=4 * 3 * 8 * 160, positions=4 * 3 * 8 * 160)
    own = dict(lengths=1 << 20, seen=2 << 20, scores=3 << 20, positions=4 << 20)
    apart = {name: at + (8 << 20) for name, at in own.items()}
    for call in (attend, append, evict):
        assert call(lib, desc(**own), desc(**own)) not in (0, -1, -2)  # past every host check (no device)
        assert call(lib, desc(**own), desc(**apart)) not in (0, -1, -2)
        for name in own:
            assert call(lib, desc(**own), desc(**{**apart, name: own[name]})) == -1, name
            for other in own:
                for at in (own[other] + size[other] - 4, own[other] - size[name] + 4):
                    assert call(lib, desc(**own), desc(**{**apart, name: at})) == -1, (name, other)
                for at in (own[other] + size[other], own[other] - size[name]):  # next to each other
                    assert call(lib, desc(**own), desc(**{**apart, name: at})) not in (0, -1, -2), (name, other)
    plain = dict(seen=0, scores=0, positions=0)
    for at, ok in ((1 << 20, True), ((1 << 20) + 4, False), ((1 << 20) + 12, True)):
        code = attend(lib, desc(lengths=1 << 20, **plain), desc(lengths=at, **plain), flags=0)
        assert (code not in (0, -1, -2)) if ok else code == -1


def test_scales_that_32_bits_do_not_hold_are_refused(lib):  # noqa: F811
    for scale in (3e38, -3e38, 1e300):  # (times log2(e))
        assert attend(lib, scale=scale) == -1


def test_too_many_quanta_have_no_workspace(lib):  # noqa: F811
    """2^30 slots of 1024 query heads on a KV head are 2^31 quanta of 32 slots; of 512 heads half of it."""
    for group, fits in ((1024, False), (512, True)):
        need = lib.query("prismkv_paged_attend_work_bytes", 1, 1, group, 64, 1 << 30, 0, 0)
        assert (need > 0) == fits
    wide = dict(sequences=1, kv_heads=1, page_size=1 << 20, max_pages=1 << 10, pages=1, page_stride=128 << 20,
                head_stride=128 << 20)
    assert attend(lib, desc(**wide), group=1024, flags=0) == -1
