"""CPU checks of the paged cache's C entries (refusals before anything is
enqueued) and of its 64-bit definition (oracle/paged.py)."""
import random

import pytest
import torch

from oracle import paged
from tests.test_abi import BIG, call_raw, lib  # noqa: F401

# sequences, kv_heads, head_dim, page_size, max_pages | pages, page_stride, head_stride, slot_stride, dtype
SHAPE, STRIDES = (3, 8, 128, 16, 10), (40, 8 * 16 * 128, 16 * 128, 128)


def attend(lib, pointers=(16,) * 11, shape=SHAPE, group=4, strides=STRIDES, scale=0.1, dtype=0, work=BIG):
    b, h, d, ps, mp = shape
    return call_raw(lib, "prismkv_paged_attend", *pointers, b, h, group, d, ps, mp, *strides, scale, dtype, work)


def append(lib, pointers=(16,) * 15, rows=5, row_strides=(1024, 128, 1024, 128), shape=SHAPE, strides=STRIDES, dtype=0):
    return call_raw(lib, "prismkv_paged_append", *pointers, rows, *row_strides, *shape, *strides, dtype)


def evict(lib, pointers=(16,) * 11 + (0, 16, 16), keep=5, recent=0, sinks=0, shape=SHAPE, strides=STRIDES, dtype=0,
          work=BIG):
    return call_raw(lib, "prismkv_paged_evict", *pointers, keep, recent, sinks, *shape, *strides, dtype, work)


BAD_SHAPES = [(0, 8, 128, 16, 10), (65536, 8, 128, 16, 10), (3, 0, 128, 16, 10), (3, 8, 96, 16, 10), (3, 8, 128, 0, 10),
              (3, 8, 128, 16, 0), (3, 8, 128, 1 << 20, 1 << 11), (3, 8, 128, 1 << 30, 1), (2, 8, 128, 1 << 30, 2)]
BAD_STRIDES = [(0, *STRIDES[1:]), (40, 8 * 16 * 128 + 1, 2048, 128), (40, 16384, 2048 + 4, 128), (40, 16384, 2048, 120),
               (40, -16384, 2048, 128), (1 << 31, 16384, 2048, 128), (40, 1 << 35, 2048, 128), (40, 1 << 62, 2048, 128),
               (40, 16384, 2048, 1 << 60)]


@pytest.mark.parametrize("call", [attend, append, evict])
def test_refused_sizes(lib, call):  # noqa: F811
    for shape in BAD_SHAPES:
        assert call(lib, shape=shape) == -1, shape
    for strides in BAD_STRIDES:
        assert call(lib, strides=strides) == -1, strides
    for dtype in (-1, 3):
        assert call(lib, dtype=dtype) == -2


def _without(pointers, i, value=0):
    return tuple(value if j == i else x for j, x in enumerate(pointers))


def test_refused_pointers(lib):  # noqa: F811
    good = (16,) * 11
    for i in (0, 1, 2, 3, 4, 5, 6, 8, 9, 10):  # scores and their destination come together
        assert attend(lib, _without(good, i)) == -1, i
    for i, off in ((0, 24), (1, 24), (2, 24), (3, 18), (4, 18), (7, 18), (8, 24), (9, 20)):
        assert attend(lib, _without(good, i, off)) == -1, i
    good = (16,) * 15
    for i in (0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11, 13, 14):  # (0: no offsets; 12: not scored)
        assert append(lib, _without(good, i)) == -1, i
    for i, off in ((0, 24), (2, 24), (5, 18), (12, 18), (14, 20)):
        assert append(lib, _without(good, i, off)) == -1, i
    good = (16,) * 11 + (0, 16, 16)
    for i in range(14):
        if i != 11:
            assert evict(lib, _without(good, i)) == -1, i
    assert evict(lib, _without(good, 12, 24)) == -1 and evict(lib, _without(good, 13, 20)) == -1


def test_refused_arguments(lib):  # noqa: F811
    assert attend(lib, group=0) == -1 and attend(lib, group=1025) == -1
    assert attend(lib, scale=float("nan")) == -1
    assert append(lib, rows=-1) == -1 and append(lib, rows=1 << 31) == -1
    no_offsets = _without((16,) * 15, 5)
    assert append(lib, no_offsets, rows=4) == -1  # one row per sequence without offsets
    for i in range(4):
        assert append(lib, row_strides=_without((1024, 128, 1024, 128), i, 1028)) == -1
    for bad in (dict(keep=-1), dict(recent=-1), dict(sinks=-1)):
        assert evict(lib, **bad) == -1
    assert evict(lib, (16,) * 14, keep=5) == -1  # a budget for all and one for each


def test_workspace_sizes(lib):  # noqa: F811
    need = lib.query("prismkv_paged_attend_work_bytes", 3, 8, 4, 128, 160, 1, 0)
    # the weighed logits of every query head and slot, at least
    assert need >= 3 * 32 * 160 * 4 + lib.query("prismkv_paged_attend_work_bytes", 3, 8, 4, 128, 160, 0, 0)
    assert attend(lib, work=need - 1) == -1
    assert attend(lib, work=need) not in (0, -1, -2)  # past every host check, refused by the runtime (no device)
    for bad in ((0, 8, 4, 128, 160, 0, 0), (3, 0, 4, 128, 160, 0, 0), (3, 8, 0, 128, 160, 0, 0), (3, 8, 4, 128, 0, 0, 0),
                (3, 8, 4, 128, 160, 0, 3)):
        assert lib.query("prismkv_paged_attend_work_bytes", *bad) == 0
    need = lib.query("prismkv_paged_evict_work_bytes", 3, 8, 160)
    assert need >= 24 * 160 * 4
    assert evict(lib, work=need - 1) == -1 and evict(lib, work=need) not in (0, -1, -2)
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
