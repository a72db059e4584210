"""Prompts over the paged cache on the device against their 64-bit definition
(oracle/paged.py), within bounds derived there."""
import math

import pytest
import torch

from oracle import paged
from prismkv_amd import PagedCache
from tests.serving_util import BF16, FP16, FP32, check_prompt, ends, make, rows_like

pytestmark = pytest.mark.gpu

CASES = [
    # slots, new rows, kv_heads, group, dim, page, dtype
    ([1], [1], 1, 1, 128, 16, BF16),
    ([75], [75], 2, 4, 128, 16, BF16),
    ([33], [5], 1, 1, 64, 16, BF16),
    ([64, 65, 63], [64, 65, 63], 2, 4, 128, 16, BF16),
    ([0, 7, 300, 128], [0, 7, 129, 0], 2, 4, 128, 64, BF16),
    ([500], [200], 1, 3, 128, 17, BF16),
    ([300, 41], [300, 40], 2, 5, 64, 24, BF16),
    ([200, 90], [130, 33], 1, 4, 256, 32, BF16),
    ([150], [150], 1, 40, 64, 1, BF16),
    ([75, 130], [75, 3], 2, 6, 64, 24, FP16),
    ([200, 1], [129, 1], 1, 4, 128, 16, FP16),
    ([150], [70], 1, 7, 256, 7, FP16),
    ([75, 130], [75, 3], 2, 4, 64, 24, FP32),
    ([200, 31], [129, 31], 1, 4, 128, 16, FP32),
    ([150, 40], [70, 2], 1, 8, 256, 32, FP32),
    ([40 + 7 * b % 90 for b in range(70)], [1 + 5 * b % 30 for b in range(70)], 1, 2, 64, 16, BF16),
    ([3000, 700], [9, 1], 2, 4, 128, 64, BF16),       # keys cut into chunks
    ([2100, 900, 64], [100, 3, 64], 1, 8, 64, 16, FP16),
    ([1500], [20], 1, 16, 256, 16, FP32),
]


@pytest.mark.parametrize("storage", [None, "mxfp4"])
@pytest.mark.parametrize("lengths,new,kv_heads,group,dim,page,dtype", CASES)
def test_prompts(lengths, new, kv_heads, group, dim, page, dtype, storage):
    if storage and dtype == FP32:
        pytest.skip("no fp32 rows in 4 bits")
    cache, host = make(lengths, kv_heads, dim, page, dtype, storage)
    q = rows_like(cache, sum(new), kv_heads * group)
    lse = torch.full((sum(new), kv_heads * group), 7.0, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends(new), lse=lse)
    torch.cuda.synchronize()
    cache.check_errors()
    assert out.dtype == dtype and out.shape == q.shape
    check_prompt(q, host, lengths, new, out, lse)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.7, 40.0])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_scales(scale, dtype):
    cache, host = make([90, 40], 1, 64, 16, dtype)
    q = rows_like(cache, 70, 2)
    lse = torch.empty(70, 2, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends([50, 20]), scale=scale, lse=lse)
    check_prompt(q, host, [90, 40], [50, 20], out, lse, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_special_values_reach_the_rows_that_see_them_only(dim, dtype):
    n, m, special = 170, 150, (40, 41, 97, 168)

    def edit(k, v, table):
        for t, x in zip(special, (math.inf, math.nan, -math.inf, math.inf)):
            v[table[0, t // 16], :, t % 16, t % dim] = x
        k[table[0, 169 // 16], :, 169 % 16, 3] = math.nan

    cache, _ = make([n], 2, dim, 16, dtype, edit=edit)
    clean, host = make([n], 2, dim, 16, dtype)
    q = rows_like(cache, m, 6)
    out, want = cache.attend_prompt(q.cuda(), ends([m])).cpu(), clean.attend_prompt(q.cuda(), ends([m])).cpu()
    check_prompt(q, host, [n], [m], want)
    (_, _), (bound, _) = paged.prompt(q, *(paged.rows(host[x], host["table"][0], n) for x in "kv"), m)
    slot = n - m + torch.arange(m)
    seen = torch.zeros(m, dim, dtype=torch.bool)
    for t in special:
        seen[:, t % dim] |= slot >= t
    seen[slot >= 169] = True
    seen = seen[:, None].expand_as(out)
    assert (torch.isfinite(out) == ~seen).all()
    assert ((out.double() - want.double()).abs() <= 2 * bound)[~seen].all()
    only = (slot >= 40) & (slot < 169)  # an infinity stays one, with its sign, where no other special value meets it
    assert (out[only][:, :, 40 % dim] == math.inf).all()
    assert torch.isnan(out[(slot >= 41) & (slot < 97)][:, :, 41 % dim]).all()


def test_scores_of_minus_infinity():
    def edit(k, v, table):
        k[table[0, :5], :, :, 0] = -math.inf
    cache, _ = make([80], 1, 64, 16, BF16, edit=edit)
    q = rows_like(cache, 60, 1)
    q[..., 0] = 1.0
    lse = torch.empty(60, 1, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends([60]), lse=lse)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_large_scores():
    # the largest score's weight is 1 whatever its size
    cache, host = make([100], 1, 64, 16, FP32)
    q = rows_like(cache, 30, 2)
    out = cache.attend_prompt(q.cuda(), ends([30]), scale=1e30).cpu()
    v = paged.rows(host["v"], host["table"][0], 100)[0]
    k = paged.rows(host["k"], host["table"][0], 100)[0]
    for i in range(30):
        for h in range(2):
            best = (k[:71 + i].double() @ q[i, h].double()).argmax()
            assert torch.equal(out[i, h], v[best])


def test_chunks_are_the_whole_prompt():
    cache, host = make([0, 0], 2, 128, 16, BF16, room=220, scored=True)
    k, v = (rows_like(cache, 360, 2, seed) for seed in (5, 6))
    q = rows_like(cache, 360, 8)
    pieces = [([100, 7], 0), ([1, 120], 107), ([99, 33], 228)]
    lengths = [0, 0]
    at = [0, 200]
    held = {name: [[], []] for name in "kvq"}
    for new, _ in pieces:
        parts = {name: [] for name in "kvq"}
        for b in (0, 1):
            for name, x in (("k", k), ("v", v), ("q", q)):
                parts[name].append(x[at[b]:at[b] + new[b]])
                held[name][b].append(parts[name][-1])
            at[b] += new[b]
            lengths[b] += new[b]
        qq, kk, vv = (torch.cat(parts[name]).cuda() for name in "qkv")
        out = cache.prompt(qq, kk, vv, ends(new))
        now = dict(k=cache.k.cpu(), v=cache.v.cpu(), table=host["table"])
        assert cache.lengths.tolist() == lengths
        check_prompt(qq.cpu(), now, lengths, new, out)
    got_k, got_v = cache.read(ends(lengths), rows=sum(lengths))
    assert torch.equal(got_k.cpu(), torch.cat(held["k"][0] + held["k"][1]))
    assert torch.equal(got_v.cpu(), torch.cat(held["v"][0] + held["v"][1]))


def test_a_prompt_of_one_row_each_is_attend():
    for storage in (None, "mxfp4"):
        cache, host = make([5, 77, 3000], 2, 128, 64, FP16, storage)
        q = rows_like(cache, 3, 8)
        out = cache.attend_prompt(q.cuda())
        check_prompt(q, host, [5, 77, 3000], [1, 1, 1], out)
        check_prompt(q, host, [5, 77, 3000], [1, 1, 1], cache.attend(q.cuda()))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths,new", [([230, 61], [90, 61]), ([1300], [10])])
def test_pages_of_every_size_give_the_same(lengths, new, dim, dtype):
    """Rows that a wave loads at once lie in one page or in several: no result tells."""
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn(sum(lengths), 2, dim, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(sum(new), 6, dim, generator=gen).to(dtype).cuda()
    v[lengths[0] - 4, 0, 5] = math.inf
    v[lengths[0] - 6, 1, dim - 1] = math.nan
    k[lengths[0] - 2, 1, 7] = math.nan
    want = None
    for page in (64, 1, 2, 5, 12, 24):
        cache = PagedCache(len(lengths), sum(-(-n // page) for n in lengths) + 3, -(-max(lengths) // page), page_size=page,
                           kv_heads=2, head_dim=dim, dtype=dtype)
        for x in (cache.k, cache.v):
            x.fill_(math.nan)
        cache.reserve(lengths)
        cache.append(k.cuda(), v.cuda(), ends(lengths))
        lse = torch.empty(sum(new), 6, device="cuda")
        got = cache.attend_prompt(q, ends(new), lse=lse), lse
        cache.check_errors()
        want = got if want is None else want
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True, msg=f"pages of {page}")
    assert want[0].isnan().any() and not want[0].isnan().all()
