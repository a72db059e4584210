"""The paged cache in 4 bits on the device: what append holds and read gives back,
exactly; attention, accumulated weights and cuts over it."""
import math

import pytest
import torch

from oracle import paged
from prismkv_amd import PagedCache
from tests.serving_util import BF16, FP16, FP32, ends, make, rows_like

pytestmark = pytest.mark.gpu


def special_rows(dtype, dim):
    """Rows with every kind of block: ties, zeros, the smallest and the largest numbers, infinities, NaN."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(64, 2, dim, generator=gen) * torch.exp(4 * torch.randn(64, 2, 1, generator=gen))
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 6.9375] * 2)
    x[0, :, :32], x[1, :, :32], x[2, :, :32] = ties, ties * 2.0 ** -9, ties * 2.0 ** 10
    x[3] = 0
    x[4] = -0.0
    x[5, 0, 7], x[5, 1, 8] = math.inf, math.nan
    x[6, 0, 7] = -math.inf
    finfo = torch.finfo(dtype)
    x[7], x[8], x[9, :, 5] = finfo.max, finfo.tiny, finfo.max
    x[10] = finfo.smallest_normal / 4
    x[11] = 7.0
    x[12] = torch.nextafter(torch.tensor(7.0, dtype=dtype), torch.tensor(8.0, dtype=dtype)).float()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append_and_read(dim, dtype):
    x = special_rows(dtype, dim)
    cache = PagedCache(2, 8, 4, page_size=24, kv_heads=2, head_dim=dim, dtype=dtype, storage="mxfp4")
    cache.reserve([40, 30])
    assert cache.k.dtype == torch.uint8 and cache.k_scales.shape == (8, 2, 24, dim // 32)
    cache.append(x.cuda(), x.flip(0).contiguous().cuda(), ends([40, 24]))
    k, v = cache.read(ends([40, 24]), rows=64)
    for got, rows in ((k.cpu(), x), (v.cpu(), x.flip(0))):
        codes, scales = paged.hold(rows)
        want = paged.value(codes, scales).to(dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    # the bytes themselves
    codes, scales = paged.hold(x[:40])
    for t in (0, 1, 5, 7, 23, 24, 39):
        page = int(cache.table[0, t // 24])
        assert torch.equal(cache.k_scales[page, :, t % 24].cpu(), scales[t])
        fine = (scales[t] != 255).repeat_interleave(16, -1)
        assert torch.equal(cache.k[page, :, t % 24].cpu()[fine], paged.pack(codes)[t][fine])
    # the last ones only, and one each
    k2, v2 = cache.read(ends([3, 0]), rows=3)
    assert torch.equal(torch.nan_to_num(k2), torch.nan_to_num(k[37:40]))
    k1, _ = cache.read()
    assert torch.equal(torch.nan_to_num(k1), torch.nan_to_num(k[[39, 63]]))
    cache.check_errors()


def test_read_of_pages_as_they_are():
    for dtype in (BF16, FP16, FP32):
        for dim in (64, 128, 256):
            cache, host = make([30, 0, 75], 3, dim, 17, dtype)
            k, v = cache.read(ends([30, 0, 41]), rows=71)
            for name, got in (("k", k), ("v", v)):
                want = torch.cat([paged.rows(host[name], host["table"][0], 30).transpose(0, 1),
                                  paged.rows(host[name], host["table"][2], 75).transpose(0, 1)[34:]])
                assert torch.equal(got.cpu(), want)
            cache.check_errors()


ATTEND = [
    ([1], 1, 1, 128, 16, BF16),
    ([75], 8, 4, 128, 16, BF16),
    ([0, 1, 31, 32, 33], 2, 4, 128, 16, BF16),
    ([129, 5, 0, 640], 2, 4, 64, 16, FP16),
    ([300, 77], 2, 4, 256, 32, BF16),
    ([1000], 1, 3, 128, 17, BF16),
    ([513, 100], 2, 16, 128, 64, FP16),
    ([200, 3], 1, 17, 128, 1, BF16),
    ([150], 1, 40, 64, 24, BF16),
    ([300, 77], 1, 16, 256, 7, FP16),
    ([1000, 31], 2, 5, 128, 16, FP16),
    ([40 + 7 * b % 90 for b in range(70)], 8, 2, 64, 16, BF16),
    ([5000], 2, 4, 128, 64, BF16),
]


@pytest.mark.parametrize("lengths,kv_heads,group,dim,page,dtype", ATTEND)
def test_attend(lengths, kv_heads, group, dim, page, dtype):
    cache, host = make(lengths, kv_heads, dim, page, dtype, "mxfp4", scored=True)
    before = host["scores"].clone()
    q = rows_like(cache, len(lengths), kv_heads * group)
    lse = torch.empty(len(lengths), kv_heads * group, device="cuda")
    out = cache.attend(q.cuda(), accumulate=True, lse=lse).cpu()
    weights = cache.scores.cpu() - before
    cache.check_errors()
    for b, ((want, w, l), (tol, w_tol, l_tol)) in enumerate(paged.attend(q, host["k"], host["v"], host["table"], lengths)):
        assert ((out[b].double() - want).abs() <= tol).all(), b
        n = lengths[b]
        # (a sum with a score of up to 1, and the difference taken here)
        assert ((weights[b, :, :n].double() - w).abs() <= w_tol + (1 + w) * 2.0 ** -23).all(), b
        assert torch.equal(cache.scores[b, :, n:].cpu(), before[b, :, n:])
        assert (((lse[b].cpu().double() - l).abs() <= l_tol) | (torch.isinf(l) & (lse[b].cpu() == l))).all(), b


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_evict_moves_rows_with_their_scales(dim):
    lengths = [200, 77, 30]
    cache, host = make(lengths, 2, dim, 16, BF16, "mxfp4", scored=True)
    cache.evict(50, recent=5, sinks=2)
    after = [min(n, 50) for n in lengths]
    k, v = cache.read(ends(after), rows=sum(after))
    at = 0
    for b, n in enumerate(lengths):
        for h in range(2):
            slot = list(range(after[b]))
            for src, dst in paged.evict(host["scores"][b, h].tolist(), host["positions"][b, h].tolist(), n, 50,
                                        int(host["seen"][b]), 5, 2):
                slot[dst] = src
            for name, got in (("k", k), ("v", v)):
                want = paged.rows(host[name], host["table"][b], n)[h][slot].to(BF16)
                assert torch.equal(got[at:at + after[b], h].cpu(), want)
        at += after[b]
    cache.check_errors()


def test_steps_forks_and_a_larger_table():
    cache = PagedCache(3, 12, 4, page_size=16, kv_heads=2, head_dim=128, dtype=FP16, storage="mxfp4", scored=True)
    cache.reserve(20)
    x = rows_like(cache, 30, 2, 9).cuda()
    cache.append(x, x.flip(0).contiguous(), ends([10, 3, 17]))
    q = rows_like(cache, 3, 8).cuda()
    new = rows_like(cache, 3, 2, 11).cuda()
    fork = cache.fork()
    out = cache(q, new, new, accumulate=True, into=fork)
    assert cache.lengths.tolist() == [10, 3, 17] and fork.lengths.tolist() == [11, 4, 18]
    again = cache(q, new, new, accumulate=True)
    assert torch.equal(out, again) and torch.equal(cache.scores, fork.scores)
    big = cache.resized(30, 8)
    assert torch.equal(big.attend(q), cache.attend(q))
    held = [t.cpu() for t in cache.read(ends([11, 4, 18]), rows=33)]
    for a, b in zip(held, big.read(ends([11, 4, 18]), rows=33)):
        assert torch.equal(a, b.cpu())
    assert {"k_scales", "v_scales"} <= set(cache.buffer_bytes())
