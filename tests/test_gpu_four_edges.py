"""Attention over pages in 4 bits where it has branches of its own: scales of any sign,
blocks that held an infinity or NaN in slots that count, scores past 2^22."""
import math

import pytest
import torch

from oracle import paged
from tests.serving_util import BF16, FP16, FP32, check_prompt, ends, make, rows_like

pytestmark = pytest.mark.gpu

DIMS = [64, 128, 256]
PAGES = [16, 24]  # looked up by the block of 16 slots, and by the row


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.7, 40.0])
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scales(dtype, dim, page, scale):
    lengths = [90, 0, 700]
    cache, host = make(lengths, 2, dim, page, dtype, "mxfp4", scored=True)
    before = host["scores"].clone()
    q = rows_like(cache, 3, 8)
    lse = torch.empty(3, 8, device="cuda")
    out = cache.attend(q.cuda(), scale=scale, accumulate=True, lse=lse).cpu()
    weights = cache.scores.cpu() - before
    for b, ((want, w, l), (tol, w_tol, l_tol)) in enumerate(
            paged.attend(q, host["k"], host["v"], host["table"], lengths, scale=scale)):
        assert ((out[b].double() - want).abs() <= tol).all(), b
        n = lengths[b]
        # (a sum with a score of up to 1, and the difference taken here)
        assert ((weights[b, :, :n].double() - w).abs() <= w_tol + (1 + w) * 2.0 ** -23).all(), b
        assert torch.equal(cache.scores[b, :, n:].cpu(), before[b, :, n:])
        assert (((lse[b].cpu().double() - l).abs() <= l_tol) | (torch.isinf(l) & (lse[b].cpu() == l))).all(), b
    new = [50, 0, 9]
    q = rows_like(cache, 59, 8)
    lse = torch.empty(59, 8, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends(new), scale=scale, lse=lse)
    check_prompt(q, host, lengths, new, out, lse, scale=scale)
    cache.check_errors()


SPECIAL = ((40, math.inf), (41, math.nan), (97, -math.inf), (168, math.inf))


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_special_blocks_reach_the_rows_that_see_them_only(dtype, dim, page):
    """A block of 32 dims that held an infinity or NaN is NaN: of V in its dims alone, of K
    in all.  Whatever does not meet one is what it is without."""
    n, m = 170, 150

    def edit_v(k, v, table):
        for i, (t, x) in enumerate(SPECIAL):
            v[table[0, t // page], :, t % page, 32 * i % dim + 3] = x

    def edit(k, v, table):
        edit_v(k, v, table)
        k[table[0, 169 // page], :, 169 % page, dim - 1] = -math.inf

    cache, _ = make([n], 2, dim, page, dtype, "mxfp4", edit=edit)
    clean, host = make([n], 2, dim, page, dtype, "mxfp4")
    q = rows_like(cache, m, 6)
    lse = torch.empty(m, 6, device="cuda")
    out, want = cache.attend_prompt(q.cuda(), ends([m]), lse=lse).cpu(), clean.attend_prompt(q.cuda(), ends([m])).cpu()
    check_prompt(q, host, [n], [m], want)
    _, (bound, _) = paged.prompt(q, *(paged.rows(host[x], host["table"][0], n) for x in "kv"), m)
    slot = n - m + torch.arange(m)
    seen = torch.zeros(m, dim, dtype=torch.bool)
    for i, (t, _) in enumerate(SPECIAL):
        block = 32 * i % dim
        seen[:, block:block + 32] |= (slot >= t)[:, None]
    seen[slot >= 169] = True
    seen = seen[:, None].expand_as(out)
    assert torch.isnan(out[seen]).all() and torch.isfinite(out[~seen]).all()
    assert ((out.double() - want.double()).abs() <= 2 * bound)[~seen].all()
    assert torch.isfinite(lse[:-1]).all() and torch.isnan(lse[-1]).all()
    # one token of each sequence: NaN where V's blocks are, and everywhere with K's
    cache, _ = make([n, n], 2, dim, page, dtype, "mxfp4", edit=edit_v)
    clean, host = make([n, n], 2, dim, page, dtype, "mxfp4")
    q = rows_like(cache, 2, 6)
    out = cache.attend(q.cuda()).cpu()
    (want, *_), (tol, *_) = paged.attend(q, host["k"], host["v"], host["table"], [n, n])[0]
    seen = torch.zeros(dim, dtype=torch.bool)
    for i in range(len(SPECIAL)):
        seen[32 * i % dim:32 * i % dim + 32] = True
    assert torch.isnan(out[0, :, seen]).all()
    assert ((out[0].double() - want).abs() <= tol)[:, ~seen].all()
    assert torch.isfinite(out[1]).all()
    cache, _ = make([n], 2, dim, page, dtype, "mxfp4", edit=edit)
    assert torch.isnan(cache.attend(q[:1].cuda())).all()


@pytest.mark.parametrize("storage", [None, "mxfp4"])
@pytest.mark.parametrize("n", [100, 1100])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_large_scores(dtype, dim, n, storage):
    """The largest score's weight is 1 whatever its size: its values come back."""
    if storage and dtype == FP32:
        pytest.skip("no fp32 rows in 4 bits")
    m = 20
    cache, host = make([n], 1, dim, 16, dtype, storage)
    q = rows_like(cache, m, 2)
    k, v = (paged.rows(host[x], host["table"][0], n)[0] for x in "kv")
    for scale in (1e30, -1e30, 2.0 ** 24):
        out = cache.attend_prompt(q.cuda(), ends([m]), scale=scale).cpu()
        one = cache.attend(q[-1:].cuda(), scale=scale).cpu()
        for i in range(m):
            for h in range(2):
                s = k[:n - m + 1 + i].double() @ q[i, h].double() * math.copysign(1, scale)
                best, second = s.topk(2).values
                assert best - second > 2.0 ** -17 * (k.double().abs() @ q[i, h].double().abs()).max()  # (of these inputs)
                assert torch.equal(out[i, h].double(), v[s.argmax()].double()), (i, h, scale)
                if i == m - 1:
                    assert torch.equal(one[0, h].double(), v[s.argmax()].double()), (h, scale)
    cache.check_errors()
