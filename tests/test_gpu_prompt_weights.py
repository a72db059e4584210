"""What the rounding of a prompt's weights to 16 bits leaves of the output: a slot that
outweighs the others comes back as its values."""
import math

import pytest
import torch

from oracle import paged
from tests.serving_util import BF16, FP16, FP32, check_prompt, ends, make, rows_like

pytestmark = pytest.mark.gpu

TYPES = [(BF16, None), (FP16, None), (FP32, None), (BF16, "mxfp4"), (FP16, "mxfp4")]


def growing(k, v, table):
    """Keys that outrank those of the slots before them, as they lie in order."""
    slots = table.shape[1] * k.shape[2]
    for t in range(slots):
        k[table[0, t // k.shape[2]], :, t % k.shape[2]] *= 3 * (t + 1) / slots


@pytest.mark.parametrize("dtype,storage", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,m", [(300, 200), (1100, 9)])
def test_maxima_that_rise(n, m, dim, dtype, storage):
    cache, host = make([n], 2, dim, 16, dtype, storage, edit=growing)
    q = rows_like(cache, m, 6)
    lse = torch.empty(m, 6, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends([m]), lse=lse)
    check_prompt(q, host, [n], [m], out, lse)


@pytest.mark.parametrize("dtype,storage", TYPES)
@pytest.mark.parametrize("n", [300, 1100])
def test_a_slot_that_outweighs_the_others(n, dtype, storage):
    """Slot n - 9, tiles behind slot 5, whose score is up to 2^7 times less, and all others
    next to nothing: the output is between the two rows, held to one rounding of it, that
    of the lesser weight (1 - p), and what the other's leaves, p (v - out) of it."""
    D, best = 64, n - 9

    def edit(k, v, table):
        k[:] = 0
        k[..., 0] = -96
        for t, x in ((5, 0.0), (best, 4.0)):
            k[table[0, t // 16], :, t % 16, 0] = x

    cache, host = make([n], 1, D, 16, dtype, storage, edit=edit)
    # the row's score of the slot, in powers of 2: from 1 on, in steps that bf16 holds
    q = torch.zeros(8, 1, D, dtype=dtype)
    q[:, 0, 0] = torch.tensor([0.25, 0.40625, 0.625, 0.84375, 0.9765625, 1.21875, 1.453125, 1.796875])
    lse = torch.empty(8, 1, device="cuda")
    out = cache.attend_prompt(q.cuda(), ends([8]), scale=math.log(2), lse=lse)
    check_prompt(q, host, [n], [8], out, lse, scale=math.log(2))
    v = paged.rows(host["v"], host["table"][0], n)[0].double()
    p = 1 / (1 + 2.0 ** (-4 * q[:, 0, :1].double()))
    want = p * v[best] + (1 - p) * v[5]
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() + 1.01 * half * (1 - p) * (v[5].abs() + p * (v[best] - v[5]).abs())
    bound += 2.0 ** -18 * (v[best].abs() + v[5].abs())  # (fp32: (64 + 8) 2^-24 of scores up to 8, twice, and the sums)
    # (the others: 2^-24 each at most, and a fp16 weight is 2^-39 of the largest at least)
    bound += n * 2.0 ** -24 * v.abs().amax(0)
    assert ((out[:, 0].cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,storage", TYPES)
def test_the_same_call_gives_the_same_bits(dtype, storage):
    for n, m in ((75, 75), (2000, 300), (3000, 5)):
        cache, _ = make([n, 50], 2, 128, 16, dtype, storage)
        q = rows_like(cache, m + 40, 8).cuda()
        calls = []
        for _ in range(3):
            lse = torch.empty(m + 40, 8, device="cuda")
            calls.append((cache.attend_prompt(q, ends([m, 40]), lse=lse), lse))
        for out, lse in calls[1:]:
            assert torch.equal(out, calls[0][0]) and torch.equal(lse, calls[0][1])
