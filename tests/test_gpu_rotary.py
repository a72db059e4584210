"""Rows turned by rotary positions on their way into the paged cache, against the
64-bit definition (oracle/paged.py)."""
import pytest
import torch

from oracle import paged
from prismkv_amd import PagedCache, Rotary
from tests.serving_util import BF16, FP16, FP32, ends, make, rows_like

pytestmark = pytest.mark.gpu

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
CASES = [
    # dim, dtype, rotary_dim, interleaved, scaling, scored
    (128, BF16, 128, False, None, False),
    (128, BF16, 128, True, YARN, True),
    (128, FP16, 64, False, LLAMA3, True),
    (128, FP32, 48, True, {"rope_type": "linear", "factor": 4.0}, False),
    (64, BF16, 16, False, None, True),
    (64, FP16, 64, True, LLAMA3, False),
    (64, FP32, 32, False, YARN, True),
    (256, BF16, 256, False, YARN, False),
    (256, FP32, 128, True, None, True),
    (256, FP16, 240, False, None, False),
]


def check(got, x, positions, rotary):
    want, bound = paged.turn(x, positions, rotary.frequencies, rotary.amplitude, rotary.interleaved)
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), float((err / bound.clamp_min(1e-300)).max())


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dim,dtype,part,interleaved,scaling,scored", CASES)
def test_turned_appends(dim, dtype, part, interleaved, scaling, scored, packed):
    lengths, new = [5, 0, 40], [13, 1, 30] if packed else [1, 1, 1]
    cache, host = make(lengths, 2, dim, 17, dtype, room=31, scored=scored)
    if scored:
        cache.seen.copy_(torch.tensor([3_000_000, 0, 2 ** 31 - 100]))
    rotary = Rotary(dim, base=5e5, rotary_dim=part, interleaved=interleaved, scaling=scaling)
    rows = sum(new)
    qkv = rows_like(cache, rows, 6 + 2 + 2)  # parts of one projection
    on = qkv.cuda()
    q, k, v = on[:, :6], on[:, 6:8], on[:, 8:]
    first = [3_000_000, 0, 2 ** 31 - 100] if scored else lengths
    positions = torch.cat([f + torch.arange(m) for f, m in zip(first, new)])
    fork = cache.fork()
    turned = cache.append(k, v, ends(new) if packed else None, q=q, rotary=rotary, into=fork)
    assert turned.is_contiguous() and turned.dtype == dtype
    check(turned, qkv[:, :6], positions, rotary)
    assert fork.lengths.tolist() == [n + m for n, m in zip(lengths, new)] and cache.lengths.tolist() == lengths
    got_k, got_v = fork.read(ends(new), rows=rows)
    check(got_k, qkv[:, 6:8], positions, rotary)
    assert torch.equal(got_v.cpu(), qkv[:, 8:])
    fork.check_errors()
    if scored:
        assert fork.seen.tolist() == [f + m for f, m in zip(first, new)]
        for b, (n, m) in enumerate(zip(lengths, new)):
            assert (fork.scores[b, :, n:n + m] == 0).all()
            assert fork.positions[b, 0, n:n + m].tolist() == [first[b] + i for i in range(m)]
    # without queries, in place: the same keys
    assert cache.append(k, v, ends(new) if packed else None, rotary=rotary) is None
    assert torch.equal(cache.read(ends(new), rows=rows)[0], got_k)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_turned_rows_in_four_bits_are_those_turned_before(dtype):
    rotary = Rotary(128, base=1e6)
    plain, _ = make([7, 20], 2, 128, 16, dtype, room=20)
    four, _ = make([7, 20], 2, 128, 16, dtype, "mxfp4", room=20)
    again, _ = make([7, 20], 2, 128, 16, dtype, "mxfp4", room=20)
    k, v, q = (rows_like(plain, 18, h, s).cuda() for h, s in ((2, 1), (2, 2), (8, 3)))
    e = ends([11, 7])
    q0 = plain.append(k, v, e, q=q, rotary=rotary)
    q1 = four.append(k, v, e, q=q, rotary=rotary)
    assert torch.equal(q0, q1)
    turned, values = plain.read(e, rows=18)
    again.append(turned, values, e)
    for a, b in zip(four.read(e, rows=18), again.read(e, rows=18)):
        assert torch.equal(a, b)


def test_steps_and_prompts_with_a_rotary():
    rotary = Rotary(128)
    for storage in (None, "mxfp4"):
        cache, _ = make([3, 50], 2, 128, 16, BF16, storage, room=30)
        other, _ = make([3, 50], 2, 128, 16, BF16, storage, room=30)
        k, v, q = (rows_like(cache, 20, h, s).cuda() for h, s in ((2, 1), (2, 2), (8, 3)))
        e = ends([5, 15])
        out = cache.prompt(q, k, v, e, rotary=rotary)
        turned = other.append(k, v, e, q=q, rotary=rotary)
        assert torch.equal(out, other.attend_prompt(turned, e))
        out = cache(q[:2], k[:2], v[:2], rotary=rotary)
        turned = other.append(k[:2], v[:2], q=q[:2], rotary=rotary)
        assert torch.equal(out, other.attend(turned))
        cache.check_errors()
