"""The workspaces of prompts whose keys are cut: one cache's and its forks', and their bytes."""
import pytest
import torch

from prismkv_amd import Rotary
from tests.serving_util import BF16, FP32, ends, make, rows_like

pytestmark = pytest.mark.gpu


def workspaces(cache):
    return sorted(size for name, size in cache.buffer_bytes().items() if name.startswith("prompt_work"))


def test_a_prompt_into_a_new_fork_inside_a_capture():
    cache, _ = make([3000, 400], 2, 128, 16, BF16, room=100)
    rotary = Rotary(128)
    q, k, v = (rows_like(cache, 60, h, s).cuda() for h, s in ((8, 1), (2, 2), (2, 3)))
    e = ends([40, 20])
    want = cache.prompt(q, k, v, e, rotary=rotary, into=cache.fork())
    held = workspaces(cache)
    assert held and held[-1] > 16
    fork = cache.fork()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.prompt(q, k, v, e, rotary=rotary, into=fork)
    for _ in range(3):
        out.zero_()
        fork.lengths.zero_()
        graph.replay()
        cache.attend_prompt(q, e)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and fork.lengths.tolist() == [3040, 420]
    cache.check_errors()
    assert workspaces(cache) == held and not workspaces(fork)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (256, FP32)])
def test_bytes(dim, dtype):
    """1024 states at most, of 128 rows of products, a maximum and a sum in fp32, and no
    more than that; a smaller prompt takes what is there, a larger one twice as much."""
    state = 128 * (dim + 2) * 4
    cache, _ = make([20000], 1, dim, 64, dtype)
    prompt = lambda rows: cache.attend_prompt(rows_like(cache, rows, 1).cuda(), ends([rows]))  # noqa: E731
    prompt(1000)
    assert workspaces(cache) == [1024 * state]
    for rows in (1, 130, 500, 2000):
        prompt(rows)
    assert workspaces(cache) == [1024 * state]
    cache, _ = make([2000], 1, dim, 64, dtype)
    for rows in (100, 1000, 1900):
        prompt(rows)
    assert all(size % state == 0 and bin(size // state).count("1") == 1 for size in workspaces(cache))
    assert len(workspaces(cache)) > 1
    cache.check_errors()
