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
