"""Reports of what the device finds in calls with nothing to do."""
import pytest
import torch

from tests.serving_util import BF16, FP16, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,storage", [(BF16, None), (FP16, "mxfp4")])
@pytest.mark.parametrize("bad", [[0, 0, 5], [1, 1, 1], [0, 3, 0], [0, -2, 0]])
def test_offsets_of_a_read_of_no_rows(bad, dtype, storage):
    cache, _ = make([30, 20], 1, 64, 16, dtype, storage)
    offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
    k, v = cache.read(offsets, rows=0)
    assert k.shape == v.shape == (0, 1, 64)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="offsets of a prompt or a read"):
        cache.check_errors()
    cache.read(torch.zeros(3, dtype=torch.int32, device="cuda"), rows=0)
    torch.cuda.synchronize()
    cache.check_errors()
