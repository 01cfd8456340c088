"""A block copied onto itself is left alone; one outside the pool is flagged there too."""

import pytest
import torch

from nano_vllm_ascend_b200 import ops
from tests.test_pages_gpu import pools_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block,flagged", [(0, 0), (8, 0), (-1, 0), (9, 2), (-2, 2), (1 << 30, 2)])
def test_a_block_onto_itself(cuda_device, block, flagged):
    dev = cuda_device
    (pool,) = pools_of(dev, 2, 9, (16, 1, 128), torch.bfloat16, 1)
    want = pool.clone()
    want[:, 4] = pool[:, 3]
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.copy_blocks(pool, torch.tensor([(block, block), (3, 4)], dtype=torch.int32, device=dev), error_word=err)
    assert torch.equal(want.view(torch.int16), pool.view(torch.int16)) and int(err.item()) == flagged
