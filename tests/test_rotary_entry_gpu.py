"""Calls of ``nvk_rotary`` that ``ops.rotary`` does not make, against the formula in 64 bits (see test_rotary_gpu)."""

import pytest
import torch

from nano_vllm_ascend_b200 import _lib
from tests.test_rotary_gpu import check, formula, frequencies

pytestmark = pytest.mark.gpu


# whole vectors of eight and of two elements, and element by element
@pytest.mark.parametrize("dim,rotated", [(128, 64), (20, 12), (130, 66)])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("weights", ["neither", "query's", "key's", "both"])
@pytest.mark.parametrize("has", ["query", "key"])
def test_weights_of_an_absent_side_are_not_used(cuda_device, has, weights, interleaved, dim, rotated):
    """With heads of q or of k alone, that side's weight says whether it is normed, and the other side's pointers are
    not looked at."""
    dev, t, h = cuda_device, 7, 3
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(t, h, dim, generator=g).to(torch.bfloat16).to(dev)
    w = (1 + 0.3 * torch.randn(2, dim, generator=g)).to(torch.bfloat16).to(dev)
    inv, pos = frequencies(rotated // 2).to(dev), torch.randint(0, 1000, (t,), generator=g).to(dev)
    out, side = torch.full_like(x, float("nan")), int(has == "key")
    given = [weights in ("query's", "both"), weights in ("key's", "both")]

    def two(mine):  # (q's, k's) arguments
        return (0, mine) if side else (mine, 0)

    _lib.call("nvk_rotary", *two(out.data_ptr()), *two(x.data_ptr()), *two(h * dim), *two(h * dim),
              *(w[i].data_ptr() if given[i] else 0 for i in (0, 1)), 1e-6, inv.data_ptr(), pos.data_ptr(), 1.0, t,
              *two(h), dim, rotated, interleaved, 0, torch.cuda.current_stream(dev).cuda_stream)
    want, mag = formula(x, w[side] if given[side] else None, 1e-6, inv, pos, bool(interleaved), 1.0)
    check(out, want, mag)
