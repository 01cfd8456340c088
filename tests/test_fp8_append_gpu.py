"""Longer appends into the 8-bit pool whose blocks share their units with other blocks, bit for bit.

Above 512 rows a block takes 16 rows, and where there are few such blocks up to
16 more work on the same rows, each on a share of the (unit, head, K or V)
items: every item has to be done by exactly one of them, so they have to agree
on the order of the units.
"""

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import ops_fp8
from oracle import fp8_oracle as orc
from tests.test_fp8_gpu import append_both, random_rows

pytestmark = pytest.mark.gpu


def own_sequences(tokens, seed):
    """One row each of as many sequences: any offset of a unit of its own, the units in any order."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(tokens, generator=g) * 16 + torch.randint(0, 16, (tokens,), generator=g)


def prompt_from(offset, tokens):
    return torch.arange(tokens) + offset


def ragged(tokens, seed):
    """Prompts of 1 to 40 rows, each from the start of a block of 64."""
    g = torch.Generator().manual_seed(seed)
    parts, left, at = [], tokens, 0
    while left:
        n = min(left, int(torch.randint(1, 41, (1,), generator=g)))
        parts.append(torch.arange(n) + at)
        left, at = left - n, at + 64
    return torch.cat(parts)


SHORTER = [("own", 513), ("own", 600), ("own", 1024), ("prompt", 1000), ("ragged", 700)]
LONGER = [("own", 2369), ("own", 4000), ("prompt", 4700), ("ragged", 3000)]


@pytest.mark.parametrize("kind,tokens,kvh", [(*case, kvh) for case in SHORTER for kvh in (1, 2, 8)]
                         + [(*case, kvh) for case in LONGER for kvh in (1, 2)])
def test_every_item_of_shared_blocks_is_done_once(cuda_device, kind, tokens, kvh):
    dev = cuda_device
    slots = {"own": lambda: own_sequences(tokens, 3), "prompt": lambda: prompt_from(5, tokens),
             "ragged": lambda: ragged(tokens, 4)}[kind]()
    bs = 64
    nb = int(slots.max()) // bs + 1
    want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    for step in range(2):  # the second time over what the first one left: raised, or anew
        k, v = random_rows(tokens, kvh, tokens + step)
        append_both(dev, want, pool, (k * 4.0 ** step).to(dev), (v * 4.0 ** step).to(dev), slots)


@pytest.mark.parametrize("tokens", [600, 1500])
def test_shared_blocks_repeat(cuda_device, tokens):
    """Many calls from the same bytes end in the same bytes."""
    dev, kvh, bs = cuda_device, 3, 16
    slots = own_sequences(tokens, 7).to(dev)
    start = torch.zeros(ops_fp8.pool_shape(tokens, bs, kvh), dtype=torch.uint8, device=dev)
    k, v = (t.to(dev) for t in random_rows(tokens, kvh, 1))
    ops_fp8.kv_append_fp8(start, k, v, torch.arange(tokens, device=dev) * 16 + 3)
    first = None
    for _ in range(200):
        pool = start.clone()
        ops_fp8.kv_append_fp8(pool, k * 2, v * 8, slots)
        first = pool if first is None else first
        assert torch.equal(pool, first)
    want = start.cpu().numpy()
    orc.append(want, (k * 2).cpu().float().numpy(), (v * 8).cpu().float().numpy(), slots.cpu().numpy())
    assert np.array_equal(first.cpu().numpy(), want)
