"""Pages of a pool: copies, clearing and remapped tables, bit for bit against indexing."""

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import ops

pytestmark = pytest.mark.gpu


def pools_of(dev, layers, blocks, shape, dtype, tensors, seed=0):
    g = torch.Generator().manual_seed(seed)
    words = int(np.prod(shape)) * dtype.itemsize // 2
    return [torch.randint(-(1 << 15), 1 << 15, (layers, blocks, words), generator=g, dtype=torch.int16)
            .to(dev).view(dtype).view(layers, blocks, *shape) for _ in range(tensors)]


@pytest.mark.parametrize("layers,blocks,shape,dtype,tensors", [
    (1, 3, (16, 1, 8), torch.bfloat16, 1), (28, 40, (16, 2, 128), torch.bfloat16, 2),
    (3, 50, (128, 8, 128), torch.float16, 2), (5, 33, (2, 4, 4128), torch.uint8, 1),
    (2, 30, (3, 1, 2304), torch.uint8, 1), (4, 9, (8,), torch.float32, 1), (2, 9, (8, 16, 4128), torch.uint8, 1),
    (1, 700, (16, 1, 128), torch.bfloat16, 2)])
def test_copies_and_clears(cuda_device, layers, blocks, shape, dtype, tensors):
    dev = cuda_device
    pools = pools_of(dev, layers, blocks, shape, dtype, tensors)
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist()
    n = blocks // 3
    pairs = [(perm[i], perm[n + i]) for i in range(n)] + [(-1, perm[2 * n]), (5 % blocks, -1), (-1, -1)]
    pairs += [(perm[0], perm[2 * n + 1])] if 2 * n + 1 < blocks else []  # one source, two destinations
    want = [p.clone() for p in pools]
    for w, p in zip(want, pools):
        for s, d in pairs:
            if d >= 0:
                w[:, d] = p[:, s] if s >= 0 else 0
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.copy_blocks(pools, torch.tensor(pairs, dtype=torch.int32, device=dev), error_word=err)
    for w, p in zip(want, pools):
        assert torch.equal(w.view(torch.uint8), p.view(torch.uint8))
    assert int(err.item()) == 0


def test_blocks_outside_the_pool_are_skipped_and_flagged(cuda_device):
    dev = cuda_device
    for bad in ((9, 1), (0, 9), (-2, 1), (0, -2), (1 << 30, 1), (0, 1 << 30)):
        (pool,) = pools_of(dev, 2, 9, (16, 1, 128), torch.bfloat16, 1)
        want = pool.clone()
        want[:, 4] = pool[:, 3]
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.copy_blocks(pool, torch.tensor([bad, (3, 4)], dtype=torch.int32, device=dev), error_word=err)
        assert torch.equal(want.view(torch.int16), pool.view(torch.int16)) and int(err.item()) == 2, bad
        ops.copy_blocks(pool, torch.tensor([bad], dtype=torch.int32, device=dev))  # nowhere to report to


def test_one_block_onto_itself_and_no_pairs(cuda_device):
    dev = cuda_device
    (pool,) = pools_of(dev, 2, 5, (16, 1, 128), torch.bfloat16, 1)
    want = pool.clone()
    ops.copy_blocks(pool, torch.tensor([(2, 2)], dtype=torch.int32, device=dev))
    ops.copy_blocks(pool, torch.empty(0, 2, dtype=torch.int32, device=dev))
    assert torch.equal(want.view(torch.int16), pool.view(torch.int16))


def test_far_offsets(cuda_device):
    """Layers and blocks past 4 GiB."""
    dev = cuda_device
    pool = torch.zeros(3, 700, 8, 128, 4128, dtype=torch.uint8, device=dev)
    pool[:, 699] = torch.arange(3, device=dev, dtype=torch.uint8)[:, None, None, None] + 7
    pool[:, 1] = 3
    ops.copy_blocks(pool, torch.tensor([(699, 0), (1, 698), (-1, 697)], dtype=torch.int32, device=dev))
    assert torch.equal(pool[:, 0], pool[:, 699]) and bool((pool[:, 698] == 3).all())
    assert bool((pool[2, 0] == 9).all()) and not pool[:, 2:697].any()


@pytest.mark.parametrize("rows,width,gap", [(1, 1, 0), (3, 7, 0), (33, 48, 16), (1, 5000, 3), (700, 320, 0)])
def test_tables_follow(cuda_device, rows, width, gap):
    dev = cuda_device
    nb = 1000
    g = torch.Generator().manual_seed(1)
    whole = torch.randint(0, nb, (rows, width + gap), generator=g, dtype=torch.int32).to(dev)
    block_map = torch.randperm(nb, generator=g).to(torch.int32).to(dev)
    want = whole.clone()
    want[:, :width] = block_map[whole[:, :width].long()]
    ops.remap_blocks(whole[:, :width], block_map)
    assert torch.equal(whole, want)


def test_ids_outside_the_map_stay_and_are_flagged(cuda_device):
    dev = cuda_device
    tables = torch.tensor([[0, 1, 2], [-1, 3, 900]], dtype=torch.int32, device=dev)
    block_map = torch.tensor([3, 2, -1, 4], dtype=torch.int32, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.remap_blocks(tables, block_map, error_word=err)
    assert tables.tolist() == [[3, 2, 2], [-1, 3, 900]] and int(err.item()) == 2


def test_in_a_graph_with_padding(cuda_device):
    dev = cuda_device
    (pool,) = pools_of(dev, 4, 20, (2, 4, 4128), torch.uint8, 1)
    pairs = torch.full((6, 2), -1, dtype=torch.int32, device=dev)
    ops.copy_blocks(pool, pairs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_blocks(pool, pairs)
    want = pool.clone()
    for step in ([(1, 2)], [(2, 3), (0, 5), (-1, 7)], []):
        pairs.fill_(-1)
        for i, p in enumerate(step):
            pairs[i] = torch.tensor(p, dtype=torch.int32)
            want[:, p[1]] = want[:, p[0]] if p[0] >= 0 else 0
        graph.replay()
        assert torch.equal(pool, want)
