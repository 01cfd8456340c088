"""Device errors of 4-bit decode: from calls that the caller's own graph captured, and from other streams."""

import pytest
import torch

from nano_vllm_ascend_b200 import KVCacheDeviceError, NpuPagedAttention, PagedKVCacheFp4, check_errors, ops_fp4

pytestmark = pytest.mark.gpu

D, BS = 128, 16
SLEEP = 100_000_000  # cycles: 50 ms and more


def setup(dev, h=4, kvh=2):
    check_errors(dev)
    kv = PagedKVCacheFp4(1, 4, BS, kvh, D, dev)
    q = torch.randn(1, h, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    ctx = torch.full((1,), 3, dtype=torch.int32, device=dev)
    return NpuPagedAttention(h, kvh, D), kv.get_physical_cache(0), q, table, ctx


def test_a_replayed_call_reports(cuda_device):
    """A bad block id or a context that is too long in a replay of the caller's own graph raises, in each replay that
    has one and in no other."""
    dev = cuda_device
    attn, layer, q, table, ctx = setup(dev)
    attn(q, *layer, table, ctx)  # (loads the library outside the capture)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [attn(q, *layer, table, ctx) for _ in range(2)]
    graph.replay()
    check_errors(dev)
    table.fill_(9)
    graph.replay()
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        check_errors(dev)
    table.fill_(1)
    graph.replay()
    check_errors(dev)
    ctx.fill_(BS + 1)
    graph.replay()
    graph.replay()
    with pytest.raises(RuntimeError, match="missing block"):
        check_errors(dev)
    ctx.fill_(3)
    graph.replay()
    check_errors(dev)
    want = attn(q, *layer, table, ctx)
    assert all(torch.equal(o, want) for o in outs)
    check_errors(dev)


def test_decode_reports_where_it_is_told_to(cuda_device):
    """The given word gets the bits, the workspace's own stays clear; what is no int32 of the device is refused."""
    dev = cuda_device
    _, (layer, _), q, table, ctx = setup(dev)
    ws = torch.zeros(ops_fp4.decode_fp4_workspace_bytes(4, 2), dtype=torch.uint8, device=dev)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    ops_fp4.paged_decode_fp4(out, q, layer.pool, table + 9, ctx, 0.1, ws, error_word=word)
    assert int(word.item()) == 2 and not ws[:4].any()
    ops_fp4.paged_decode_fp4(out, q, layer.pool, table, ctx + BS, 0.1, ws)
    assert int(word.item()) == 2 and int(ws[:4].view(torch.int32).item()) == 8
    for wrong in (word.long(), word.cpu(), word[:0]):
        with pytest.raises(ValueError, match="error_word"):
            ops_fp4.paged_decode_fp4(out, q, layer.pool, table, ctx, 0.1, ws, error_word=wrong)


def test_check_errors_waits_for_other_streams(cuda_device):
    """A call on a stream that is still busy when another stream asks for errors."""
    dev = cuda_device
    attn, layer, q, table, ctx = setup(dev)
    attn(q, *layer, table, ctx)
    check_errors(dev)
    bad = table + 9
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
        attn(q, *layer, table, ctx)  # its read of the word is in flight for a while ...
        torch.cuda._sleep(SLEEP)
        attn(q, *layer, bad, ctx)    # ... so this call's waits for the next one
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        check_errors(dev)
    check_errors(dev)


def test_clearing_a_word_loses_nothing_of_another_stream(cuda_device):
    """One stream's error is raised there and cleared late, behind other work; a replay on another stream sets
    another one meanwhile."""
    dev = cuda_device
    attn, layer, q, table, ctx = setup(dev)
    bad, far = table + 9, ctx + BS
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        attn(q, *layer, table, ctx)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(q, *layer, table, far)
    attn(q, *layer, bad, ctx)
    torch.cuda.synchronize(dev)  # the read of the word has landed
    torch.cuda._sleep(SLEEP)
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        attn(q, *layer, table, ctx)  # raises before it launches; the word is cleared behind the sleep
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.synchronize(dev)
    with pytest.raises(RuntimeError, match="missing block"):
        check_errors(dev)
    check_errors(dev)


def test_an_error_is_not_raised_twice(cuda_device):
    dev = cuda_device
    attn, layer, q, table, ctx = setup(dev)
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            attn(q, *layer, table + 9, ctx)
            s.synchronize()
        with pytest.raises(KVCacheDeviceError):
            check_errors(dev)
        check_errors(dev)


def test_a_larger_workspace_keeps_the_error_of_the_smaller_one(cuda_device):
    """A call with more heads, which needs a larger workspace, comes before the error of an earlier call was read."""
    dev = cuda_device
    attn, layer, q, table, ctx = setup(dev)
    big, big_layer, big_q, _, _ = setup(dev, 64, 8)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        torch.cuda._sleep(SLEEP)
        attn(q, *layer, table, ctx)      # its read of the word is in flight for a while ...
        attn(q, *layer, table + 9, ctx)  # ... so this call's waits for the next one
        big(big_q, *big_layer, table, ctx)
        with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
            check_errors(dev)
        check_errors(dev)
