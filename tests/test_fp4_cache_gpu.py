"""The 4-bit pool behind the drop-in classes: PagedKVCacheFp4 with
PagedAttention, BatchPrefillAttention and DecodeGraphRunner in the reference's
call order, errors from the device, and StepRunner with kv_cache_dtype="fp4".

Attention is compared with 64-bit arithmetic over the rows that the cache reads
back (tolerances: tests/test_fp4_gpu.py). StepRunner's tokens are compared with
a torch forward of the same model whose attention runs over the rows that the
runner's own pool holds, so that only bf16 roundings lie between the two, as
in tests/test_step_runner_gpu.py, whose tolerance of a logit is used.
"""

import pytest
import torch
import torch.nn.functional as F

from nano_vllm_ascend_b200 import (BlockManager, DecodeGraphRunner, KVCacheDeviceError, NpuBatchPrefillAttention,
                                   NpuPagedAttention, PagedKVCacheFp4, check_errors)
from nano_vllm_ascend_b200.step_runner import StepRunner, _rms_norm
from oracle import fp4_oracle as orc
from tests.test_fp4_gpu import D, DECODE, PREFILL, SCALE, check, seq_slots
from tests.test_step_runner_gpu import LOGIT_TOL, SHAPE, Seq, _head_norm_rope

pytestmark = pytest.mark.gpu


def rows(n, heads, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, heads, D, generator=g).to(torch.bfloat16).to(dev)


def slots_of(bm, seq, n, dev):
    return seq_slots(torch.tensor(bm.block_tables[seq]), n, bm.block_size, dev)


@pytest.mark.parametrize("bs", [32, 128])
def test_drop_in_classes_in_the_reference_call_order(cuda_device, bs):
    """Dense prefill, prefill over a cached prefix, then decode, layer by layer, with constants of each layer."""
    dev, h, kvh, layers = cuda_device, 8, 2, 2
    bm = BlockManager(32, bs, dev)
    kv = PagedKVCacheFp4(layers, 32, bs, kvh, D, dev, k_scale=[1.0, 2.0], v_scale=[0.25, 1.0])
    prefill = NpuBatchPrefillAttention(h, kvh, D, bs, max_mask_len=2048)
    decode = NpuPagedAttention(h, kvh, D)
    lens = [bs + 9, 50]
    md = bm.prepare_prefill_metadata([0, 1], lens, [0, 0], [[], []])
    assert not md.use_paged_prefill
    for layer in range(layers):
        q, k, v = (rows(sum(lens), n, 10 * layer + i, dev) for i, n in enumerate((h, kvh, kvh)))
        kv.write(layer, k, v, md.slot_mapping)
        out = prefill(q, k, v, md, *kv.get_physical_cache(layer))
        for at, n in ((0, lens[0]), (lens[0], lens[1])):  # this step's own rows, not the pool's
            want, a = orc.attention(q[at:at + n], k[at:at + n].double(), v[at:at + n].double(), SCALE)
            err = (out[at:at + n].double() - want).abs()
            assert bool((err <= want.abs() * 2.0 ** -8 + a * (2.0 ** -8 + 2.0 ** -10)).all())
    prefix = bm.block_tables[0][:1]  # sequence 2 shares a block of sequence 0
    md = bm.prepare_prefill_metadata([2], [30], [bs], [list(prefix)])
    assert md.use_paged_prefill
    for layer in range(layers):
        q, k, v = (rows(30, n, 50 + 10 * layer + i, dev) for i, n in enumerate((h, kvh, kvh)))
        kv.write(layer, k, v, md.slot_mapping)
        out = prefill(q, k, v, md, *kv.get_physical_cache(layer))
        kr, vr = kv.read(layer, slots_of(bm, 2, bs + 30, dev))
        want, a = orc.attention(q, kr.double(), vr.double(), SCALE)
        check(out, want, a, vr.double(), PREFILL)
    ctx = [lens[0], lens[1], bs + 30]
    md = bm.prepare_decode_metadata([0, 1, 2], ctx, q_len=1)
    for layer in range(layers):
        q, k, v = (rows(3, n, 90 + 10 * layer + i, dev) for i, n in enumerate((h, kvh, kvh)))
        kv.write(layer, k, v, md.slot_mapping)
        out = decode(q, *kv.get_physical_cache(layer), md.block_tables, md.context_lens)
        for s, n in enumerate(ctx):
            kr, vr = kv.read(layer, slots_of(bm, s, n + 1, dev))
            want, a = orc.attention(q[s:s + 1], kr.double(), vr.double(), SCALE)
            check(out[s:s + 1], want, a, vr.double(), DECODE)
    check_errors(dev)


class TwoLayers:
    """A model of two attention layers over a 4-bit cache, in the graph runner's calling convention."""

    def __init__(self, h, kvh, dev):
        self.attn = NpuPagedAttention(h, kvh, D)
        self.q, self.k, self.v = (torch.zeros(2, 4, n, D, dtype=torch.bfloat16, device=dev) for n in (h, kvh, kvh))

    def __call__(self, input_ids_flat, position_ids_flat, kv_cache, attn_metadata, is_prefill=False):
        n = input_ids_flat.numel()
        outs = []
        for layer in range(2):
            kv_cache.write(layer, self.k[layer, :n], self.v[layer, :n], attn_metadata.slot_mapping)
            outs.append(self.attn(self.q[layer, :n], *kv_cache.get_physical_cache(layer), attn_metadata.block_tables,
                                  attn_metadata.context_lens))
        return type("Out", (), dict(logits=torch.stack(outs)))


def test_graph_runner_over_a_4_bit_cache(cuda_device):
    """Two batch sizes captured, then replayed in turn with new rows, lengths and tables."""
    dev, h, kvh, bs = cuda_device, 8, 2, 32
    bm = BlockManager(64, bs, dev)
    kv = PagedKVCacheFp4(2, 64, bs, kvh, D, dev)
    model = TwoLayers(h, kvh, dev)
    runner = DecodeGraphRunner(model, kv, batch_sizes=[2, 4], max_model_len=512, block_size=bs, device=dev)
    ctx = [0, 0, 0, 0]
    try:
        lens = [40, 33, 31, 64]
        md = bm.prepare_prefill_metadata([0, 1, 2, 3], lens, [0] * 4, [[]] * 4)
        for layer in range(2):
            kv.write(layer, rows(sum(lens), kvh, layer, dev), rows(sum(lens), kvh, 5 + layer, dev), md.slot_mapping)
        ctx = list(lens)
        for step, batch in enumerate((4, 2, 4, 2, 4)):
            seqs = list(range(batch)) if step != 3 else [1, 3]
            md = bm.prepare_decode_metadata(seqs, [ctx[s] for s in seqs], q_len=1)
            for i, t in enumerate((model.q, model.k, model.v)):
                t.copy_(rows(8, t.shape[2], 100 * step + i, dev).view_as(t))
            got = runner.forward(torch.zeros(batch, dtype=torch.long, device=dev),
                                 torch.zeros(batch, dtype=torch.long, device=dev), md)
            assert got is not None
            for s in seqs:
                ctx[s] += 1
            for layer in range(2):
                for i, s in enumerate(seqs):
                    kr, vr = kv.read(layer, slots_of(bm, s, ctx[s], dev))
                    want, a = orc.attention(model.q[layer, i:i + 1], kr.double(), vr.double(), SCALE)
                    check(got[layer, i:i + 1], want, a, vr.double(), DECODE, f"step {step} layer {layer} seq {s}")
        assert runner.stats_dict()["captures"] == 2 and runner.stats_dict()["replays"] == 5
        check_errors(dev)
    finally:
        runner.release()


def test_two_streams_and_a_captured_call_do_not_share_workspaces(cuda_device):
    """Long calls issued to two streams at once, and the same call captured by the caller's own graphs."""
    dev, h, kvh, bs = cuda_device, 4, 1, 64
    n = 3000
    kv = PagedKVCacheFp4(1, 96, bs, kvh, D, dev)
    kv.write(0, rows(96 * bs, kvh, 1, dev), rows(96 * bs, kvh, 2, dev), torch.arange(96 * bs))
    attn = NpuPagedAttention(h, kvh, D)
    layer = kv.get_physical_cache(0)
    tables = [torch.arange(48, dtype=torch.int32, device=dev)[None], torch.arange(48, 96, dtype=torch.int32, device=dev)[None]]
    ctx = torch.tensor([n], dtype=torch.int32, device=dev)
    q = [rows(1, h, 7 + i, dev) for i in range(2)]
    alone = [attn(q[i], *layer, tables[i], ctx) for i in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attn(q[i], *layer, tables[i], ctx))
    graphs, captured = [], []
    for s in streams:
        s.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured.append(attn(q[i], *layer, tables[i], ctx))
        graphs.append(g)
    for _ in range(3):
        for i in (1, 0):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        for out in outs[i] + [captured[i]]:
            assert torch.equal(out, alone[i])
    check_errors(dev)


def test_device_errors_raise(cuda_device):
    dev = cuda_device
    kv = PagedKVCacheFp4(1, 4, 16, 2, D, dev)
    attn = NpuPagedAttention(4, 2, D)
    layer = kv.get_physical_cache(0)
    k = rows(2, 2, 1, dev)
    kv.write(0, k, k, torch.tensor([1, 64], device=dev))
    with pytest.raises(IndexError):
        check_errors(dev)
    q = rows(1, 4, 2, dev)
    attn(q, *layer, torch.tensor([[9]], dtype=torch.int32, device=dev), torch.tensor([3], dtype=torch.int32, device=dev))
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        check_errors(dev)
    attn(q, *layer, torch.tensor([[1]], dtype=torch.int32, device=dev), torch.tensor([17], dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="missing block"):
        check_errors(dev)
    check_errors(dev)


def logits_over_pool(runner, seq):
    """The last position's logits of the runner's model in torch, attending over the rows that its pool holds."""
    model, s = runner.model, runner.model.shape
    tokens = seq.token_ids().to(runner.device)
    n = tokens.numel()
    slots = slots_of(runner.block_manager, runner._rows[seq.seq_id], n, runner.device)
    cos, sin = model.cos[:n], model.sin[:n]
    x = model.embed[tokens]
    for i, layer in enumerate(model.layers):
        h = _rms_norm(x, layer.in_norm, s.rms_norm_eps)
        qkv = F.linear(h, layer.qkv).view(n, -1, s.head_dim)
        q = _head_norm_rope(qkv[:, :s.num_heads], layer.q_norm, cos, sin, s.rms_norm_eps)
        k, v = runner.kv_cache.read(i, slots)
        if i == 0:  # what was stored is the first layer's own rows, off by at most half of the largest step (one scale)
            own = (_head_norm_rope(qkv[:, s.num_heads:s.num_heads + s.num_kv_heads], layer.k_norm, cos, sin,
                                   s.rms_norm_eps), qkv[:, s.num_heads + s.num_kv_heads:])
            for got, want in zip((k, v), own):
                amax = want.float().unflatten(-1, (8, 16)).abs().amax(-1, keepdim=True)
                err = (got.float() - want.float()).unflatten(-1, (8, 16)).abs()
                # the scale is at most 17/16 of a sixth of the largest; bf16 rows differ by 2^-7 of it between matmuls
                assert bool((err <= amax * (17 / 96 + 2.0 ** -6)).all())
        attn, _ = orc.attention(q, k.double(), v.double(), s.head_dim ** -0.5)
        x = x + F.linear(attn.reshape(n, -1).to(torch.bfloat16), layer.o)
        h = _rms_norm(x, layer.post_norm, s.rms_norm_eps)
        gate, up = F.linear(h, layer.gate_up).chunk(2, dim=-1)
        x = x + F.linear(F.silu(gate) * up, layer.down)
    return _rms_norm(x, model.final_norm, s.rms_norm_eps)[-1].float() @ model.embed.float().T


def test_step_runner_over_a_4_bit_cache(cuda_device):
    runner = StepRunner(SHAPE, cuda_device, max_model_len=1024, num_blocks=64, block_size=128, max_num_seqs=8,
                        enable_prefix_cache=True, decode_graph_batch_sizes=[1, 2, 4], seed=3, kv_cache_dtype="fp4",
                        k_scale=1.0, v_scale=0.5)
    g = torch.Generator().manual_seed(11)

    def greedy(seqs, what):
        for seq in seqs:
            logits = logits_over_pool(runner, seq)
            tok = seq.next_token_id
            assert float(logits[tok]) >= float(logits.max()) - LOGIT_TOL, f"{what}: seq {seq.seq_id}"

    try:
        a, b, c = (Seq(10 + i, torch.randint(0, 512, (n,), generator=g)) for i, n in enumerate((300, 129, 60)))
        runner.prepare_sequences([a, b, c])
        runner.prefill([a, b, c])
        greedy([a, b, c], "prefill")
        d = Seq(13, torch.cat([a.prompt_token_ids[:256], torch.randint(0, 512, (40,), generator=g)]))
        runner.prepare_sequences([d])
        assert d.cached_prefix_len == 256
        runner.prefill([d])
        greedy([d], "prefill (prefix hit)")
        for step in range(3):
            runner.decode([a, b, c, d])
            greedy([a, b, c, d], f"decode bs4 step {step}")
        runner.free_seq(c)
        for step in range(2):
            runner.decode([a, b, d])  # no graph of three
            greedy([a, b, d], f"decode bs3 step {step}")
        stats = runner.decode_graph_stats()
        assert stats["captures"] == 1 and stats["replays"] == 3 and stats["fallbacks"] == 2
    finally:
        runner.release()


def test_step_runner_sizes_the_pool_from_memory(cuda_device):
    """With the same share of memory a 4-bit pool has 3.5 times the blocks (512 / 144 bytes a row)."""
    counts = []
    for kind in ("bf16", "fp4"):
        free, total = torch.cuda.mem_get_info(cuda_device)
        share = (total - free + (2 << 30)) / total  # the model and about 2 GiB
        runner = StepRunner(SHAPE, cuda_device, max_model_len=256, memory_utilization=share, enable_decode_graph=False,
                            kv_cache_dtype=kind)
        counts.append(runner.num_blocks)
        runner.release()
        del runner
        torch.cuda.empty_cache()
    assert 3.3 < counts[1] / counts[0] < 3.8
    with pytest.raises(ValueError, match="neither"):
        StepRunner(SHAPE, cuda_device, num_blocks=4, kv_cache_dtype="int4")
