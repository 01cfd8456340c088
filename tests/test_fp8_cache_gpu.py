"""The 8-bit pool behind the drop-in classes: PagedKVCacheFp8 with
PagedAttention, BatchPrefillAttention and DecodeGraphRunner in the reference's
call order, errors from the device, and StepRunner with kv_cache_dtype="fp8";
then sequences forked and the pool compacted between steps, over each kind of
pool.

Attention is compared with 64-bit arithmetic over the rows that the cache reads
back (tolerances: tests/test_fp8_gpu.py). StepRunner's tokens are compared with
a torch forward of the same model whose attention runs over the rows that the
runner's own pool holds, so that only bf16 roundings lie between the two, as
in tests/test_step_runner_gpu.py, whose tolerance of a logit is used.
"""

import pytest
import torch
import torch.nn.functional as F

from nano_vllm_ascend_b200 import (BlockManager, DecodeGraphRunner, KVCacheDeviceError, NpuBatchPrefillAttention,
                                   NpuPagedAttention, PagedKVCache, PagedKVCacheFp4, PagedKVCacheFp8, check_errors,
                                   ops)
from nano_vllm_ascend_b200.device_metadata import DeviceBlockTables
from nano_vllm_ascend_b200.step_runner import StepRunner, _rms_norm
from oracle import fp4_oracle as orc
from tests.test_fp8_gpu import D, DECODE, PREFILL, SCALE, check, seq_slots
from tests.test_step_runner_gpu import LOGIT_TOL, SHAPE, Seq, _head_norm_rope

pytestmark = pytest.mark.gpu


def rows(n, heads, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, heads, D, generator=g).to(torch.bfloat16).to(dev)


def slots_of(bm, seq, n, dev):
    return seq_slots(torch.tensor(bm.block_tables[seq]), n, bm.block_size, dev)


@pytest.mark.parametrize("bs", [16, 128])
def test_drop_in_classes_in_the_reference_call_order(cuda_device, bs):
    """Dense prefill, prefill over a cached prefix, then decode, layer by layer."""
    dev, h, kvh, layers = cuda_device, 8, 2, 2
    bm = BlockManager(32, bs, dev)
    kv = PagedKVCacheFp8(layers, 32, bs, kvh, D, dev)
    prefill = NpuBatchPrefillAttention(h, kvh, D, bs, max_mask_len=2048)
    decode = NpuPagedAttention(h, kvh, D)
    lens = [bs + 9, 50]
    md = bm.prepare_prefill_metadata([0, 1], lens, [0, 0], [[], []])
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
        check(out, want, a, bs + 30, float(vr.abs().max()), PREFILL)
    ctx = [lens[0], lens[1], bs + 30]
    md = bm.prepare_decode_metadata([0, 1, 2], ctx, q_len=1)
    for layer in range(layers):
        q, k, v = (rows(3, n, 90 + 10 * layer + i, dev) for i, n in enumerate((h, kvh, kvh)))
        kv.write(layer, k, v, md.slot_mapping)
        out = decode(q, *kv.get_physical_cache(layer), md.block_tables, md.context_lens)
        for s, n in enumerate(ctx):
            kr, vr = kv.read(layer, slots_of(bm, s, n + 1, dev))
            want, a = orc.attention(q[s:s + 1], kr.double(), vr.double(), SCALE)
            check(out[s:s + 1], want, a, n + 1, float(vr.abs().max()), DECODE)
    check_errors(dev)


class TwoLayers:
    """A model of two attention layers, the rows turned by their positions, in the graph runner's calling convention."""

    def __init__(self, h, kvh, dev):
        self.attn = NpuPagedAttention(h, kvh, D)
        self.q, self.k, self.v = (torch.zeros(2, 4, n, D, dtype=torch.bfloat16, device=dev) for n in (h, kvh, kvh))
        self.inv = torch.rand(D // 2, dtype=torch.float64, device=dev)

    def turned(self, layer, n, pos):
        return ops.rotary(self.q[layer, :n], self.k[layer, :n], self.inv, pos)

    def __call__(self, input_ids_flat, position_ids_flat, kv_cache, attn_metadata, is_prefill=False):
        n = input_ids_flat.numel()
        outs = []
        for layer in range(2):
            q, k = self.turned(layer, n, position_ids_flat)
            kv_cache.write(layer, k, self.v[layer, :n], attn_metadata.slot_mapping)
            outs.append(self.attn(q, *kv_cache.get_physical_cache(layer), attn_metadata.block_tables,
                                  attn_metadata.context_lens))
        return type("Out", (), dict(logits=torch.stack(outs)))


def test_graph_runner_over_an_8_bit_cache(cuda_device):
    """Two batch sizes captured, then replayed in turn with new rows, positions, lengths and tables."""
    dev, h, kvh, bs = cuda_device, 8, 2, 32
    bm = BlockManager(64, bs, dev)
    kv = PagedKVCacheFp8(2, 64, bs, kvh, D, dev)
    model = TwoLayers(h, kvh, dev)
    runner = DecodeGraphRunner(model, kv, batch_sizes=[2, 4], max_model_len=512, block_size=bs, device=dev)
    try:
        ctx = [40, 33, 31, 64]
        md = bm.prepare_prefill_metadata([0, 1, 2, 3], ctx, [0] * 4, [[]] * 4)
        for layer in range(2):
            kv.write(layer, rows(sum(ctx), kvh, layer, dev), rows(sum(ctx), kvh, 5 + layer, dev), md.slot_mapping)
        for step, batch in enumerate((4, 2, 4, 2, 4)):
            seqs = list(range(batch)) if step != 3 else [1, 3]
            held = [kv.read(layer, slots_of(bm, s, ctx[s], dev)) for layer in range(2) for s in seqs]
            md = bm.prepare_decode_metadata(seqs, [ctx[s] for s in seqs], q_len=1)
            for i, t in enumerate((model.q, model.k, model.v)):
                t.copy_(rows(8, t.shape[2], 100 * step + i, dev).view_as(t))
            pos = torch.tensor([ctx[s] for s in seqs], device=dev)
            got = runner.forward(torch.zeros(batch, dtype=torch.long, device=dev), pos, md)
            assert got is not None
            for s in seqs:
                ctx[s] += 1
            for layer in range(2):
                q, k = model.turned(layer, batch, pos)
                for i, s in enumerate(seqs):
                    kr, vr = kv.read(layer, slots_of(bm, s, ctx[s], dev))
                    for now, before, new in zip((kr, vr), held[layer * batch + i], (k[i], model.v[layer, i])):
                        # codes keep half a step of a value, or of the unit's largest (below 2^5 here) at 2^-17
                        assert bool(((now[:-1] - before).abs() <= before.abs() * 2.0 ** -4 + 2.0 ** -12).all())
                        assert bool(((now[-1] - new).abs() <= new.abs() * 2.0 ** -4 + 2.0 ** -12).all())
                    want, a = orc.attention(q[i:i + 1], kr.double(), vr.double(), SCALE)
                    check(got[layer, i:i + 1], want, a, ctx[s], float(vr.abs().max()), DECODE,
                          f"step {step} layer {layer} seq {s}")
        assert runner.stats_dict()["captures"] == 2 and runner.stats_dict()["replays"] == 5
        check_errors(dev)
    finally:
        runner.release()


def test_two_streams_and_a_captured_call_do_not_share_workspaces(cuda_device):
    """Long calls issued to two streams at once, and the same call captured by the caller's own graphs."""
    dev, h, kvh, bs = cuda_device, 4, 1, 64
    n = 3000
    kv = PagedKVCacheFp8(1, 96, bs, kvh, D, dev)
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


def test_one_attention_over_pools_of_both_kinds_in_turn(cuda_device):
    """Their workspace is one: calls over a 4- and an 8-bit pool alternate on a stream, each split over many CTAs."""
    dev, h, kvh, bs = cuda_device, 8, 2, 64
    caches = [PagedKVCacheFp4(1, 64, bs, kvh, D, dev), PagedKVCacheFp8(1, 64, bs, kvh, D, dev)]
    for kv in caches:
        kv.write(0, rows(64 * bs, kvh, 1, dev), rows(64 * bs, kvh, 2, dev), torch.arange(64 * bs))
    attn = NpuPagedAttention(h, kvh, D)
    q = rows(2, h, 3, dev)
    table = torch.arange(64, dtype=torch.int32, device=dev).view(2, 32)
    ctx = torch.tensor([2000, 1500], dtype=torch.int32, device=dev)
    alone = [attn(q, *kv.get_physical_cache(0), table, ctx) for kv in caches]
    for _ in range(5):
        for kv, want in zip(caches, alone):
            assert torch.equal(attn(q, *kv.get_physical_cache(0), table, ctx), want)
    check_errors(dev)


def test_device_errors_raise(cuda_device):
    dev = cuda_device
    kv = PagedKVCacheFp8(1, 4, 16, 2, D, dev)
    attn = NpuPagedAttention(4, 2, D)
    layer = kv.get_physical_cache(0)
    k = rows(2, 2, 1, dev)
    kv.write(0, k, k, torch.tensor([1, 64], device=dev))
    with pytest.raises(IndexError):
        check_errors(dev)
    kv.read(0, torch.tensor([1, 64], device=dev))
    with pytest.raises(IndexError):
        check_errors(dev)
    q = rows(1, 4, 2, dev)
    attn(q, *layer, torch.tensor([[9]], dtype=torch.int32, device=dev), torch.tensor([3], dtype=torch.int32, device=dev))
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        check_errors(dev)
    attn(q, *layer, torch.tensor([[1]], dtype=torch.int32, device=dev), torch.tensor([17], dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="missing block"):
        check_errors(dev)
    kv.copy_blocks(torch.tensor([[0, 4]], dtype=torch.int32, device=dev))
    with pytest.raises(KVCacheDeviceError, match="outside the KV pool"):
        check_errors(dev)
    check_errors(dev)


# ------------------------------------------------------------ StepRunner ---
def held_rows(runner, layer, slots):
    kv = runner.kv_cache
    if isinstance(kv, PagedKVCache):
        s = runner.shape
        return tuple(t[layer].view(-1, s.num_kv_heads, s.head_dim)[slots] for t in (kv.key_cache, kv.value_cache))
    return kv.read(layer, slots)


def runner_slots(runner, seq, n):
    return slots_of(runner.block_manager, runner._rows[seq.seq_id], n, runner.device)


def turned(runner, x, w, n):
    """Heads normed and turned as the runner's kernel of its kind of pool rounds them: the 8-bit path once, the others
    (and the reference) the norm, the tables and the result."""
    model, eps = runner.model, runner.shape.rms_norm_eps
    if not isinstance(runner.kv_cache, PagedKVCacheFp8):
        return _head_norm_rope(x, w, model.cos[:n], model.sin[:n], eps)
    y = x.double()
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    angle = torch.arange(n, device=x.device).double()[:, None, None] * model.inv_freq
    a, b = y.chunk(2, dim=-1)
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], dim=-1).to(torch.bfloat16)


def logits_over_pool(runner, seq):
    """The last position's logits of the runner's model in torch, attending over the rows that its pool holds."""
    model, s = runner.model, runner.model.shape
    tokens = seq.token_ids().to(runner.device)
    n = tokens.numel()
    slots = runner_slots(runner, seq, n)
    x = model.embed[tokens]
    for i, layer in enumerate(model.layers):
        h = _rms_norm(x, layer.in_norm, s.rms_norm_eps)
        qkv = F.linear(h, layer.qkv).view(n, -1, s.head_dim)
        q = turned(runner, qkv[:, :s.num_heads], layer.q_norm, n)
        k, v = held_rows(runner, i, slots)
        if i == 0 and isinstance(runner.kv_cache, PagedKVCacheFp8):  # what was stored is the first layer's own rows
            own = (turned(runner, qkv[:, s.num_heads:s.num_heads + s.num_kv_heads], layer.k_norm, n),
                   qkv[:, s.num_heads + s.num_kv_heads:])
            for got, want in zip((k, v), own):
                want = want.float()
                # half a step of the code, or of its unit's least (2^-17 of the unit's largest, again each time that
                # the exponent rises: below 2^-13 in all); bf16 rows differ by 2^-7 of their largest between matmuls
                tol = want.abs() * 2.0 ** -4 + want.abs().amax() * 2.0 ** -13 + want.abs().amax(-1, True) * 2.0 ** -6
                assert bool(((got.float() - want).abs() <= tol).all())
        attn, _ = orc.attention(q, k.double(), v.double(), s.head_dim ** -0.5)
        x = x + F.linear(attn.reshape(n, -1).to(torch.bfloat16), layer.o)
        h = _rms_norm(x, layer.post_norm, s.rms_norm_eps)
        gate, up = F.linear(h, layer.gate_up).chunk(2, dim=-1)
        x = x + F.linear(F.silu(gate) * up, layer.down)
    return _rms_norm(x, model.final_norm, s.rms_norm_eps)[-1].float() @ model.embed.float().T


def greedy(runner, seqs, what):
    for seq in seqs:
        logits = logits_over_pool(runner, seq)
        assert float(logits[seq.next_token_id]) >= float(logits.max()) - LOGIT_TOL, f"{what}: seq {seq.seq_id}"


def prompts(lengths, first_id, seed=11):
    g = torch.Generator().manual_seed(seed)
    return [Seq(first_id + i, torch.randint(0, 512, (n,), generator=g)) for i, n in enumerate(lengths)]


def test_step_runner_over_an_8_bit_cache(cuda_device):
    runner = StepRunner(SHAPE, cuda_device, max_model_len=1024, num_blocks=64, block_size=128, max_num_seqs=8,
                        enable_prefix_cache=True, decode_graph_batch_sizes=[1, 2, 4], seed=3, kv_cache_dtype="fp8")
    try:
        a, b, c, tail = prompts((300, 129, 60, 40), 10)
        runner.prepare_sequences([a, b, c])
        runner.prefill([a, b, c])
        greedy(runner, [a, b, c], "prefill")
        d = Seq(13, torch.cat([a.prompt_token_ids[:256], tail.prompt_token_ids]))
        runner.prepare_sequences([d])
        assert d.cached_prefix_len == 256
        runner.prefill([d])
        greedy(runner, [d], "prefill (prefix hit)")
        for step in range(3):
            runner.decode([a, b, c, d])
            greedy(runner, [a, b, c, d], f"decode bs4 step {step}")
        runner.free_seq(c)
        for step in range(2):
            runner.decode([a, b, d])  # no graph of three
            greedy(runner, [a, b, d], f"decode bs3 step {step}")
        stats = runner.decode_graph_stats()
        assert stats["captures"] == 1 and stats["replays"] == 3 and stats["fallbacks"] == 2
    finally:
        runner.release()


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
def test_forks_and_compaction_between_steps(cuda_device, kind):
    """A sequence forked inside a block and at a block's end, its copies decoded apart; sequences freed, the pool
    compacted, and all of them decoded on (replayed graphs and eager steps), over rows that stayed bit for bit."""
    dev, bs = cuda_device, 128 if kind == "bf16" else 32  # the bf16 prefill takes blocks of 128
    runner = StepRunner(SHAPE, dev, max_model_len=1024, num_blocks=48, block_size=bs, max_num_seqs=8,
                        enable_prefix_cache=True, decode_graph_batch_sizes=[4], seed=3, kv_cache_dtype=kind)
    layers = range(SHAPE.num_layers)

    def held(seqs):
        return [held_rows(runner, i, runner_slots(runner, s, s.cache_position)) for s in seqs for i in layers]

    def same(before, after):
        assert all(torch.equal(x, y) for a, b in zip(before, after) for x, y in zip(a, b))

    try:
        gone, a, b = prompts((6 * bs + 8, 4 * bs, 2 * bs + 13), 20)
        runner.prepare_sequences([gone, a, b])
        runner.prefill([gone, a, b])
        c, d = Seq(30, b.prompt_token_ids), Seq(31, a.prompt_token_ids)
        before = held([b, a])
        runner.fork(b, c)                     # 2 blocks shared, the one of 13 rows copied
        runner.fork(a, d, next_token_id=7)    # 4 blocks, all shared
        assert c.next_token_id == b.next_token_id and d.next_token_id == 7
        same(before, held([c, d]))
        tables = runner.block_manager.block_tables
        ta, tb, tc, td = (tables[runner._rows[s.seq_id]] for s in (a, b, c, d))
        assert tc[:2] == tb[:2] and tc[2] != tb[2] and td == ta
        for step in range(3):
            if step == 1:
                c.next_token_id = 9           # the copies part
            runner.decode([a, b, c, d])
            greedy(runner, [a, b, c, d], f"forked, step {step}")
        runner.free_seq(gone)
        waiting = Seq(40, torch.cat([gone.prompt_token_ids[:2 * bs], torch.tensor([3, 4])]))
        runner.prepare_sequences([waiting])
        assert waiting.cached_prefix_len == 2 * bs
        before = held([a, b, c, d])
        moved = runner.compact()
        live = len({x for s in (a, b, c, d) for x in tables[runner._rows[s.seq_id]]})
        assert moved > 0 and all(x < live for s in (a, b, c, d) for x in tables[runner._rows[s.seq_id]])
        same(before, held([a, b, c, d]))
        with pytest.raises(RuntimeError, match="prepared before compact"):
            runner.prefill([waiting])
        for step in range(2):
            runner.decode([a, b, c, d])
            greedy(runner, [a, b, c, d], f"compacted, step {step}")
        runner.decode([d, b])                 # eager: no graph of two
        greedy(runner, [d, b], "compacted, eager")
        hit = Seq(41, torch.cat([a.prompt_token_ids[:3 * bs], torch.tensor([5, 6, 7])]))
        runner.prepare_sequences([hit])
        assert hit.cached_prefix_len == 3 * bs  # its keys moved along
        runner.prefill([hit])
        greedy(runner, [hit], "prefix found after the compaction")
        for s in (a, b):
            runner.free_seq(s)
        runner.compact()
        runner.compact()                      # nothing left to move
        for step in range(2):
            runner.decode([c, d, hit])
            greedy(runner, [c, d, hit], f"compacted twice, step {step}")
        assert runner.decode_graph_stats()["captures"] == 1
        check_errors(dev)
    finally:
        runner.release()


def test_a_fork_without_a_free_block_leaves_the_runner_as_it_was(cuda_device):
    runner = StepRunner(SHAPE, cuda_device, max_model_len=128, num_blocks=2, block_size=32, max_num_seqs=2,
                        enable_decode_graph=False, seed=3, kv_cache_dtype="fp8")
    try:
        a, other, more = prompts((40, 3, 3), 50)
        runner.prepare_sequences([a])
        runner.prefill([a])
        with pytest.raises(RuntimeError, match="out of free blocks"):
            runner.fork(a, other)
        with pytest.raises(ValueError, match="in flight"):
            runner.fork(a, a)
        with pytest.raises(KeyError):
            runner.fork(other, more)
        runner.decode([a])
        greedy(runner, [a], "after the refusals")
        runner.free_seq(a)
        runner.prepare_sequences([other, more])
        runner.prefill([other, more])         # both rows and both blocks are there
        greedy(runner, [other, more], "the next sequences")
    finally:
        runner.release()


@pytest.mark.parametrize("remap", [True, False])
def test_device_tables_follow_a_compaction(cuda_device, remap):
    """The mirror renumbered in place, or sent again where remap() was not called: the host path's tables either way."""
    dev = cuda_device
    bm, host = (BlockManager(40, 16, d) for d in (dev, "cpu"))
    mirror = DeviceBlockTables(bm, 6, 16, dev)
    lens = [20, 70, 5, 33, 48, 1]
    for m in (bm, host):
        m.prepare_prefill_metadata(list(range(6)), lens, [0] * 6, [[]] * 6)
    steps = 0

    def step(slots):
        got = mirror.prepare_decode_metadata(slots, [lens[s] + steps for s in slots], 1)
        want = host.prepare_decode_metadata(slots, [lens[s] + steps for s in slots], 1)
        for name in ("block_tables", "context_lens", "slot_mapping"):
            assert torch.equal(getattr(got, name).cpu(), getattr(want, name).cpu()), name

    step([0, 1, 2, 3, 4, 5])
    for gone in ([1], [0, 4]):
        for m in (bm, host):
            for s in gone:
                m.free_slot(s)
        moved = [m.compact() for m in (bm, host)]
        assert moved[0] == moved[1] and moved[0]
        if remap:
            mirror.remap(moved[0])
        left = [s for s in range(6) if s in bm.block_tables]
        for _ in range(3):
            steps += 16
            step(left)
    assert int(mirror.error_word.item()) == 0


def test_step_runner_sizes_the_pool_from_memory(cuda_device):
    """With the same share of memory an 8-bit pool has nearly twice the blocks (512 / 258 bytes a row)."""
    counts = []
    for kind in ("bf16", "fp8"):
        free, total = torch.cuda.mem_get_info(cuda_device)
        share = (total - free + (2 << 30)) / total  # the model and about 2 GiB
        runner = StepRunner(SHAPE, cuda_device, max_model_len=256, memory_utilization=share, enable_decode_graph=False,
                            kv_cache_dtype=kind)
        counts.append(runner.num_blocks)
        runner.release()
        del runner
        torch.cuda.empty_cache()
    assert 1.85 < counts[1] / counts[0] < 2.1
