"""BlockManager.fork and compact, and what the pool classes refuse to copy, without a GPU.

A pool of token ids stands in for the rows: a script of random admissions
(over cached prefixes), decode steps, forks, releases and compactions keeps
every sequence's tokens readable through its table, counts references, and
finds the same prefixes with the native index as with the Python one.
"""

import random

import pytest
import torch

from nano_vllm_ascend_b200 import BlockManager, PagedKVCache, PagedKVCacheFp4, PagedKVCacheFp8
from nano_vllm_ascend_b200.paged_kv_cache import copy_pool_blocks

BS = 4


class World:
    def __init__(self, num_blocks, native):
        self.bm = BlockManager(num_blocks, BS, "cpu", native_prefix=native)
        self.pool = [[None] * BS for _ in range(num_blocks)]
        self.tokens = {}

    def put(self, slot, pos, token):
        self.pool[self.bm.block_tables[slot][pos // BS]][pos % BS] = token

    def copy(self, pairs):
        rows = [list(self.pool[s]) for s, _ in pairs]
        for (_, d), row in zip(pairs, rows):
            self.pool[d] = row

    def admit(self, slot, tokens):
        t = torch.tensor(tokens)
        full = len(tokens) // BS
        prefix = self.bm.find_longest_prefix_blocks(t, max_cache_blocks=(len(tokens) - 1) // BS)
        start = len(prefix) * BS
        self.bm.prepare_prefill_metadata([slot], [len(tokens) - start], [start], [prefix])
        for pos in range(start, len(tokens)):
            self.put(slot, pos, tokens[pos])
        self.bm.cache_full_blocks(slot=slot, token_ids=t, num_cached_blocks=len(prefix), num_full_blocks=full)
        self.tokens[slot] = list(tokens)
        return list(prefix)

    def step(self, slot, token):
        n = len(self.tokens[slot])
        self.bm.prepare_decode_metadata([slot], [n], 1)
        self.put(slot, n, token)
        self.tokens[slot].append(token)

    def fork(self, slot, new):
        self.copy(self.bm.fork(slot, new))
        self.tokens[new] = list(self.tokens[slot])

    def check(self):
        bm = self.bm
        assert sorted(bm.block_tables) == sorted(self.tokens)
        for slot, tokens in self.tokens.items():
            assert bm.seq_lens[slot] == len(tokens)
            got = [self.pool[bm.block_tables[slot][i // BS]][i % BS] for i in range(len(tokens))]
            assert got == tokens
        counts = [0] * bm.num_blocks
        for table in bm.block_tables.values():
            for b in table:
                counts[b] += 1
        assert counts == [b.ref_count for b in bm.blocks]
        free = bm.free_block_ids
        assert len(free) == len(set(free)) and set(free) == {b for b, c in enumerate(counts) if c == 0}


@pytest.mark.parametrize("seed", range(6))
def test_a_script_of_forks_and_compactions(seed):
    rng = random.Random(seed)
    worlds = [World(24, True), World(24, False)]
    stems = [[rng.randrange(9) for _ in range(13)] for _ in range(2)]
    moved = forked = hits = 0
    for step in range(300):
        slots = sorted(worlds[0].tokens)
        op = rng.choice(["admit", "step", "step", "step", "fork", "free", "compact"])
        fresh = next(s for s in range(20) if s not in slots)
        stem, pick = rng.choice(stems), rng.choice(slots) if slots else None
        tokens = stem[:rng.randrange(1, 14)] + [rng.randrange(9) for _ in range(rng.randrange(3))]
        seen = []
        for w in worlds:
            if op == "admit" and w.bm.num_free_blocks() >= 5:
                seen.append(w.admit(fresh, tokens))
                hits += bool(seen[-1])
            elif op == "step" and slots and w.bm.num_free_blocks():
                w.step(pick, step)
            elif op == "fork" and slots and w.bm.num_free_blocks():
                w.fork(pick, fresh)
                forked += 1
            elif op == "free" and slots:
                w.bm.free_slot(pick)
                del w.tokens[pick]
            elif op == "compact":
                pairs = w.bm.compact(w.copy)
                moved += len(pairs)
                live = sum(b.ref_count > 0 for b in w.bm.blocks)
                assert all((b.ref_count > 0) == (i < live) for i, b in enumerate(w.bm.blocks))
                seen.append(pairs)
            w.check()
        assert len(seen) < 2 or seen[0] == seen[1]
        for s in stems:
            found = [w.bm.find_longest_prefix_blocks(torch.tensor(s), 3) for w in worlds]
            assert found[0] == found[1]
            for w, blocks in zip(worlds, found):
                for i, b in enumerate(blocks):
                    assert w.pool[b] == s[i * BS:(i + 1) * BS]
    assert moved and forked and hits  # the script does reach all three


@pytest.mark.parametrize("length,copies", [(1, 1), (4, 0), (5, 1), (8, 0), (11, 1)])
def test_a_fork_shares_full_blocks_and_copies_the_rest(length, copies):
    w = World(8, True)
    w.admit(0, list(range(length)))
    pairs = w.bm.fork(0, 1)
    assert len(pairs) == copies
    a, b = w.bm.block_tables[0], w.bm.block_tables[1]
    assert len(a) == len(b) and a[:length // BS] == b[:length // BS] and a is not b
    assert not copies or (a[-1], b[-1]) == pairs[0] and a[-1] != b[-1]
    md = w.bm.prepare_decode_metadata([0, 1], [length, length], 1)
    assert len(set(md.slot_mapping.tolist())) == 2


def test_a_fork_that_cannot_be_made_changes_nothing():
    w = World(2, True)
    w.admit(0, list(range(5)))
    with pytest.raises(RuntimeError, match="out of free blocks"):
        w.bm.fork(0, 1)
    with pytest.raises(ValueError, match="slot 0 is in use"):
        w.bm.fork(0, 0)
    with pytest.raises(KeyError):
        w.bm.fork(7, 8)
    w.check()


def test_a_compaction_whose_copies_fail_changes_nothing():
    w = World(8, True)
    w.admit(0, [1, 2, 3, 4, 5])
    w.admit(1, [6, 7, 8])
    w.bm.free_slot(0)
    del w.tokens[0]

    def fails(pairs):
        raise RuntimeError("an earlier step's error")

    with pytest.raises(RuntimeError, match="earlier"):
        w.bm.compact(fails)
    w.check()
    assert w.bm.moves == 0 and w.bm.block_tables[1] == [2]
    assert w.bm.compact(w.copy) == [(2, 0)] and w.bm.moves == 1
    w.check()
    assert w.bm.compact(w.copy) == [] and w.bm.moves == 1


def test_a_moved_key_keeps_its_place_and_a_moved_over_one_goes():
    for native in (True, False):
        w = World(8, native)
        w.admit(0, [1, 2, 3, 4, 5])     # blocks 0 and 1
        w.admit(1, [9, 9, 9, 9, 9])     # 2, 3
        w.bm.free_slot(0)
        del w.tokens[0]
        assert w.bm.find_longest_prefix_blocks(torch.tensor([1, 2, 3, 4, 5]), 1) == [0]
        assert w.bm.compact(w.copy) == [(2, 0), (3, 1)]
        assert w.bm.find_longest_prefix_blocks(torch.tensor([1, 2, 3, 4, 5]), 1) == []
        assert w.bm.find_longest_prefix_blocks(torch.tensor([9, 9, 9, 9, 9]), 1) == [0]
        assert w.bm.blocks[2].block_hash is None and 2 in w.bm.free_block_ids


def test_index_refuses_blocks_out_of_range():
    index = BlockManager(4, BS, "cpu")._native
    for src, dst in ((-1, 0), (0, -1), (4, 0), (0, 4)):
        with pytest.raises((RuntimeError, ValueError), match="out of range"):
            index.move(src, dst)


def test_caches_refuse_copies():
    caches = [PagedKVCache(2, 4, 16, 2, 128, torch.bfloat16, "cpu"), PagedKVCacheFp4(2, 4, 16, 2, 128, "cpu"),
              PagedKVCacheFp8(2, 4, 16, 2, 128, "cpu")]
    for kv in caches:
        kv.copy_blocks([])
        kv.copy_blocks(torch.empty(0, 2, dtype=torch.int64))
        for pairs in ([(0, 4)], [(4, 0)], [(-2, 0)], [(0, -1)]):
            with pytest.raises(IndexError, match="in a pool of 4 blocks"):
                kv.copy_blocks(pairs)
        for pairs in ([(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], torch.tensor([(-1, 1), (-1, 1)])):
            with pytest.raises(ValueError, match="is also another copy's"):
                kv.copy_blocks(pairs)
        for pairs in ([0, 1], [(0, 1, 2)], [(0.5, 1)], [(True, False)]):
            with pytest.raises(ValueError, match="must be \\(source, destination\\)"):
                kv.copy_blocks(pairs)
    with caches[0].deferred_appends():
        caches[0]._pending[0] = ()
        with pytest.raises(RuntimeError, match="held back"):
            caches[0].copy_blocks([(0, 1)])
        caches[0]._pending.clear()
    copy_pool_blocks([caches[0].key_cache], [])
