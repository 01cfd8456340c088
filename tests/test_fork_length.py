"""Forks of a sequence whose blocks' bookkeeping is ahead of what its rows hold, without a GPU.

A decode step does the allocator's bookkeeping (one more token) before its
kernels run: where it fails behind that, or because another sequence finds no
free block, the block manager counts a token that was never written, which the
next step writes. A fork counts what the sequence holds.
"""

from types import SimpleNamespace

import pytest

from nano_vllm_ascend_b200 import BlockManager
from nano_vllm_ascend_b200.step_runner import StepRunner, StepSequence

BS = 4


def manager(length, blocks=8):
    bm = BlockManager(blocks, BS, "cpu")
    bm.prepare_prefill_metadata([0], [length], [0], [[]])
    return bm


@pytest.mark.parametrize("held", [1, 3, 4, 5, 7, 8])
@pytest.mark.parametrize("ahead", [0, 1, 4])
def test_a_fork_of_the_first_tokens(held, ahead):
    bm = manager(held + ahead)
    pairs = bm.fork(0, 1, held)
    a, b = bm.block_tables[0], bm.block_tables[1]
    full = held // BS
    assert b[:full] == a[:full] and bm.seq_lens[1] == held
    assert pairs == ([(a[full], b[full])] if held % BS else []) and len(b) == full + len(pairs)
    slots = bm.prepare_decode_metadata([0, 1], [held, held], 1).slot_mapping.tolist()
    assert slots[0] != slots[1]


@pytest.mark.parametrize("length", [-1, 6])
def test_a_fork_of_tokens_that_are_not_there_is_refused(length):
    bm = manager(5)
    free = bm.free_block_ids
    with pytest.raises(ValueError, match=f"{length} tokens of slot 0, which has 5"):
        bm.fork(0, 1, length)
    assert bm.free_block_ids == free and 1 not in bm.block_tables


@pytest.mark.parametrize("held", [6, 7])
def test_a_runners_fork_behind_a_failed_step(held):
    """Both go on at the same position, each in a block of its own."""
    bm, copied = manager(held), []
    runner = StepRunner.__new__(StepRunner)
    runner.block_manager, runner._rows, runner._free_rows, runner._prepared_at = bm, {5: 0}, [1, 2], {}
    runner.kv_cache = SimpleNamespace(copy_blocks=lambda pairs: copied.extend(pairs))
    runner.device_tables = SimpleNamespace(forget=lambda row: None)
    seq, new = StepSequence(5, None), StepSequence(6, None)
    seq.set_prefill_result(next_token_id=11, prompt_len=held)
    bm.prepare_decode_metadata([0], [held], 1)  # a step's bookkeeping, and then no step
    runner.fork(seq, new)
    assert new.cache_position == held and new.next_token_id == 11
    assert copied == [(bm.block_tables[0][1], bm.block_tables[1][1])]
    slots = bm.prepare_decode_metadata([0, 1], [held, held], 1).slot_mapping.tolist()
    assert slots[0] != slots[1]
