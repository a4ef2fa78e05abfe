"""``LLMEngine.fork`` makes all the continuations that it was asked for or none."""
import itertools

import pytest


class _Runner:
    def __init__(self, blocks):
        self.num_kv_blocks, self.copied, self.fails = blocks, [], False

    def run(self, seqs, is_prefill):
        return [s.num_tokens + 100 * s.seq_id for s in seqs]

    def copy_blocks(self, pairs):
        if self.fails:
            raise RuntimeError("the copy failed")
        self.copied += pairs

    def exit(self):
        pass


def engine(blocks, tokens=20, steps=2):
    from llm_from_scratch_b200.engine import SamplingParams, Sequence
    from llm_from_scratch_b200.engine.llm_engine import LLMEngine
    Sequence.counter, Sequence.reference_exact = itertools.count(), False
    eng = LLMEngine(dict(block_size=4, max_num_sequences=16, max_num_batched_tokens=512, eos=-1), runner=_Runner(blocks))
    seq = eng.add_request(list(range(tokens)), SamplingParams(max_tokens=30, ignore_eos=True))
    for _ in range(steps):
        eng.step()
    return eng, seq


def state(eng):
    s = eng.scheduler
    return [x.seq_id for x in s.running], [list(x.block_table) for x in s.running], list(s.block_manager.free_block_ids), \
        [b.ref_count for b in s.block_manager.blocks], s.block_manager.hash_to_block_id


@pytest.mark.parametrize("blocks", [6, 7, 9])
@pytest.mark.parametrize("n", [5, 8])
def test_a_pool_that_runs_out_midway_changes_nothing(blocks, n):
    eng, seq = engine(blocks)
    before = state(eng)
    with pytest.raises(IndexError, match="exhausted"):
        eng.fork(seq, n)
    assert state(eng) == before and not eng.model_runner.copied
    left = blocks - 6
    assert len(eng.fork(seq, left)) == left and len(eng.scheduler.running) == 1 + left      # what the pool covers
    assert len(eng.model_runner.copied) == left


def test_a_copy_that_fails_leaves_no_fork_behind():
    eng, seq = engine(12)
    running, tables, free, refs, _ = state(eng)
    eng.model_runner.fails = True
    with pytest.raises(RuntimeError, match="copy failed"):
        eng.fork(seq, 3)
    now = state(eng)
    assert now[:2] == (running, tables) and sorted(now[2]) == sorted(free) and now[3] == refs
    eng.model_runner.fails = False
    a, b = eng.fork(seq, 2)
    while not eng.is_finished():
        assert eng.step()[1]
    assert len(a.token_ids) == len(b.token_ids) == len(seq.token_ids) and eng.scheduler.block_manager.num_free_blocks == 12


def test_forks_of_sequences_that_do_not_run_are_refused():
    eng, seq = engine(12, steps=0)
    with pytest.raises(ValueError, match="running"):
        eng.fork(seq, 2)
    assert eng.fork(seq, 0) == []
    while not eng.is_finished():
        eng.step()
    with pytest.raises(ValueError, match="running"):
        eng.fork(seq)
    assert eng.scheduler.block_manager.num_free_blocks == 12
