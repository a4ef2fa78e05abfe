"""Prefix hits of both block managers, followed by the contents of the pages: every key that a step reads belongs to the sequence that reads
it, and the tables that captured decode steps keep on the device name the same pages, with blocks given back behind a window, forks, preemption and recomputed last blocks, in pools that evict all the time."""
import itertools
import random

import numpy as np
import pytest

BS = 4


class Trace:
    """A scheduler whose pages hold, for every slot, the tokens up to and with the one whose key was written there last."""

    def __init__(self, native, blocks, cut=None, max_tokens=512):
        from llm_from_scratch_b200.engine import Sequence
        from llm_from_scratch_b200.engine.scheduler import Scheduler
        Sequence.block_size, Sequence.counter, Sequence.reference_exact = BS, itertools.count(), False
        self.s = Scheduler(max_num_sequences=16, max_num_batched_tokens=max_tokens, max_cached_blocks=blocks, block_size=BS, eos=-1, native_pool=native)
        self.s.attention_cut = cut
        self.window, self.first = cut or (1 << 30, 0)
        from llm_from_scratch_b200.engine.metadata import DecodeBatchBuilder
        self.pages = {}
        self.builder = DecodeBatchBuilder(BS, 128, rows=8, device_rows=16)      # what captured decode steps take their tables from
        self.device = np.full((16, 128), -9, dtype=np.int32)
        self.log = []                       # what was scheduled, to compare two managers

    def add(self, tokens, n):
        from llm_from_scratch_b200.engine import SamplingParams, Sequence
        seq = Sequence(tokens, SamplingParams(max_tokens=n, ignore_eos=True))
        self.s.add_sequence(seq)
        return seq

    def fork(self, seq, n=None):
        from llm_from_scratch_b200.engine import SamplingParams
        child, copies = self.s.fork(seq, None if n is None else SamplingParams(max_tokens=n, ignore_eos=True))
        for a, b in copies:
            for o in range(BS):
                self.pages[b, o] = self.pages.get((a, o))
        return child

    def _compute(self, tokens, table, begin, end):
        for p in range(begin, end):
            self.pages[table[p // BS], p % BS] = tuple(tokens[:p + 1])
        for p in range(begin, end):
            for j in range(p + 1):
                if p - j < self.window or j < self.first:
                    assert table[j // BS] >= 0 and self.pages.get((table[j // BS], j % BS)) == tuple(tokens[:j + 1]), \
                        f"the token at {p} reads a key at {j} that is not its own"

    def _device_tables(self, batch):
        """The table on the device, kept up by patches, names the pages of all that a decode step sees."""
        ids, slots, lens, tables = (np.zeros(s, dtype=d) for s, d in ((16, np.int64), (16, np.int64), (16, np.int64), ((16, 128), np.int32)))
        patches = np.zeros((24, 3), dtype=np.int32)
        count = self.builder.build(batch, ids, slots, lens, tables, patches=patches)
        if count < 0:
            self.device[:len(batch)] = tables[:len(batch)]
        for pos, col, block in patches[:max(count, 0)]:
            self.device[pos, col] = block
        for i, x in enumerate(batch):
            p = x.num_tokens - 1
            assert slots[i] == x.block_table[p // BS] * BS + p % BS and lens[i] == p + 1
            for b in {j // BS for j in range(p + 1) if p - j < self.window or j < self.first}:
                assert self.device[i, b] == x.block_table[b]

    def step(self, token, steps=1):
        batch, prefill = self.s.schedule()
        self.log.append((prefill, [(x.seq_id, list(x.block_table), x.num_cached_tokens) for x in batch]))
        k = 1 if prefill else self.s.plan_decode_window(batch, steps, 10 ** 6)
        rows, tokens = [], [list(x.token_ids) for x in batch]
        if prefill:                         # every layer writes the keys of all prompts before it reads any
            self.builder.invalidate(batch)
            for x, t in zip(batch, tokens):
                for p in range(x.num_cached_tokens, x.num_tokens):
                    self.pages[x.block_table[p // BS], p % BS] = tuple(t[:p + 1])
        elif batch:
            self._device_tables(batch)
        for _ in range(k):
            for x, t in zip(batch, tokens):
                self._compute(t, x.block_table, x.num_cached_tokens if prefill else len(t) - 1, len(t))
            rows.append([token(x) for x in batch])
            for t, y in zip(tokens, rows[-1]):
                t.append(y)
        if k > 1:
            self.s.postprocess_window(batch, rows)
        else:
            self.s.postprocess(batch, rows[0])
        return batch

    def finish(self, token=lambda x: x.num_tokens + 100 * x.seq_id):
        while not self.s.is_finished():
            assert self.step(token)
        assert not any(b.ref_count for b in self.s.block_manager.blocks)


@pytest.mark.parametrize("native", [False, True])
def test_hits_end_at_the_first_miss(native):
    """A cached block behind one that was evicted is no hit: the tokens in front of it have to be computed."""
    from llm_from_scratch_b200.engine import BlockManager, NativeBlockManager, Sequence
    Sequence.block_size, Sequence.reference_exact = BS, False
    bm = (NativeBlockManager if native else BlockManager)(6, BS)
    a, other, b = Sequence(list(range(18))), Sequence(list(range(50, 57))), Sequence(list(range(18)))
    bm.allocate(a)
    table = list(a.block_table)
    bm.release(a, 1, 3)                                    # the middle is given back first
    bm.deallocate(a)
    bm.allocate(other)                                     # takes the block that was never in use and the later one of the middle
    assert table[2] in other.block_table and table[1] not in other.block_table
    bm.deallocate(other)
    bm.allocate(b)
    assert b.block_table[:2] == table[:2] and b.num_cached_tokens == 2 * BS
    assert len(set(b.block_table)) == 5                    # blocks 3 and on are cached too, but behind the miss


@pytest.mark.parametrize("native", [False, True])
def test_a_conversation_goes_on_behind_evicted_blocks(native):
    t = Trace(native, 30, cut=(8, 4))
    one, _ = t.add(list(range(12)), 60), t.add(list(range(200, 212)), 60)
    t.finish()
    t.add(list(range(300, 304)), 4)
    t.finish()
    again = t.add(one.token_ids + [7, 8, 9], 10)
    t.finish()
    assert len(again.completion_token_ids) == 9


FILLERS = (1, 3, 5, 9, 13, 16, 21, 29, 37, 45)


@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("length", range(9, 18))
@pytest.mark.parametrize("child_tokens", [3, 7, 11])
def test_the_parent_of_an_evicted_fork_goes_on(native, length, child_tokens):
    """Parent and fork seal the same tokens in blocks of their own; the fork's are evicted first."""
    for n in FILLERS:
        t = Trace(native, 16)
        parent = t.add(list(range(8)), 40)
        token = lambda x: 1000 + x.num_tokens
        while parent.num_tokens < length:
            t.step(token)
        t.fork(parent, child_tokens)
        t.finish(token)
        t.add(list(range(500, 500 + n)), 3)
        t.finish()
        t.add(parent.token_ids + [1, 2], 3)
        t.finish()


@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("length", range(9, 18))
def test_a_recomputed_last_block_that_is_evicted(native, length):
    """A prompt of whole blocks that are all cached computes its last one again in a block of its own, which becomes the hash's; when that
    one is evicted the first request's later blocks are still there."""
    for n in FILLERS:
        t = Trace(native, 16)
        first = t.add(list(range(8)), 24)
        while first.num_tokens < length:
            t.step(lambda x: x.num_tokens + 100)
        t.add(list(range(8)), 2)
        t.finish(lambda x: x.num_tokens + 100)
        t.add(list(range(700, 700 + n)), 3)
        t.finish()
        t.add(first.token_ids + [1, 2], 3)
        t.finish()


@pytest.mark.parametrize("cut", [(6, 0), (9, 3), None])
def test_preempted_sequences_read_their_own_keys(cut):
    """Sequences that are preempted in a pool too small for all of them find some of their blocks again; both managers do the same."""
    logs = []
    for native in (False, True):
        t = Trace(native, 14, cut=cut)
        for i in range(6):
            t.add([i] * (1 + 3 * i), 30)
        t.finish(lambda x: x.num_tokens % 3)
        logs.append(t.log)
    assert logs[0] == logs[1] and any(p for p, _ in logs[0][2:])      # something was read again


@pytest.mark.parametrize("forks", [False, True])
@pytest.mark.parametrize("cut", [None, (1, 0), (7, 0), (8, 4), (5, 6)])
def test_random_traces(cut, forks):
    """Requests of which some continue earlier ones or start like them, windows of decode steps, forks; both managers do the same."""
    for seed in range(25):
        logs = []
        for native in (False, True):
            rng = random.Random(1000 * seed + 7)
            t, ended = Trace(native, rng.choice([24, 30, 40]), cut=cut), []
            token = lambda x: (x.num_tokens * 7 + x.seq_id) % 5 if rng.random() < 0.5 else 0
            for _ in range(7):
                for _ in range(rng.randrange(1, 3)):
                    base = list(rng.choice(ended).token_ids) if ended and rng.random() < 0.6 else [rng.randrange(3) for _ in range(rng.randrange(1, 20))]
                    base = base[:rng.randrange(1, len(base) + 1)] if rng.random() < 0.3 else base
                    ended.append(t.add(base[:60] + [rng.randrange(3) for _ in range(rng.randrange(4))], rng.randrange(2, 25)))
                steps = rng.choice([1, 1, 3, 4])
                while not t.s.is_finished():
                    assert t.step(token, steps)
                    live = [x for x in t.s.running]
                    if forks and live and rng.random() < 0.15 and len(live) < 4 and t.s.block_manager.num_free_blocks > 3:
                        ended.append(t.fork(rng.choice(live)))
            logs.append(t.log)
        assert logs[0] == logs[1]
