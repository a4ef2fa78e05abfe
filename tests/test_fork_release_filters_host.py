"""Forks of running sequences, blocks given back behind a window, and filters of requests: the host side, on both block managers."""
import random

import numpy as np
import pytest
import torch

from test_gpu_sample_filtered import expect, filters, rows


def scheduler(native, blocks=64, bs=4, cut=None, **kw):
    from llm_from_scratch_b200.engine import Sequence
    from llm_from_scratch_b200.engine.scheduler import Scheduler
    Sequence.block_size = bs
    s = Scheduler(max_num_sequences=16, max_num_batched_tokens=512, max_cached_blocks=blocks, block_size=bs, eos=-1, native_pool=native, **kw)
    s.attention_cut = cut
    return s


def add(s, tokens, n=40, **kw):
    from llm_from_scratch_b200.engine import SamplingParams, Sequence
    seq = Sequence(tokens, SamplingParams(max_tokens=n, ignore_eos=True, **kw))
    s.add_sequence(seq)
    return seq


def steps(s, n, token=lambda seq: seq.num_tokens + 100):
    for _ in range(n):
        batch, _ = s.schedule()
        s.postprocess(batch, [token(x) for x in batch])


@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("prompt", [1, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("ahead", [0, 1, 2, 3, 4, 5])
def test_fork(native, prompt, ahead):
    """A fork shares the full blocks, copies the one being written, and both go on without touching each other's."""
    s = scheduler(native)
    seq = add(s, list(range(prompt)))
    steps(s, 1 + ahead)
    free = s.block_manager.num_free_blocks
    child, copies = s.fork(seq)
    written, bs = seq.num_tokens - 1, 4
    full = written // bs
    assert child.token_ids == seq.token_ids and child.completion_token_ids == seq.completion_token_ids
    assert child.block_table[:full] == seq.block_table[:full] and len(child.block_table) == len(seq.block_table)
    assert not set(child.block_table[full:]) & set(seq.block_table[full:])
    assert copies == ([(seq.block_table[full], child.block_table[full])] if written % bs else [])
    assert s.block_manager.num_free_blocks == free - (len(seq.block_table) - full)
    refs = [b.ref_count for b in s.block_manager.blocks]
    assert all(refs[b] == 2 for b in child.block_table[:full]) and all(refs[b] == 1 for b in child.block_table[full:])
    steps(s, 9, token=lambda x: x.num_tokens + (100 if x is seq else 500))
    assert not set(child.block_table[full:]) & set(seq.block_table[full:])
    assert child.token_ids != seq.token_ids and len(child.token_ids) == len(seq.token_ids)
    while not s.is_finished():
        steps(s, 1)
    assert s.block_manager.num_free_blocks == 64 and not any(b.ref_count for b in s.block_manager.blocks)


@pytest.mark.parametrize("native", [False, True])
def test_fork_of_a_fork_its_parameters_and_refusals(native):
    from llm_from_scratch_b200.engine import SamplingParams
    from llm_from_scratch_b200.engine.scheduler import MixedScheduler
    s = scheduler(native, blocks=7)
    seq = add(s, list(range(6)), temperature=0.5, top_k=3)
    with pytest.raises(ValueError, match="running"):
        s.fork(seq)
    steps(s, 2)
    a, _ = s.fork(seq)
    b, copies = s.fork(a, SamplingParams(temperature=0.7, top_p=0.5))
    assert (a.temperature, a.filters, a.max_tokens) == (0.5, (3, 1.0, 0.0), 40) and b.filters == (0, 0.5, 0.0)
    assert b.block_table[0] == seq.block_table[0] and copies == [(a.block_table[1], b.block_table[1])]
    assert [x.ref_count for x in s.block_manager.blocks][seq.block_table[0]] == 3
    while s.block_manager.num_free_blocks:
        s.fork(seq)
    refs, running = [x.ref_count for x in s.block_manager.blocks], len(s.running)
    with pytest.raises(IndexError):
        s.fork(seq)
    assert [x.ref_count for x in s.block_manager.blocks] == refs and len(s.running) == running
    mixed = MixedScheduler(4, 64, 16, 4, -1)
    with pytest.raises(ValueError, match="mixed"):
        mixed.fork(seq)
    exact = scheduler(False, reference_exact=True)
    with pytest.raises(ValueError, match="reference"):
        exact.block_manager.fork(seq, a)
    with pytest.raises(ValueError, match="reference"):
        exact.block_manager.release(seq, 0, 1)


@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("window,first", [(1, 0), (4, 0), (5, 1), (8, 4), (9, 5), (13, 9), (100, 2)])
def test_blocks_behind_the_window_are_given_back(native, window, first):
    """No block that a later token sees goes; what stays is bounded by the window; hashes are those of a pool that gives nothing back."""
    bs = 4
    s, whole = scheduler(native, cut=(window, first)), scheduler(native)
    seq, twin = add(s, list(range(11)), n=60), add(whole, list(range(11)), n=60)
    for _ in range(50):
        batch, _ = s.schedule()
        whole.schedule()
        p = seq.num_tokens - 1                             # the token that this step computes
        for j in range(p + 1):
            if p - j < window or j < first:
                assert seq.block_table[j // bs] >= 0, (p, j)
        if p > 11:                                         # a step behind the prompt
            kept = sum(b >= 0 for b in seq.block_table)
            assert kept <= -(-first // bs) + -(-window // bs) + 4
        hashes = lambda x, y: [x.block_manager.blocks[b].hash for b in y.block_table if b >= 0]
        mine = [(i, h) for i, h in zip([i for i, b in enumerate(seq.block_table) if b >= 0], hashes(s, seq))]
        theirs = hashes(whole, twin)
        assert all(h == theirs[i] for i, h in mine)
        s.postprocess(batch, [p + 100])
        whole.postprocess([twin], [p + 100])
    while not s.is_finished():
        steps(s, 1)
    assert s.block_manager.num_free_blocks == 64 and not any(b.ref_count for b in s.block_manager.blocks)


@pytest.mark.parametrize("native", [False, True])
def test_windows_of_decode_steps_forks_and_preemption_with_blocks_given_back(native):
    """Random traces: every block is held by exactly the tables that name it, and all come back."""
    rng = random.Random(5)
    for trial in range(12):
        bs, window, first = 4, rng.choice([1, 6, 9]), rng.choice([0, 1, 6])
        s = scheduler(native, blocks=rng.choice([20, 40]), cut=(window, first))
        for _ in range(3):
            add(s, [rng.randrange(3) for _ in range(rng.randrange(1, 20))], n=rng.randrange(5, 40))
        for _ in range(300):
            if s.is_finished():
                break
            batch, prefill = s.schedule()
            if not batch:
                break
            k = 1 if prefill else s.plan_decode_window(batch, rng.choice([1, 3, 4]), 10 ** 6)
            if k > 1:
                s.postprocess_window(batch, [[rng.randrange(3) for _ in batch] for _ in range(k)])
            else:
                s.postprocess(batch, [rng.randrange(3) for _ in batch])
            if s.running and rng.random() < 0.1 and s.block_manager.num_free_blocks > 6 and len(s.running) < 6:
                s.fork(rng.choice(list(s.running)))
            held = {}
            for seq in s.running:
                for b in seq.block_table:
                    if b >= 0:
                        held[b] = held.get(b, 0) + 1
            refs = {b.block_id: b.ref_count for b in s.block_manager.blocks if b.ref_count}
            assert refs == held
        for seq in list(s.running):
            s.block_manager.deallocate(seq)
        assert not any(b.ref_count for b in s.block_manager.blocks)


def test_sharing_blocks_that_are_not_in_use_changes_nothing():
    from llm_from_scratch_b200._lib import lib
    pool = lib.b200_pool_create(4, 2)
    ids = np.array([lib.b200_pool_open_block(pool), 3], dtype=np.int32)
    refs = np.empty(4, dtype=np.int32)
    assert lib.b200_pool_share(pool, ids.ctypes.data, 2) == -1 and lib.b200_pool_share(pool, None, 1) == -1
    lib.b200_pool_snapshot(pool, None, refs.ctypes.data, None, None)
    assert refs.tolist() == [1, 0, 0, 0]
    assert lib.b200_pool_share(pool, ids.ctypes.data, 1) == 0
    lib.b200_pool_snapshot(pool, None, refs.ctypes.data, None, None)
    assert refs.tolist() == [2, 0, 0, 0]
    lib.b200_pool_destroy(pool)


def test_filters_of_a_request():
    from llm_from_scratch_b200.engine import SamplingParams, Sequence
    for bad in (dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=1.5), dict(top_p=float("nan")), dict(min_p=float("nan"))):
        with pytest.raises(ValueError):
            SamplingParams(**bad)
    assert Sequence([1], SamplingParams()).filters is None
    assert Sequence([1], SamplingParams(temperature=0.0, top_k=5)).filters is None          # greedy
    assert Sequence([1], SamplingParams(top_k=5, min_p=0.25)).filters == (5, 1.0, 0.25)
    from llm_from_scratch_b200.model import ModelConfig
    for bad in (dict(attention_window=-1), dict(attention_first=2), dict(attention_window=5, attention_type="MLA")):
        with pytest.raises(ValueError):
            ModelConfig(**bad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_tensor_form_of_the_filters(dtype):
    from llm_from_scratch_b200.utils.sampler import Sampler, filtered_tokens
    for n, vocab in ((9, 1), (30, 50), (12, 3000)):
        x, u, t, g = rows(n, vocab, dtype, vocab)
        k, p, m = filters(n, vocab, g, vocab)
        t[0] = 0.0
        x[1, ::2] = -torch.inf
        for args in ((k, p, m), (k, None, None), (None, p, None), (None, None, m), (None, None, None)):
            assert torch.equal(filtered_tokens(x, u, t, *args), expect(x, u, t, *args))
    s = Sampler(seed=3)
    first = s(x, t, k, p, m)
    assert torch.equal(Sampler(seed=3)(x, t, k, p, m), first)
    assert torch.equal(first, expect(x, Sampler(seed=3).uniforms(n, torch.device("cpu")), t, k, p, m))
