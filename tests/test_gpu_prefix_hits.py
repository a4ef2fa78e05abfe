"""Conversations that go on in a pool which has evicted blocks in the middle of what it still caches: the answers follow the 64-bit restatement."""
import pytest
import torch

from test_gpu_window_engine import CFG, SLACK, engine, finish, greedy, restate, weights

pytestmark = pytest.mark.gpu


def best(seq, w, cfg):
    """Every generated token is the restatement's best, up to the slack."""
    logits = restate(seq.token_ids, w, cfg)[seq.num_prompt_tokens - 1:-1]
    chosen = logits.gather(1, torch.tensor(seq.completion_token_ids)[:, None])[:, 0]
    assert (logits.max(-1).values - chosen).max() <= SLACK[torch.float32] * logits.std()


@pytest.mark.parametrize("eager", [True, False])
def test_behind_blocks_that_a_window_gave_back(eager):
    cfg = dict(CFG, attention_window=48)
    eng, w = engine(cfg, eager=eager, blocks=14), weights(cfg)
    one, two = (eng.add_request([(a * i + b) % 97 for i in range(40)], greedy(60)) for a, b in ((7, 0), (5, 3)))
    finish(eng, [one, two])
    finish(eng, [eng.add_request([(3 * i + 50) % 97 for i in range(40)], greedy(3))])
    for s in (one, two):
        eng.add_request(s.token_ids + [7, 8, 9], greedy(20))
    seqs, prefill = eng.scheduler.schedule()
    assert prefill and len(seqs) == 2
    logits = eng.model_runner.run_logits(seqs, True)
    for s, got in zip(seqs, logits.double().cpu()):
        want = restate(s.token_ids, w, cfg)[-1]
        assert (got - want).abs().max() <= SLACK[torch.float32] * want.std()
    eng.exit()


@pytest.mark.parametrize("eager", [True, False])
def test_behind_a_block_that_a_fork_sealed(eager):
    cfg = dict(CFG, attention_window=0, attention_first=0)
    eng, w = engine(cfg, eager=eager, blocks=20), weights(cfg)
    one, two = (eng.add_request([(a * i + b) % 97 for i in range(32)], greedy(100)) for a, b in ((7, 0), (5, 3)))
    while one.num_tokens < 48:
        eng.step()
    eng.fork(one, 1, greedy(29))
    finish(eng, [one, two])
    finish(eng, [eng.add_request([(3 * i + 50) % 97 for i in range(40)], greedy(3))])
    again = eng.add_request(one.token_ids + [7, 8, 9], greedy(20))
    finish(eng, [again])
    best(again, w, dict(cfg, attention_window=1 << 20))
    eng.exit()
