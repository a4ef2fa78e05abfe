"""Forks under filters of their own in one batch: every drawn token is among those that its filters leave."""
import pytest
import torch

from test_gpu_window_engine import PROMPTS, SLACK, engine, finish, restate, weights

pytestmark = pytest.mark.gpu
T = 0.3
FILTERS = [dict(top_p=0.5), dict(min_p=0.3), dict(top_k=2), dict(top_p=0.9, min_p=0.2), dict(top_k=6, top_p=0.6), dict(top_k=9, top_p=0.8, min_p=0.25)]


def left(logits, delta, top_k=97, top_p=1.0, min_p=0.0):
    """Tokens that the filters may leave where every logit is off by up to ``delta``: weights are then off by a factor of e^(delta / T), and a
    token lies behind all those whose logits are higher by more than 2 delta."""
    out = torch.zeros_like(logits, dtype=torch.bool)
    f = torch.exp(2 * delta / T)
    for row, x in enumerate(logits):
        w = torch.exp((x - x.max()) / T)
        before = x[None] > x[:, None] + 2 * delta
        out[row] = (before.sum(1) < top_k) & ((before * w).sum(1) < top_p * f * w.sum()) & (w >= min_p / f)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eager", [True, False])
def test_drawn_tokens_are_among_those_left(eager, dtype):
    from llm_from_scratch_b200.engine import SamplingParams
    torch.manual_seed(3)
    eng, w = engine(dtype=dtype, eager=eager), weights()
    sp = lambda **kw: SamplingParams(temperature=T, max_tokens=81, ignore_eos=True, **kw)
    parents = [eng.add_request(p, sp()) for p in PROMPTS[2:4]]
    eng.step()
    forks = [(eng.fork(parents[i % 2], 1, sp(**f))[0], f) for i, f in enumerate(FILTERS + FILTERS[:4])]
    finish(eng, parents)
    out = 0
    for s, f in [(p, {}) for p in parents] + forks:
        logits = restate(s.token_ids, w)[s.num_prompt_tokens:-1]                 # the first token is the parent's
        drawn = torch.tensor(s.completion_token_ids[1:])[:, None]
        assert len(drawn) == 79
        for check in [f] if f else FILTERS:
            allowed = left(logits, SLACK[dtype] * logits.std(), **check)
            assert allowed.sum(1).double().mean() < 97 / 4
            if f:
                assert allowed.gather(1, drawn).all(), f
            else:
                out += int((~allowed.gather(1, drawn)).sum())
    assert out > 50                                                              # draws without filters leave these sets
    eng.exit()
