"""A decoder with a sliding window and visible first tokens through the engine: against a plain restatement in 64 bits, with pages given back
behind the window, forks of running sequences and filtered sampling, one by one and together."""
import itertools
import json
import os
import subprocess
import sys

import pytest
import torch

from engine_helpers import write_model

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=97, context_length=1024, d_model=256, num_layers=2, num_heads=4, num_kv_heads=2, d_ff=96, attention_type="GQA",
           use_moe=False, attention_window=20, attention_first=3)


def weights(cfg=CFG):
    from llm_from_scratch_b200.model import ModelConfig, init_reference_order
    return init_reference_order(ModelConfig.from_dict(cfg), 4)


def engine(cfg=CFG, dtype=torch.float32, eager=True, blocks=256, **kw):
    from llm_from_scratch_b200.engine import Sequence
    from llm_from_scratch_b200.engine.llm_engine import LLMEngine
    Sequence.counter = itertools.count()
    return LLMEngine(dict(model=cfg, weights=weights(cfg), dtype=dtype, block_size=16, max_num_sequences=16, max_num_batched_tokens=2048,
                          max_cached_blocks=blocks, eos=-1, enforce_eager=eager, device="cuda:0", max_model_length=1024, **kw))


def restate(tokens, w, cfg=CFG):
    """Logits [n, vocab] of a token list, in 64 bits and without a cache."""
    w = {k: v.double() for k, v in w.items()}
    n, H, G = len(tokens), cfg["num_heads"], cfg["num_kv_heads"]
    hd = cfg["d_model"] // H
    eps = float(torch.finfo(torch.float32).eps)
    rms = lambda x, e, g: g * x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + e)
    lin = lambda x, name: x @ w[name + ".weight"].t() + w[name + ".bias"]
    angle = torch.arange(n)[:, None].double() / 10000.0 ** (torch.arange(0, hd, 2).double() / hd)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    gap = torch.arange(n)[:, None] - torch.arange(n)[None]
    hidden = (gap < 0) | ((gap >= cfg["attention_window"]) & (torch.arange(n)[None] >= cfg["attention_first"]))
    x = w["token_embeddings.weight"][torch.tensor(tokens)]
    for i in range(cfg["num_layers"]):
        a, f = f"layers.{i}.att", f"layers.{i}.ffn"
        h = rms(x, 1e-5, w[f"layers.{i}.att_norm.weight"])
        q = turn(rms(lin(h, a + ".q_proj"), eps, w[a + ".q_norm.weight"]).view(n, H, hd))
        k = turn(rms(lin(h, a + ".k_proj"), eps, w[a + ".k_norm.weight"]).view(n, G, hd)).repeat_interleave(H // G, 1)
        v = lin(h, a + ".v_proj").view(n, G, hd).repeat_interleave(H // G, 1)
        s = torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5
        s = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
        x = x + lin(torch.einsum("hij,jhd->ihd", s, v).reshape(n, -1), a + ".output_proj")
        h = rms(x, 1e-5, w[f"layers.{i}.ffn_norm.weight"])
        x = x + lin(torch.nn.functional.silu(lin(h, f + ".w1")) * lin(h, f + ".w3"), f + ".w2")
    return lin(rms(x, 1e-5, w["final_norm.weight"]), "lm_head")


PROMPTS = [[(7 * i + j * j) % 97 for j in range(n)] for i, n in enumerate([1, 5, 40, 70, 16, 33])]
SLACK = {torch.float32: 1e-3, torch.bfloat16: 0.1}       # of a logit, in units of the logits' spread: fp32 as in the engine's other tests


def follow(seq, w, dtype, keep=1):
    """Every generated token is among the ``keep`` best of the restatement, up to the slack."""
    logits = restate(seq.token_ids, w)[seq.num_prompt_tokens - 1:-1]
    chosen = logits.gather(1, torch.tensor(seq.completion_token_ids)[:, None])[:, 0]
    kth = logits.topk(keep, -1).values[:, -1]
    assert (kth - chosen).max() <= SLACK[dtype] * logits.std()


def finish(eng, seqs):
    from llm_from_scratch_b200 import ops
    while not eng.is_finished():
        _, n, _ = eng.step()
        assert n
    ops.check_status()
    return [s.completion_token_ids for s in seqs]


def greedy(n):
    from llm_from_scratch_b200.engine import SamplingParams
    return SamplingParams(temperature=0.0, max_tokens=n + 1, ignore_eos=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eager", [True, False])
def test_streams_follow_the_restatement(eager, dtype):
    eng, w = engine(dtype=dtype, eager=eager), weights()
    seqs = [eng.add_request(p, greedy(60)) for p in PROMPTS]
    finish(eng, seqs)
    for s in seqs:
        assert len(s.completion_token_ids) == 60
        follow(s, w, dtype)
    again = [eng.add_request(p, greedy(20)) for p in PROMPTS]       # prompts whose blocks are cached, some given back in between
    assert [x[:20] for x in finish(eng, again)] == [s.completion_token_ids[:20] for s in seqs] or dtype == torch.bfloat16
    for s in again:
        follow(s, w, dtype)
    eng.exit()


def test_several_steps_per_decision():
    eng, w = engine(eager=False, decode_window=8), weights()
    seqs = [eng.add_request(p, greedy(70)) for p in PROMPTS]
    finish(eng, seqs)
    for s in seqs:
        follow(s, w, torch.float32)
    eng.exit()


@pytest.mark.parametrize("eager", [True, False])
def test_a_pool_far_smaller_than_the_context(eager):
    """300 tokens at 16 a block in a pool of 8 blocks: only what the window and the first tokens need stays."""
    eng, w = engine(eager=eager, blocks=8), weights()
    seq = eng.add_request(PROMPTS[2], greedy(260))
    finish(eng, [seq])
    assert len(seq.token_ids) == 300
    follow(seq, w, torch.float32)
    assert eng.scheduler.block_manager.num_free_blocks == 8
    eng.exit()


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("eager", [True, False])
def test_forks_continue_like_their_parent(eager, cut):
    """Greedy forks, forks that draw from the best token only, and forks of forks give the parent's continuation; the parent is not disturbed."""
    from llm_from_scratch_b200.engine import SamplingParams
    cfg = CFG if cut else dict(CFG, attention_window=0, attention_first=0)
    eng = engine(cfg, eager=eager)
    want = finish(eng, [eng.add_request(p, greedy(50)) for p in PROMPTS])
    eng = engine(cfg, eager=eager)
    seqs = [eng.add_request(p, greedy(50)) for p in PROMPTS]
    children = []
    for step in range(30):
        eng.step()
        if step in (1, 7, 15, 16, 25):
            i = step % len(seqs)
            new = eng.fork(seqs[i], 2)
            new += eng.fork(new[0], 1, SamplingParams(temperature=1.0, top_k=1, max_tokens=51, ignore_eos=True))
            new += eng.fork(new[1], 1, SamplingParams(temperature=2.0, top_p=1e-6, max_tokens=51, ignore_eos=True))
            children += [(c, i) for c in new]
            if len(eng.scheduler.running) > 14:
                break
    assert finish(eng, seqs) == want
    assert len(children) >= 8
    for c, i in children:
        assert c.completion_token_ids == want[i]
    assert eng.scheduler.block_manager.num_free_blocks == 256
    eng.exit()


def test_forks_of_latent_attention():
    cfg = dict(vocab_size=97, context_length=256, d_model=128, num_layers=2, num_heads=8, d_ff=96, use_moe=False, attention_type="MLA")
    from llm_from_scratch_b200.engine import SamplingParams
    eng = engine(cfg)
    want = finish(eng, [eng.add_request(p, greedy(30)) for p in PROMPTS[:3]])
    eng = engine(cfg)
    seqs = [eng.add_request(p, greedy(30)) for p in PROMPTS[:3]]
    for _ in range(6):
        eng.step()
    children = eng.fork(seqs[2], 3)
    assert finish(eng, seqs) == want and all(c.completion_token_ids == want[2] for c in children)
    eng.exit()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eager", [True, False])
def test_all_together(eager, dtype):
    """Several answers to each prompt: forked behind the prompt, drawn under filters of their own, past many windows, in a pool that holds
    no whole context."""
    from llm_from_scratch_b200.engine import SamplingParams
    torch.manual_seed(1)
    eng, w = engine(dtype=dtype, eager=eager, blocks=60), weights()
    sp = lambda **kw: SamplingParams(max_tokens=121, ignore_eos=True, **kw)
    seqs = [eng.add_request(p, sp(temperature=0.8, top_k=4)) for p in PROMPTS[:4]]
    eng.step()
    answers = [(s, 4) for s in seqs]
    answers += [(c, 2) for c in eng.fork(seqs[2], 2, sp(temperature=1.5, top_k=2, top_p=0.9))]
    answers += [(c, 97) for c in eng.fork(seqs[3], 2, sp(temperature=1.0, top_p=0.9, min_p=0.05))]
    answers += [(c, 1) for c in eng.fork(seqs[0], 1, sp(temperature=0.0))]
    finish(eng, seqs)
    for s, keep in answers:
        assert len(s.completion_token_ids) == 120
        logits = restate(s.token_ids, w)[s.num_prompt_tokens - 1:-1]
        chosen = logits.gather(1, torch.tensor(s.completion_token_ids)[:, None])[:, 0][1:]     # the first one is the parent's
        kth = logits.topk(keep, -1).values[1:, -1]
        assert (kth - chosen).max() <= SLACK[dtype] * logits.std()
    pairs = [(a.completion_token_ids, b.completion_token_ids) for a, b in ((answers[4][0], answers[5][0]), (answers[6][0], answers[7][0]))]
    assert all(a != b for a, b in pairs)                                                      # they draw on their own
    assert eng.scheduler.block_manager.num_free_blocks == 60
    eng.exit()


@pytest.mark.parametrize("options,keep", [(["--temperature", "0.8", "--top-k", "1"], 1), (["--temperature", "2", "--top-k", "3", "--top-p", "0.9", "--min-p", "0.01"], 3)])
def test_generate_command_line(tmp_path, options, keep):
    w = weights()
    write_model(tmp_path / "m", CFG, w)
    prompts = [PROMPTS[2], PROMPTS[4]]
    r = subprocess.run([sys.executable, "-m", "llm_from_scratch_b200", "generate", "--model", str(tmp_path / "m"), "--dtype", "float32",
                        "--max-tokens", "31", "--max-model-length", "1024", "--max-cached-blocks", "64", "--ignore-eos"] + options
                       + [" ".join(map(str, p)) for p in prompts],
                       capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]
    for prompt, line in zip(prompts, r.stdout.splitlines(), strict=True):
        got = json.loads(line)["token_ids"]
        logits = restate(prompt + got, w)[len(prompt) - 1:-1]
        assert len(got) == 30
        chosen = logits.gather(1, torch.tensor(got)[:, None])[:, 0]
        assert (logits.topk(keep, -1).values[:, -1] - chosen).max() <= SLACK[torch.float32] * logits.std()
