"""What the serving operators on cut contexts, sampled tokens and cache pages are timed on.

Three groups, as a serving engine uses them together: attention over a paged cache in which a query sees a sliding window and a few first
tokens (for prompts and portions of prompts, and for single tokens), the draw of the next token under temperature, top-k, top-p and
min-p, and the page operations behind it (copies for forks and moves, compaction of a pool).

``own`` chooses between the plain form, elementary tensor operations in fp32 (64 bits where a border is near), and the framework's calls.
A case names its ``kind``; the functions of a kind are collected in ``KINDS`` at the end of the file.  Lengths follow from the case alone
(``mix`` seeds them), values and the order of cache pages from the seed of ``prepare``.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    from llm_from_scratch_b200 import ops
    return ops


# ------------------------------------------------------------------------------------------------ shared pieces
def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _spread(rng: np.random.Generator, n: int, lo: int, hi: int) -> np.ndarray:
    """n lengths in [lo, hi], spread over their logarithm (from 0 on: over that of length + 1), the first one hi."""
    x = np.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1), size=n)) - 1
    x[0] = hi
    return np.clip(np.rint(x), lo, hi).astype(np.int64)


class _Values:
    """Seeded values on the GPU."""

    def __init__(self, seed: int):
        self.device = torch.device("cuda")
        self.gen = torch.Generator(device=self.device).manual_seed(seed)
        self.order = np.random.default_rng(seed)

    def normal(self, *shape, dtype=torch.bfloat16, std=1.0):
        out = torch.empty(shape, dtype=dtype, device=self.device)
        flat = out.view(-1)
        for at in range(0, flat.numel(), 1 << 28):
            part = flat[at:at + (1 << 28)]
            part.copy_(torch.randn(part.numel(), generator=self.gen, device=self.device).mul_(std))
        return out

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device=self.device)

    def put(self, values, dtype):
        return torch.as_tensor(np.asarray(values), dtype=dtype).to(self.device)


def _cut_tables(v: _Values, lens, starts, page: int):
    """Block tables over a shuffled pool that holds only the pages that something is seen of: of every sequence the first
    ``starts[i][0]`` tokens and those from ``starts[i][1]`` on; the entries of the others, which the engine has freed, are -1."""
    used = []
    for n, (first, low) in zip(lens, starts):
        p = np.arange(-(-int(n) // page))
        used.append((p * page < first) | ((p + 1) * page > low))
    total = int(sum(u.sum() for u in used)) + 4
    perm = v.order.permutation(total).astype(np.int32)
    tables = np.full((len(used), max([1] + [len(u) for u in used])), -1, dtype=np.int32)
    at = 0
    for i, u in enumerate(used):
        n = int(u.sum())
        tables[i, :len(u)][u] = perm[at:at + n]
        at += n
    return v.put(tables, torch.int32), tables, total


# ------------------------------------------------------------------------------------------------ window attention, single tokens
# A decode step of a layer with a sliding window whose first tokens stay visible.  The pages between them are freed.
def _decode_lens(case):
    return _spread(np.random.default_rng(case["mix"]), case["seqs"], case["lo"], case["hi"])


def _seen(n: int, case) -> int:
    """Keys that the token at position n - 1 sees."""
    return min(n, case["window"] + min(case["first"], max(n - case["window"], 0)))


def _prepare_decode(case, seed):
    v, dt, lens = _Values(seed), DTYPES[case["dtype"]], _decode_lens(case)
    tables, host, pages = _cut_tables(v, lens, [(case["first"], n - case["window"]) for n in lens], case["page"])
    pool = (pages, case["page"], case["kv_heads"], case["dim"])
    return dict(q=v.normal(len(lens), case["heads"], case["dim"], dtype=dt), k=v.normal(*pool, dtype=dt), v=v.normal(*pool, dtype=dt),
                tables=tables, lens=v.put(lens, torch.int64), host_lens=[int(n) for n in lens], scale=case["dim"] ** -0.5,
                window=case["window"], first=case["first"])


def _positions(n: int, low: int, first: int, device):
    """The positions below n that are among the first or not below ``low``, in order."""
    if low <= first:
        return torch.arange(n, device=device)
    return torch.cat([torch.arange(first, device=device), torch.arange(low, n, device=device)])


def _rows(pool, table, positions):
    page = pool.shape[1]
    return pool[table[positions // page].long(), positions % page]


def _plain_attention(q, k, v, visible, scale: float):
    """fp32 attention of q [n, H, d] over k, v [m, G, d] with the mask ``visible`` [n, m]; rows that see nothing are zeros."""
    n, H, d = q.shape
    G = k.shape[1]
    qs = q.float().view(n, G, H // G, d).permute(1, 2, 0, 3).reshape(G, -1, d)
    s = torch.bmm(qs, k.float().permute(1, 2, 0)).mul_(scale).view(G, H // G, n, -1)
    s = s.masked_fill(~visible, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), -math.inf)
    w = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(G, -1, w.shape[-1]), v.float().transpose(0, 1)).view(G, H // G, n, -1)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(2, 0, 1, 3).reshape(n, H, -1).to(q.dtype)


def _run_decode(s):
    if own:
        return _ops().window_decode(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["scale"], s["window"], s["first"])
    out = []
    for i, n in enumerate(s["host_lens"]):
        at = _positions(n, n - s["window"], s["first"], s["q"].device)
        visible = torch.ones(1, at.numel(), dtype=torch.bool, device=at.device)
        out.append(_plain_attention(s["q"][i:i + 1], _rows(s["k"], s["tables"][i], at), _rows(s["v"], s["tables"][i], at), visible, s["scale"]))
    return torch.cat(out)


def _exact_attention(q, pool_k, pool_v, table, first_position: int, scale, window, first):
    """64-bit attention of the rows of q, at positions first_position .., from the definition: key j is seen by the query at position p
    when 0 <= p - j and either p - j < window or j < first."""
    n, H, d = q.shape
    page, G = pool_k.shape[1], pool_k.shape[2]
    out = torch.zeros(n, H, d, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 25) // (H * min(first_position + n, window + first + 512)))
    for at in range(0, n, step):
        part = q[at:at + step].double()
        p = torch.arange(part.shape[0], device=q.device) + first_position + at
        j = torch.arange(int(p[-1]) + 1, device=q.device)
        j = j[(j < first) | (j > int(p[0]) - window)]
        if not j.numel():
            continue
        k = pool_k[table[j // page].long(), j % page].double().repeat_interleave(H // G, 1)
        v = pool_v[table[j // page].long(), j % page].double().repeat_interleave(H // G, 1)
        gap = p[:, None] - j[None, :]
        hidden = (gap < 0) | ((gap >= window) & (j[None, :] >= first))
        s = torch.matmul(part.transpose(0, 1), k.permute(1, 2, 0)) * scale                 # [H, rows, keys]
        s.masked_fill_(hidden, -math.inf)
        out[at:at + step] = torch.nan_to_num(torch.softmax(s, -1)).matmul(v.transpose(0, 1)).transpose(0, 1)
    return out


def _exact_decode(case, seed):
    s = _prepare_decode(case, seed)
    return torch.cat([_exact_attention(s["q"][i:i + 1], s["k"], s["v"], s["tables"][i], n - 1, s["scale"], s["window"], s["first"])
                      for i, n in enumerate(s["host_lens"])])


def _work_decode(case):
    lens, size = _decode_lens(case), 4 if case["dtype"] == "f32" else 2
    seen = sum(_seen(int(n), case) for n in lens)
    entries = sum(-(-_seen(int(n), case) // case["page"]) for n in lens)
    return {"bytes": seen * 2 * case["kv_heads"] * case["dim"] * size + entries * 4
            + len(lens) * (2 * case["heads"] * case["dim"] * size + 8),
            "flops": seen * 4 * case["heads"] * case["dim"]}


HEADS = [(16, 4, 64), (32, 8, 128), (16, 16, 128), (12, 4, 64), (8, 1, 128), (10, 2, 128)]


def _draw_decode(rng):
    heads, kv, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    window, hi = _log(rng, 16, 4096), _log(rng, 1, 16384)
    most = 256 * 4160 * 8 * 128 // (min(window + 16, hi) * kv * dim * (2 if dtype == "f32" else 1))
    return dict(kind="window_decode", dtype=dtype, heads=heads, kv_heads=kv, dim=dim, page=rng.choice([16, 16, 32, 64, 256]),
                seqs=min(_log(rng, 1, 256), max(1, most)), lo=min(hi, rng.choice([0, 1, hi // 4])), hi=hi, window=window,
                first=rng.choice([0, 1, 4, 5, 16, 64]), mix=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------------------------ window attention, prompts
# Prompts and portions of prompts (``before`` tokens are already cached) of the same layer; keys and values lie in the pages.
def _prompt_lens(case):
    rng = np.random.default_rng(case["mix"])
    return _spread(rng, case["seqs"], case["lo"], case["hi"]), _spread(rng, case["seqs"], case["before_lo"], case["before_hi"])


def _prepare_prompt(case, seed):
    v, dt = _Values(seed), DTYPES[case["dtype"]]
    new, before = _prompt_lens(case)
    tables, _, pages = _cut_tables(v, new + before, [(case["first"], b - case["window"] + 1) for b in before], case["page"])
    pool = (pages, case["page"], case["kv_heads"], case["dim"])
    cu = lambda x: np.concatenate([[0], np.cumsum(x)])
    return dict(q=v.normal(int(new.sum()), case["heads"], case["dim"], dtype=dt), k=v.normal(*pool, dtype=dt), v=v.normal(*pool, dtype=dt),
                tables=tables, cu_q=v.put(cu(new), torch.int32), cu_k=v.put(cu(new + before), torch.int32),
                new=[int(n) for n in new], before=[int(n) for n in before], longest=int(new.max()), scale=case["dim"] ** -0.5,
                window=case["window"], first=case["first"])


def _run_prompt(s):
    if own:
        return _ops().window_attention(s["q"], s["k"], s["v"], s["tables"], s["cu_q"], s["cu_k"], s["longest"], s["scale"], s["window"],
                                       s["first"])
    out, row, device = [s["q"][:0]], 0, s["q"].device
    for i, (n, before) in enumerate(zip(s["new"], s["before"])):
        for at in range(0, n, 512):                       # rows whose windows overlap share the gathered keys
            m = min(512, n - at)
            p = torch.arange(before + at, before + at + m, device=device)
            j = _positions(before + at + m, before + at - s["window"] + 1, s["first"], device)
            visible = (j[None] <= p[:, None]) & ((p[:, None] - j[None] < s["window"]) | (j[None] < s["first"]))
            out.append(_plain_attention(s["q"][row:row + m], _rows(s["k"], s["tables"][i], j), _rows(s["v"], s["tables"][i], j), visible,
                                        s["scale"]))
            row += m
    return torch.cat(out)


def _exact_prompt(case, seed):
    s = _prepare_prompt(case, seed)
    parts = s["q"].split(s["new"])
    return torch.cat([_exact_attention(q, s["k"], s["v"], s["tables"][i], b, s["scale"], s["window"], s["first"])
                      for i, (q, b) in enumerate(zip(parts, s["before"]))])


def _pairs(n: int, before: int, case) -> int:
    """(query, visible key) pairs of a portion."""
    p = np.arange(before + 1, before + n + 1, dtype=np.int64)
    return int(np.minimum(p, case["window"] + np.minimum(case["first"], np.maximum(p - case["window"], 0))).sum())


def _work_prompt(case):
    new, before = _prompt_lens(case)
    size = 4 if case["dtype"] == "f32" else 2
    low = np.maximum(before - case["window"] + 1, 0)
    keys = int(np.where(new > 0, new + before - low + np.minimum(low, case["first"]), 0).sum())
    pairs = sum(_pairs(int(n), int(b), case) for n, b in zip(new, before))
    return {"bytes": keys * 2 * case["kv_heads"] * case["dim"] * size + int(new.sum()) * 2 * case["heads"] * case["dim"] * size,
            "flops": pairs * 4 * case["heads"] * case["dim"]}


def _draw_prompt(rng):
    heads, kv, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    window, hi, before = _log(rng, 16, 4096), _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 16384)])
    tokens = 32768 if dtype == "bf16" else 4096
    return dict(kind="window_prompts", dtype=dtype, heads=heads, kv_heads=kv, dim=dim, page=rng.choice([16, 16, 32, 64, 256]),
                seqs=min(_log(rng, 1, 64), max(1, tokens // hi)), lo=min(hi, rng.choice([0, 1, hi // 4])), hi=hi, before_lo=before // 4,
                before_hi=before, window=window, first=rng.choice([0, 1, 4, 5, 16, 64]), mix=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------------------------ the next token
# Rows of logits that a few tokens stand out of, under filters that every request sets for itself ("mixed": some leave some off).
def _prepare_sample(case, seed):
    v, dt = _Values(seed), DTYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    logits = v.normal(rows, vocab, dtype=torch.float32, std=1.0)
    logits *= 1.5 + 2.5 * v.uniform(rows, 1)                              # flat and peaked rows
    hot = torch.randint(0, vocab, (rows, 8), generator=v.gen, device=v.device)
    logits.scatter_add_(1, hot, 10 * v.uniform(rows, 8))
    pick = lambda name, on, off: torch.where(v.uniform(rows) < (0.5 if "mixed" in case["filters"] else 1.0), on, torch.full_like(on, off)) \
        if name in case["filters"] else None
    k = torch.randint(1, case["top"] + 1, (rows,), generator=v.gen, device=v.device, dtype=torch.int32)
    return dict(logits=logits.to(dt), uniforms=v.uniform(rows), temperatures=0.5 + v.uniform(rows), top_k=pick("top-k", k, 0),
                top_p=pick("top-p", 0.5 + 0.49 * v.uniform(rows), 1.0), min_p=pick("min-p", 0.1 * v.uniform(rows), 0.0))


def _run_sample(s):
    if own:
        return _ops().sample_filtered(s["logits"], s["uniforms"], s["temperatures"], s["top_k"], s["top_p"], s["min_p"])
    x = s["logits"].double()                              # the borders of the filters and of the draw lie between sums of many tokens
    rows, vocab = x.shape
    t = s["temperatures"].double()[:, None]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)          # of equal logits the lower token first
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (torch.arange(vocab, device=x.device)[None] < k) | (k <= 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        mass = torch.where(keep, w, torch.zeros_like(w))
        before = torch.cumsum(mass, 1) - mass
        near = (before < p * mass.sum(1, keepdim=True)) | (p >= 1)
        near[:, 0] = True
        keep &= near
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    upto = torch.cumsum(mass, 1)                          # by token
    drawn = (upto <= s["uniforms"].double()[:, None] * upto[:, -1:]).sum(1)
    last = vocab - 1 - (mass.flip(1) > 0).to(torch.uint8).argmax(1)
    return torch.where(t[:, 0] > 0, torch.minimum(drawn, last), order[:, 0])


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    host = {k: None if x is None else x.cpu() for k, x in s.items()}
    logits = host["logits"].double().numpy()
    out = np.empty(case["rows"], dtype=np.int64)
    for r in range(case["rows"]):
        value = lambda name, off: off if host[name] is None else host[name][r].item()
        x, t = logits[r], value("temperatures", 0.0)
        if not t > 0:
            out[r] = int(np.argmax(x))
            continue
        w = np.exp((x - x.max()) / t)
        rank = np.argsort(-x, kind="stable")
        k, p, floor = value("top_k", 0), value("top_p", 1.0), value("min_p", 0.0)
        if 0 < k < len(rank):
            rank = rank[:k]
        if p < 1:
            sums = np.cumsum(w[rank])
            rank = rank[:max(1, int(np.searchsorted(sums, p * sums[-1], side="left")) + 1)]
        rank = np.sort(rank[w[rank] >= floor])
        sums = np.cumsum(w[rank])
        out[r] = rank[min(int(np.searchsorted(sums, host["uniforms"][r].item() * sums[-1], side="right")), len(rank) - 1)]
    return torch.from_numpy(out)


def _work_sample(case):
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 28, "flops": 4 * n}


def _draw_sample(rng):
    vocab = _log(rng, 100, 131072)
    names = [x for x in ("top-k", "top-p", "min-p") if rng.random() < 0.6]
    return dict(kind="sample", dtype=rng.choice(["bf16", "f32"]), rows=min(_log(rng, 1, 512), max(1, (1 << 25) // vocab)), vocab=vocab,
                filters=" ".join(names + rng.choice([[], ["mixed"]])), top=min(vocab, _log(rng, 1, 2000)))


# ------------------------------------------------------------------------------------------------ pages of a cache
# All layers' key and value pools share page ids.  A fork copies the page that its sequences go on writing; a compaction moves the pages in
# use to the front of the pools and renames them in the block tables.
def _pools(v: _Values, case):
    shape = (case["pages"], case["page"], case["kv_heads"], case["dim"])
    return [v.normal(*shape, dtype=DTYPES[case["dtype"]]) for _ in range(case["pools"])]


def _prepare_copy(case, seed):
    v = _Values(seed)
    pools, perm = _pools(v, case), v.order.permutation(case["pages"])
    n = min(case["copies"], case["pages"] // 2)
    source, target = perm[:n].copy(), perm[n:2 * n].copy()
    source[n // 2:] = source[:n - n // 2]                                   # pages that are forked more than once
    s = dict(pools=pools, source=v.put(source, torch.int32), target=v.put(target, torch.int32))
    if own:
        s["handle"] = _ops().PagePools(pools)
    return s


def _run_copy(s):
    if own:
        _ops().copy_pages(s["handle"], s["source"], s["target"])
        return s["pools"]
    source, target = s["source"].long(), s["target"].long()
    for pool in s["pools"]:
        pool[target] = pool[source]
    return s["pools"]


def _exact_copy(case, seed):
    s = _prepare_copy(case, seed)
    out = [pool.clone() for pool in s["pools"]]
    for a, b in zip(s["source"].tolist(), s["target"].tolist()):
        for old, new in zip(s["pools"], out):
            new[b].copy_(old[a])
    return out


def _page_bytes(case) -> int:
    return case["pools"] * case["page"] * case["kv_heads"] * case["dim"] * (4 if case["dtype"] == "f32" else 2)


def _work_copy(case):
    n = min(case["copies"], case["pages"] // 2)
    return {"bytes": ((n + n // 2 + n % 2) * _page_bytes(case)) + 8 * n, "flops": 0}


def _fork_tables(case) -> np.ndarray:
    """Tables of ``seqs`` sequences over at most ``live`` pages anywhere in the pool; every fourth sequence is a fork that shares its
    pages but the last with the one before it."""
    rng = np.random.default_rng(case["mix"])
    live = rng.permutation(case["pages"])[:min(case["live"], case["pages"])].astype(np.int32)
    width, rows, at = case["width"], [], 0
    for i in range(case["seqs"]):
        if i % 4 == 3 and len(rows[-1]) and at < len(live):
            rows.append(np.concatenate([rows[-1][:-1], live[at:at + 1]]))
            at += 1
            continue
        n = int(rng.integers(1, width + 1))
        rows.append(live[at:at + n])
        at += len(rows[-1])
    tables = np.full((case["seqs"], width), -1, dtype=np.int32)
    for i, r in enumerate(rows):
        tables[i, :len(r)] = r
    return tables


def _prepare_compact(case, seed):
    v = _Values(seed)
    pools, tables = _pools(v, case), _fork_tables(case)
    front = len(np.unique(tables[tables >= 0]))           # pages change places inside the front and behind it: as many move for every seed
    names = np.concatenate([v.order.permutation(front), front + v.order.permutation(case["pages"] - front)])
    s = dict(pools=pools, tables=v.put(np.where(tables >= 0, names[np.maximum(tables, 0)], -1), torch.int32))
    if own:
        s["handle"] = _ops().PagePools(pools)
    return s


def _run_compact(s):
    """Leaves the old tables and the moved pages' old places as they are, so that it can run again."""
    if own:
        r = _ops().compact_pages(s["handle"], s["tables"])
        return [r.block_tables, r.page_map, r.counts, *s["pools"]]
    tables, pages = s["tables"], s["pools"][0].shape[0]
    used = torch.zeros(pages, dtype=torch.bool, device=tables.device)
    used[tables[tables >= 0].long()] = True
    live = int(used.sum())
    holes = torch.nonzero(~used[:live])[:, 0]
    moved = torch.nonzero(used[live:])[:, 0] + live
    page_map = torch.where(used, torch.arange(pages, device=tables.device), -1)
    page_map[moved] = holes
    for pool in s["pools"]:
        pool[holes] = pool[moved]
    renamed = torch.where(tables >= 0, page_map[tables.clamp(min=0).long()], -1).int()
    return [renamed, page_map.int(), torch.tensor([live, moved.numel()], dtype=torch.int32, device=tables.device), *s["pools"]]


def _exact_compact(case, seed):
    s = _prepare_compact(case, seed)
    tables, pages = s["tables"].cpu().numpy(), case["pages"]
    used = sorted(set(tables[tables >= 0].tolist()))
    front = set(p for p in used if p < len(used))
    free = [p for p in range(len(used)) if p not in front]
    names = {p: p for p in front}
    names.update(zip([p for p in used if p >= len(used)], free))
    page_map = np.array([names.get(p, -1) for p in range(pages)], dtype=np.int32)
    out = [pool.clone() for pool in s["pools"]]
    for a, b in names.items():
        if a != b:
            for old, new in zip(s["pools"], out):
                new[b].copy_(old[a])
    renamed = np.where(tables >= 0, page_map[np.maximum(tables, 0)], -1).astype(np.int32)
    counts = np.array([len(used), len(free)], dtype=np.int32)
    return [torch.from_numpy(renamed), torch.from_numpy(page_map), torch.from_numpy(counts), *out]


def _work_compact(case):
    tables = _fork_tables(case)
    used = np.unique(tables[tables >= 0])
    return {"bytes": 2 * int((used >= len(used)).sum()) * _page_bytes(case) + 8 * tables.size + 4 * case["pages"], "flops": 0}


def _draw_pages(rng):
    """Page sizes of the configurations, pools of one layer to all layers."""
    heads, dim = rng.choice([(4, 64), (8, 128), (1, 128), (2, 64)])
    page = rng.choice([16, 16, 32, 64, 256])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    pools = rng.choice([1, 2, 7, 24, 32])
    size = pools * page * heads * dim * (4 if dtype == "f32" else 2)
    pages = min(_log(rng, 8, 8192), max(8, (1 << 31) // size))
    return dict(page=page, kv_heads=heads, dim=dim, dtype=dtype, pools=pools, pages=pages)


def _draw_copy(rng):
    shape = _draw_pages(rng)
    return dict(kind="copy_pages", **shape, copies=_log(rng, 1, max(2, shape["pages"] // 2)))


def _draw_compact(rng):
    shape = _draw_pages(rng)
    width = _log(rng, 1, 512)
    return dict(kind="compact_pages", **shape, live=_log(rng, 1, shape["pages"]), seqs=_log(rng, 1, 256), width=width,
                mix=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------------------------ the cases
# kind -> (prepare, run, exact, work, draw)
KINDS = {
    "window_decode": (_prepare_decode, _run_decode, _exact_decode, _work_decode, _draw_decode),
    "window_prompts": (_prepare_prompt, _run_prompt, _exact_prompt, _work_prompt, _draw_prompt),
    "sample": (_prepare_sample, _run_sample, _exact_sample, _work_sample, _draw_sample),
    "copy_pages": (_prepare_copy, _run_copy, _exact_copy, _work_copy, _draw_copy),
    "compact_pages": (_prepare_compact, _run_compact, _exact_compact, _work_compact, _draw_compact),
}


def listed() -> list[dict]:
    small, large = dict(heads=16, kv_heads=4, dim=64, page=16), dict(heads=32, kv_heads=8, dim=128, page=16)
    return [
        # one user's long conversation: a token against a window and the first tokens, where latency counts
        dict(name="window decode one", kind="window_decode", dtype="bf16", **large, seqs=1, lo=8192, hi=8192, window=1024, first=4, mix=0),
        # a full decode batch, conversations far longer than the window beside short ones
        dict(name="window decode batch", kind="window_decode", dtype="bf16", **large, seqs=256, lo=128, hi=16384, window=4096, first=4, mix=1),
        # the engine's fp32 mode, an ordinary batch
        dict(name="window decode fp32", kind="window_decode", dtype="f32", **small, seqs=64, lo=64, hi=2048, window=500, first=5, mix=2),
        # a mixed step: portions of prompts of a few to some hundred tokens behind what is cached of them
        dict(name="window portions", kind="window_prompts", dtype="bf16", **small, seqs=24, lo=1, hi=1000, before_lo=0, before_hi=8000,
             window=1024, first=16, mix=3),
        # long documents read at once, the largest prompts
        dict(name="window documents", kind="window_prompts", dtype="bf16", **large, seqs=4, lo=8192, hi=8192, before_lo=0, before_hi=0,
             window=4096, first=4, mix=4),
        # a single user's next token, all filters
        dict(name="sample one", kind="sample", dtype="bf16", rows=1, vocab=32000, filters="top-k top-p min-p", top=100),
        # an ordinary batch, every request with its own filters
        dict(name="sample batch", kind="sample", dtype="f32", rows=64, vocab=32000, filters="top-k top-p min-p mixed", top=1000),
        # the largest batch and vocabulary, nucleus sampling
        dict(name="sample large", kind="sample", dtype="f32", rows=256, vocab=131072, filters="top-p", top=1),
        # a few requests fork: the last page of each, in all layers
        dict(name="fork", kind="copy_pages", dtype="bf16", page=16, kv_heads=4, dim=64, pools=32, pages=2048, copies=8),
        # many beams change places
        dict(name="fork many", kind="copy_pages", dtype="bf16", page=16, kv_heads=8, dim=128, pools=16, pages=4096, copies=2000),
        # a small pool of one layer is compacted
        dict(name="compact small", kind="compact_pages", dtype="bf16", page=16, kv_heads=4, dim=64, pools=2, pages=500, live=200, seqs=16, width=13,
             mix=5),
        # the engine's pool is compacted after a burst, forks among its sequences
        dict(name="compact", kind="compact_pages", dtype="bf16", page=16, kv_heads=8, dim=128, pools=16, pages=4096, live=1800, seqs=100, width=45,
             mix=6),
    ]


def draw(rng) -> dict:
    return KINDS[rng.choice(list(KINDS))][4](rng)


def prepare(case: dict, seed: int):
    return case["kind"], KINDS[case["kind"]][0](case, seed)


def run(state):
    kind, s = state
    return KINDS[kind][1](s)


def exact(case: dict, seed: int):
    return KINDS[case["kind"]][2](case, seed)


def work(case: dict) -> dict:
    return KINDS[case["kind"]][3](case)
