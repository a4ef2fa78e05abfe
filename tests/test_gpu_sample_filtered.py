"""``ops.sample_filtered`` against its definition in 64 bits on the host: the tokens have to be the same."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def definition(x, u, t, k, p, floor):
    """The token of one row (fp64 array), from the definition."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not t > 0 or x.max() == -np.inf:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore", over="ignore"):
        e = (x - x.max()) / t
    w = np.where(x == x.max(), 1.0, np.exp(np.where(np.isnan(e), -np.inf, e)))
    rank = np.argsort(-x, kind="stable")
    if 0 < k < len(rank):
        rank = rank[:k]
    if p < 1:
        sums = np.cumsum(w[rank])
        rank = rank[:max(1, int(np.searchsorted(sums, p * sums[-1], side="left")) + 1)]
    rank = np.sort(rank[w[rank] >= min(floor, 1.0)])
    sums = np.cumsum(w[rank])
    at = min(int(np.searchsorted(sums, max(u, 0.0) * sums[-1], side="right")), int(np.flatnonzero(w[rank])[-1]))
    return int(rank[at])


def expect(logits, u, t, k=None, p=None, m=None):
    x = logits.double().cpu().numpy()
    at = lambda v, i, off: off if v is None else v[i].item()
    return torch.tensor([definition(x[i], u[i].item(), t[i].item(), at(k, i, 0), at(p, i, 1.0), at(m, i, 0.0)) for i in range(x.shape[0])])


def call(logits, u, t, k=None, p=None, m=None, **kw):
    from llm_from_scratch_b200 import ops
    return ops.sample_filtered(logits.cuda(), *(None if x is None else x.cuda() for x in (u, t, k, p, m)), **kw).cpu()


def rows(n, vocab, dtype, seed, spread=(0.5, 8.0)):
    g = torch.Generator().manual_seed(seed)
    scale = spread[0] + (spread[1] - spread[0]) * torch.rand(n, 1, generator=g)
    return (torch.randn(n, vocab, generator=g) * scale).to(dtype), torch.rand(n, generator=g), 0.3 + 1.5 * torch.rand(n, generator=g), g


def filters(n, vocab, g, most):
    """Per row each filter on or off."""
    on = lambda: torch.rand(n, generator=g) < 0.6
    k = torch.where(on(), torch.randint(1, most + 1, (n,), generator=g), 0).int()
    p = torch.where(on(), torch.rand(n, generator=g), 1.0)
    m = torch.where(on(), 0.2 * torch.rand(n, generator=g), 0.0)
    return k, p, m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,most", [(5, 1, 1), (9, 2, 2), (17, 31, 31), (40, 100, 200), (64, 1000, 50), (33, 4097, 4000), (16, 32000, 1000),
                                          (3, 32001, 32001), (2, 131072, 100000), (300, 777, 20)])
def test_filters(n, vocab, most, dtype):
    x, u, t, g = rows(n, vocab, dtype, vocab)
    k, p, m = filters(n, vocab, g, most)
    for kk, pp, mm in ((k, p, m), (k, None, None), (None, p, None), (None, None, m), (None, None, None), (k, p, None)):
        assert torch.equal(call(x, u, t, kk, pp, mm), expect(x, u, t, kk, pp, mm))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [50, 3000, 40000])
def test_flat_rows(vocab, dtype):
    """Rows whose nucleus holds most of the vocabulary."""
    x, u, t, g = rows(12, vocab, dtype, 5, spread=(0.01, 1.0))
    k, p, m = filters(12, vocab, g, vocab)
    assert torch.equal(call(x, u, t, k, p, m), expect(x, u, t, k, p, m))
    p = torch.full((12,), 0.999)
    assert torch.equal(call(x, u, t, None, p, None), expect(x, u, t, None, p, None))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,levels", [(64, 1), (1000, 1), (1000, 3), (33000, 1), (33000, 4)])
def test_equal_logits_count_in_the_order_of_their_tokens(vocab, levels, dtype):
    g = torch.Generator().manual_seed(vocab + levels)
    n = 24
    x = torch.randint(0, levels, (n, vocab), generator=g).to(dtype)
    u, t = torch.rand(n, generator=g), torch.full((n,), 0.7)
    k, p, m = filters(n, vocab, g, vocab)
    assert torch.equal(call(x, u, t, k, p, m), expect(x, u, t, k, p, m))
    # all equal: whole weights, so that every border is exact: u in steps of 1 / 8 and p of 1 / 4
    x = torch.full((n, vocab), -2.5).to(dtype)
    u, p = (torch.arange(n) % 8).float() / 8, (1 + torch.arange(n) % 4).float() / 4
    assert torch.equal(call(x, u, t, None, p, None), expect(x, u, t, None, p, None))
    one = torch.ones(n, dtype=torch.int32)
    assert (call(x, u, t, one, None, None) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [10, 5000, 70000])
def test_edges_of_the_numbers(vocab, dtype):
    """Infinities and NaN among the logits, masked rows, extreme temperatures, random numbers and filters."""
    inf, nan = math.inf, math.nan
    x, _, _, g = rows(16, vocab, dtype, 11)
    x[0] = -inf                                           # nothing to draw
    x[1] = nan
    x[2, ::2] = -inf                                      # masked tokens
    x[3, 1::2] = nan
    x[4, [3, 7]] = inf                                    # two infinite logits share the weight
    x[5] = -inf
    x[5, 4] = -3.0                                        # a single token
    x[6] = torch.finfo(dtype).min                         # masks of the type's lowest value
    x[6, [2, 5]] = 1.0
    x[7] = torch.finfo(dtype).min
    x[8, :] = 0.0
    x[8, ::3] = -0.0                                      # equal to 0
    x[9] *= 1e4
    t = torch.ones(16)
    t[10], t[11], t[12], t[13] = 0.0, -1.0, 1e-30, 1e30
    for u in (0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24):
        u = torch.full((16,), u)
        for k, p, m in ((None, None, None), (3, None, None), (vocab, 1.0, 0.0), (-4, 2.0, -1.0), (None, 0.0, None), (None, 1e-20, None),
                        (None, 0.7, None), (None, None, 1.0), (None, None, 5.0), (vocab // 2, 0.5, 0.1), (2 ** 31 - 1, 0.999999, 1e-6)):
            row = lambda v, dt: None if v is None else torch.full((16,), v, dtype=dt)
            kk, pp, mm = row(k, torch.int32), row(p, torch.float32), row(m, torch.float32)
            got, want = call(x, u, t, kk, pp, mm), expect(x, u, t, kk, pp, mm)
            assert torch.equal(got, want), (k, p, m, u[0], torch.nonzero(got != want), got, want)


def test_strided_rows_output_and_neighbours():
    """Rows of a wider tensor, a given output, and that a row's token depends on nothing beside it; twice the same."""
    from llm_from_scratch_b200 import ops
    for dtype in DTYPES:
        for offset, vocab in ((0, 9000), (1, 9001), (3, 8998)):
            wide, u, t, g = rows(70, 9010, dtype, 2)
            k, p, m = (x.cuda() for x in filters(70, vocab, g, 500))
            wide, u, t = wide.cuda(), u.cuda(), t.cuda()
            part = wide[:, offset:offset + vocab]
            out = torch.full((70,), -1, dtype=torch.int64, device="cuda")
            assert ops.sample_filtered(part, u, t, k, p, m, out=out) is out
            assert torch.equal(out.cpu(), expect(part, u, t, k, p, m))
            alone = torch.cat([ops.sample_filtered(part[i:i + 1], u[i:i + 1], t[i:i + 1], k[i:i + 1], p[i:i + 1], m[i:i + 1]) for i in range(70)])
            assert torch.equal(out, alone)
            copy = part.contiguous()
            for _ in range(3):
                assert torch.equal(ops.sample_filtered(copy, u, t, k, p, m), out)
    assert ops.sample_filtered(wide[:0], u[:0], t[:0]).shape == (0,)


def test_captured_and_on_two_streams():
    from llm_from_scratch_b200 import ops
    sets = [[v.cuda() for v in rows(n, vocab, torch.float32, n)[:3]] for n, vocab in ((4, 50000), (200, 3000))]
    half = [torch.full((x[0].shape[0],), 0.8).cuda() for x in sets]
    call = lambda i: ops.sample_filtered(*sets[i], None, half[i], None)
    want = [call(0), call(1)]
    graphs = []
    for i in (0, 1, 0, 1):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(i)
        graphs.append((g, out, want[i], torch.cuda.Stream()))
    for _ in range(3):
        for g, out, _, s in graphs:
            with torch.cuda.stream(s):
                out.fill_(-1)
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for _, out, w, _ in graphs)


# ------------------------------------------------------------------------------------------------ many long rows: passes of separate launches
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,most,spread", [(65, 66000, 1000, (0.5, 8.0)), (64, 65536, 65536, (0.5, 8.0)), (33, 131072, 50000, (0.05, 3.0)),
                                                 (45, 100001, 60, (1.0, 12.0))])
def test_many_long_rows(n, vocab, most, spread, dtype):
    from llm_from_scratch_b200._lib import lib
    assert lib.b200_sample_filtered_workspace_bytes(n, vocab) > 0
    x, u, t, g = rows(n, vocab, dtype, vocab, spread)
    k, p, m = filters(n, vocab, g, most)
    t[3], u[5] = 0.0, 0.0
    for kk, pp, mm in ((k, p, m), (k, None, None), (None, p, None), (None, None, m), (None, None, None)):
        assert torch.equal(call(x, u, t, kk, pp, mm), expect(x, u, t, kk, pp, mm))
    p = torch.where(torch.arange(n) % 2 == 0, torch.full((n,), 0.995), torch.full((n,), 1e-3))
    assert torch.equal(call(x, u, t, None, p, None), expect(x, u, t, None, p, None))


@pytest.mark.parametrize("dtype", DTYPES)
def test_edges_of_the_numbers_in_many_long_rows(dtype):
    """What one form leaves to the other, between rows that it takes: greedy, masked, infinite, equal and flat rows."""
    inf, nan = math.inf, math.nan
    vocab, n = 66000, 66
    x, u, t, g = rows(n, vocab, dtype, 3)
    x[0] = -inf
    x[1] = nan
    x[2, ::2] = -inf
    x[3, 1::2] = nan
    x[4, [3, 50007]] = inf
    x[5] = -inf
    x[5, 65999] = -3.0
    x[6] = torch.finfo(dtype).min
    x[6, [2, 40000]] = 1.0
    x[7] = torch.finfo(dtype).min
    x[8] = 0.0
    x[9] = torch.randint(0, 3, (vocab,), generator=g).to(dtype)
    x[10] *= 1e4
    x[11:20] = torch.randint(0, 40, (9, vocab), generator=g).to(dtype)
    t[20], t[21], t[22], t[23] = 0.0, -1.0, 1e-30, 1e30
    u[24], u[25], u[26] = 0.0, 2.0 ** -24, 1 - 2.0 ** -24
    k, p, m = filters(n, vocab, g, vocab)
    for kk, pp, mm in ((k, p, m), (None, p, None), (k, None, None), (None, None, None), (torch.full((n,), 7, dtype=torch.int32), None, None),
                       (None, torch.full((n,), 0.5), torch.full((n,), 0.3))):
        got, want = call(x, u, t, kk, pp, mm), expect(x, u, t, kk, pp, mm)
        assert torch.equal(got, want), (torch.nonzero(got != want), got[got != want], want[got != want])


def test_many_long_rows_strided_captured_and_beside_each_other():
    """Unaligned rows of a wider tensor; the same tokens as row by row; two captured calls replayed on two streams."""
    from llm_from_scratch_b200 import ops
    for dtype in DTYPES:
        wide, u, t, g = [v.cuda() if torch.is_tensor(v) else v for v in rows(66, 66010, dtype, 2)]
        k, p, m = (v.cuda() for v in filters(66, 66000, g, 500))
        for offset in (0, 1, 6):
            part = wide[:, offset:offset + 66003]
            got = ops.sample_filtered(part, u, t, k, p, m)
            alone = torch.cat([ops.sample_filtered(part[i:i + 1], u[i:i + 1], t[i:i + 1], k[i:i + 1], p[i:i + 1], m[i:i + 1]) for i in range(66)])
            assert torch.equal(got, alone)
        graphs = []
        for args in ((k, p, m), (None, p, None)):
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            want = ops.sample_filtered(wide, u, t, *args)
            with torch.cuda.graph(graph):
                out = ops.sample_filtered(wide, u, t, *args)
            graphs.append((graph, out, want, torch.cuda.Stream()))
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, out, _, stream in graphs:
                with torch.cuda.stream(stream):
                    out.fill_(-1)
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _ in graphs)


# ------------------------------------------------------------------------------------------------ vocabularies beyond a cluster's shared memory
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabularies_beyond_a_cluster(dtype):
    n, vocab = 6, 500_001
    x, u, t, g = rows(n, vocab, dtype, 11)
    x[1] = -math.inf
    x[2, 17] = math.inf
    x[3, ::3] = math.nan
    t[4] = 0.0
    k, p, m = filters(n, vocab, g, 5000)
    for kk, pp, mm in ((k, p, m), (k, None, None), (None, p, None), (None, None, m), (None, None, None)):
        assert torch.equal(call(x, u, t, kk, pp, mm), expect(x, u, t, kk, pp, mm))


@pytest.mark.parametrize("n,vocab", [(70000, 33000), (20000, 131072)])
def test_rows_beyond_32_bits(n, vocab):
    """Logits behind 2^31 elements: the tokens of the same rows alone."""
    from llm_from_scratch_b200 import ops
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.empty(n, vocab, dtype=torch.bfloat16, device="cuda").normal_(generator=g).mul_(4)
    u, t, p = (torch.rand(n, generator=g, device="cuda") for _ in range(3))
    t += 0.3
    got = ops.sample_filtered(x, u, t, None, p, None)
    for part in (slice(0, 40), slice(n // 2, n // 2 + 40), slice(n - 40, n)):
        assert torch.equal(got[part], ops.sample_filtered(x[part], u[part], t[part], None, p[part], None))
