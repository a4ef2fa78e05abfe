"""Attention over a sliding window and visible first tokens (``ops.window_attention``, ``ops.window_decode``) against its formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def formula(q, k, v, first_position, scale, window, first):
    """q [n, H, D] at positions first_position .. against keys 0 .. of one sequence, in 64 bits: (output, bound of its error per unit of the
    rounding of a weight, of a score).  Only visible keys enter, so the others may hold anything."""
    n, H, D = q.shape
    G, Dv = k.shape[1], v.shape[2]
    out, spread = torch.zeros(n, H, Dv, dtype=torch.float64), torch.zeros(n, H, Dv, dtype=torch.float64)
    sums = torch.zeros(n, H, 1, dtype=torch.float64)
    for i in range(n):
        p = first_position + i
        seen = [j for j in range(0, min(p + 1, k.shape[0])) if p - j < window or j < first]
        if not seen:
            continue
        kk, vv = k[seen].double().repeat_interleave(H // G, 1), v[seen].double().repeat_interleave(H // G, 1)
        s = torch.einsum("hd,jhd->hj", q[i].double(), kk) * scale
        w = torch.softmax(s, -1)
        out[i] = torch.einsum("hj,jhd->hd", w, vv)
        spread[i] = torch.einsum("hj,jhd->hd", w, vv.abs())
        # a score is a sum of D products and is scaled: each of its D + 2 roundings is off by 2^-24 of the sum of magnitudes (twice that
        # where a matrix unit cuts instead of rounding); the exponential of 2 units; the sums over the keys
        size = torch.einsum("hd,jhd->hj", q[i].double().abs(), kk.abs()).amax(-1) * scale
        sums[i, :, 0] = 2 * (size * (D + 4) * 2.0 ** -23 + 2.0 ** -21) + len(seen) * 2.0 ** -23
    return out, spread, sums


def check_close(got, want, spread, sums, dtype):
    """Errors of the scores and sums move the output by that share of sum w |v|, twice (numerator and denominator are in ``sums`` already); bf16
    weights are off by 2^-8 each, the output by 2^-8 (fp32: 2^-24) of itself."""
    half = torch.finfo(dtype).eps / 2
    bound = spread * sums + half * want.abs() * (1 + sums) + 1e-30
    if dtype == torch.bfloat16:
        bound = bound + half * spread * (1 + sums)
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= bound).all(), (err / bound).max().item()


def paged(lens, page, window, first, lows, gen, dtype, Hkv, D, Dv, spare=3, poison=False):
    """Pools and tables for contexts of these lengths; pages that no query sees are not in the pool: their entries are nonsense.  With
    ``poison`` every row that no query sees is NaN or infinite."""
    keep = [[p * page < min(first, n) or (p + 1) * page > low for p in range(-(-n // page))] for n, low in zip(lens, lows)]
    total = sum(map(sum, keep)) + spare
    ids = torch.randperm(total, generator=gen).tolist()
    bt = torch.full((len(lens), max([1] + [len(x) for x in keep]) + 1), -1, dtype=torch.int32)
    k, v = (torch.randn(total, page, Hkv, d, generator=gen).to(dtype) for d in (D, Dv))
    seen = torch.zeros(total, page, dtype=torch.bool)
    rows = []
    for i, n in enumerate(lens):
        kk, vv = torch.full((n, Hkv, D), math.nan, dtype=dtype), torch.full((n, Hkv, Dv), math.nan, dtype=dtype)
        for p, used in enumerate(keep[i]):
            bt[i, p] = ids.pop() if used else (-1, 10 ** 6, -7)[p % 3]
            if used:
                m = min(page, n - p * page)
                kk[p * page:p * page + m], vv[p * page:p * page + m] = k[bt[i, p], :m], v[bt[i, p], :m]
                for r in range(m):
                    seen[bt[i, p], r] = p * page + r < first or p * page + r >= lows[i]
        rows.append((kk, vv))
    if poison:
        k[~seen] = math.nan
        v[~seen] = torch.tensor([math.nan, math.inf, -math.inf]).to(dtype)[torch.arange(int((~seen).sum())) % 3][:, None, None]
    return k, v, bt, rows


HEADS = [(4, 4, 64, 64), (16, 4, 64, 64), (8, 2, 128, 128), (8, 1, 128, 128), (6, 2, 64, 64), (5, 1, 128, 128), (4, 2, 32, 32),
         (24, 1, 64, 64), (2, 1, 40, 72), (3, 3, 16, 300)]


def decode_case(lens, Hq, Hkv, D, Dv, page, window, first, dtype, seed=0, poison=True):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(len(lens), Hq, D, generator=gen).to(dtype)
    k, v, bt, rows = paged(lens, page, window, first, [max(0, n - window) for n in lens], gen, dtype, Hkv, D, Dv, poison=poison)
    want = [formula(q[i:i + 1], *rows[i], n - 1, D ** -0.5, window, first) for i, n in enumerate(lens)]
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int64), [torch.cat(x) for x in zip(*want)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,Dv", HEADS)
@pytest.mark.parametrize("page,window,first", [(16, 20, 3), (16, 64, 0), (32, 33, 40), (64, 1, 1), (16, 1, 0), (256, 100, 5), (7, 30, 9), (16, 10 ** 6, 0)])
def test_decode(Hq, Hkv, D, Dv, page, window, first, dtype):
    from llm_from_scratch_b200 import ops
    lens = [0, 1, 2, 15, 16, 17, 33, 63, 64, 65, 100, 130, 257, 500, 0, 641]
    q, k, v, bt, cl, want = decode_case(lens, Hq, Hkv, D, Dv, page, window, first, dtype)
    got = ops.window_decode(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cl.cuda(), D ** -0.5, window, first)
    check_close(got, *want, dtype)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,lo,hi,window,first", [(1, 4000, 4000, 1024, 4), (2, 5000, 9000, 4096, 64), (70, 1, 300, 128, 4), (3, 100, 2100, 2000, 0)])
def test_decode_long(batch, lo, hi, window, first, dtype):
    """Contexts that several CTAs share, and batches that fill the device."""
    from llm_from_scratch_b200 import ops
    lens = torch.randint(lo, hi + 1, (batch,), generator=torch.Generator().manual_seed(hi)).tolist()
    q, k, v, bt, cl, want = decode_case(lens, 32, 8, 128, 128, 16, window, first, dtype, seed=batch)
    got = ops.window_decode(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cl.cuda(), 128 ** -0.5, window, first)
    check_close(got, *want, dtype)


def prompt_case(new, before, Hq, Hkv, D, Dv, page, window, first, dtype, seed=0, poison=True):
    gen = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, before)]
    lows = [max(0, b - window + 1) if a else n for a, b, n in zip(new, before, lens)]
    q = torch.randn(sum(new), Hq, D, generator=gen).to(dtype)
    k, v, bt, rows = paged(lens, page, window, first, lows, gen, dtype, Hkv, D, Dv, poison=poison)
    want = [formula(x, *rows[i], before[i], D ** -0.5, window, first) for i, x in enumerate(q.split(new))]
    cu = lambda x: torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), dtype=torch.int32)
    return q, k, v, bt, cu(new), cu(lens), max(new), [torch.cat(x) for x in zip(*want)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,Dv", HEADS)
@pytest.mark.parametrize("page,window,first", [(16, 20, 3), (16, 64, 0), (32, 33, 40), (64, 1, 1), (256, 100, 5), (7, 30, 9), (16, 10 ** 6, 0)])
def test_portions(Hq, Hkv, D, Dv, page, window, first, dtype):
    from llm_from_scratch_b200 import ops
    new, before = [1, 0, 5, 70, 33, 1, 130, 64], [0, 9, 40, 0, 100, 300, 17, 64]
    q, k, v, bt, cu_q, cu_k, longest, want = prompt_case(new, before, Hq, Hkv, D, Dv, page, window, first, dtype)
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cu_q.cuda(), cu_k.cuda(), longest, D ** -0.5, window, first)
    check_close(got, *want, dtype)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,before,window,first", [([700], [0], 129, 4), ([300, 257], [1000, 63], 500, 17), ([3], [3000], 2500, 70), ([512, 1], [512, 700], 64, 130)])
def test_portions_long(new, before, window, first, dtype):
    from llm_from_scratch_b200 import ops
    q, k, v, bt, cu_q, cu_k, longest, want = prompt_case(new, before, 8, 2, 128, 128, 16, window, first, dtype, seed=7)
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cu_q.cuda(), cu_k.cuda(), longest, 128 ** -0.5, window, first)
    check_close(got, *want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_only_some_rows_see(D, dtype):
    """An infinity or NaN in a value row reaches the rows that see it and no others; the same for a key row."""
    from llm_from_scratch_b200 import ops
    new, before, window, first = [150, 20], [30, 0], 40, 2
    q, k, v, bt, cu_q, cu_k, longest, _ = prompt_case(new, before, 4, 2, D, D, 16, window, first, dtype, poison=False)
    plain = [x.cuda() for x in (q, k, v, bt, cu_q, cu_k)]
    rows = lambda pool: pool[bt[0, :12].long()].flatten(0, 1)[:180]
    _, _, sums = formula(q[:150], rows(k), rows(v), 30, D ** -0.5, window, first)
    for odd in (math.nan, math.inf):
        for pool, j in ((v, 77), (v, 1), (k, 100)):
            marked = pool.clone()
            marked[bt[0, j // 16], j % 16, 1, 5] = odd
            args = [plain[0], *(marked.cuda() if x is pool else x.cuda() for x in (k, v)), *plain[3:]]
            got = ops.window_attention(*args, longest, D ** -0.5, window, first).float()
            sees = torch.zeros(170, dtype=torch.bool)
            for i in range(150):
                p = 30 + i
                sees[i] = 0 <= p - j and (p - j < window or j < first)
            hit = ~torch.isfinite(got).all(-1)[:, 2:].cpu()           # heads of KV head 1
            if pool is v:
                assert torch.equal(hit.all(1), sees) and torch.equal(hit.any(1), sees)
                assert torch.isfinite(got[..., [c for c in range(D) if c != 5]]).all()
            elif math.isnan(odd):
                assert torch.equal(hit.all(1), sees) and torch.equal(hit.any(1), sees)
            want, spread, _ = formula(q[:150], rows(marked if pool is k else k), rows(marked if pool is v else v), 30, D ** -0.5, window, first)
            rest = torch.nonzero(~sees[:150])[:, 0]
            check_close(got[:150][rest.cuda()].to(dtype), want[rest], spread[rest], sums[rest], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity_weigh_nothing(dtype):
    from llm_from_scratch_b200 import ops
    q, k, v, bt, cl, _ = decode_case([50, 5], 8, 2, 128, 128, 16, 30, 4, dtype, poison=False)
    q, k = q.abs() + 0.1, k.clone()
    for j in (0, 1, 30, 41, 49):
        k[bt[0, j // 16], j % 16] = -math.inf
    k[bt[1, 0], :5] = -math.inf                                       # nothing is left of the second sequence
    seen = [j for j in range(50) if (j < 4 or j >= 20) and j not in (0, 1, 30, 41, 49)]
    got = ops.window_decode(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cl.cuda(), 128 ** -0.5, 30, 4)
    rows = lambda pool: torch.stack([pool[bt[0, j // 16], j % 16] for j in seen])
    check_close(got[:1], *formula(q[:1], rows(k), rows(v), len(seen) - 1, 128 ** -0.5, 10 ** 6, 0), dtype)
    assert (got[1] == 0).all()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    got2 = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), bt.cuda(), cu, torch.tensor([0, 50, 55], dtype=torch.int32).cuda(), 1, 128 ** -0.5, 30, 4)
    check_close(got2[:1], *formula(q[:1], rows(k), rows(v), len(seen) - 1, 128 ** -0.5, 10 ** 6, 0), dtype)
    assert (got2[1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 24])
def test_rows_without_keys_and_rows_behind_the_last_sequence(D, dtype):
    """A portion longer than its context has rows before its first key; padding rows of ``out`` stay as they are; strided q and tables."""
    from llm_from_scratch_b200 import ops
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(40, 4 * D + 16, generator=gen).to(dtype).cuda()
    q = wide[:, 8:8 + 4 * D].unflatten(1, (4, D))
    k, v = (torch.randn(9, 16, 2, D, generator=gen).to(dtype).cuda() for _ in range(2))
    tables = torch.full((3, 12), -5, dtype=torch.int32).cuda()
    tables[:, 4:7] = torch.tensor([[3, 1, 8], [2, -1, -1], [0, 7, -1]])
    cu_q, cu_k = torch.tensor([0, 6, 6, 30], dtype=torch.int32).cuda(), torch.tensor([0, 48, 52, 68], dtype=torch.int32).cuda()
    out = torch.full((40, 4, D), 7.0, dtype=dtype).cuda()
    got = ops.window_attention(q, k, v, tables[:, 4:7], cu_q, cu_k, 24, D ** -0.5, 9, 1, out=out)
    assert got is out and (out[30:] == 7).all() and (out[6:14] == 0).all()
    flat = lambda pool, row, n: pool[tables[row, 4:7].clamp(min=0).long()].flatten(0, 1)[:n].cpu()
    for row, at, n, keys in ((0, 0, 6, 48), (2, 14, 16, 16)):
        want = formula(q[at:at + n].cpu(), flat(k, row, keys), flat(v, row, keys), keys - n, D ** -0.5, 9, 1)
        check_close(out[at:at + n], *want, dtype)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 24])
def test_pages_outside_the_pool_are_left_out_and_reported(D, dtype):
    from llm_from_scratch_b200 import _lib, ops
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(6, 16, 2, D, generator=gen).to(dtype).cuda() for _ in range(2))
    q = torch.randn(2, 4, D, generator=gen).to(dtype).cuda()
    tables = torch.tensor([[0, 1, 2, 3], [4, 6, 5, -1]], dtype=torch.int32).cuda()      # 6 and -1 are not pages
    lens = torch.tensor([60, 60], dtype=torch.int64).cuda()
    got = ops.window_decode(q, k, v, tables, lens, D ** -0.5, 60, 0)
    assert ops.read_status_code() == _lib.ERR_BOUNDS
    ids = [4] * 16 + [5] * 16
    rows = lambda pool: torch.stack([pool[b, j % 16] for j, b in enumerate(ids)]).cpu()
    want = formula(q[1:].cpu(), rows(k), rows(v), 31, D ** -0.5, 100, 0)
    check_close(got[1:], *want, dtype)
    cu = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    got = ops.window_attention(q, k, v, tables, cu(0, 1, 2), cu(0, 60, 120), 1, D ** -0.5, 60, 0)
    assert ops.read_status_code() == _lib.ERR_BOUNDS
    check_close(got[1:], *want, dtype)
    # a context that the table is too short for: the last keys of the table are the last of the context
    got = ops.window_decode(q, k, v, tables[:, :1], lens, D ** -0.5, 10, 0)
    assert ops.read_status_code() == _lib.ERR_BOUNDS
    check_close(got[:1], *formula(q[:1].cpu(), k[0].cpu(), v[0].cpu(), 15, D ** -0.5, 10, 0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_on_two_streams(dtype):
    """Calls captured into two graphs and replayed beside each other on two streams give what they give alone."""
    from llm_from_scratch_b200 import ops
    q, k, v, bt, cl, _ = [x.cuda() if torch.is_tensor(x) else x for x in decode_case([900, 3, 0, 2000], 32, 8, 128, 128, 16, 700, 4, dtype)]
    pq, pk, pv, pbt, cu_q, cu_k, longest, _ = [x.cuda() if torch.is_tensor(x) else x
                                               for x in prompt_case([100, 30], [500, 0], 8, 2, 128, 128, 16, 200, 4, dtype)]
    calls = [lambda: ops.window_decode(q, k, v, bt, cl, 128 ** -0.5, 700, 4),
             lambda: ops.window_attention(pq, pk, pv, pbt, cu_q, cu_k, longest, 128 ** -0.5, 200, 4)]
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    graphs = []
    for f in calls * 2:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (g, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                out.fill_(math.nan)
                g.replay()
    torch.cuda.synchronize()
    for (_, out), want in zip(graphs, alone * 2):
        assert torch.equal(out, want)


def test_empty_calls():
    from llm_from_scratch_b200 import ops
    k = torch.zeros(2, 16, 1, 64, device="cuda")
    q = torch.zeros(0, 2, 64, device="cuda")
    none = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    assert ops.window_decode(q, k, k, none, torch.zeros(0, dtype=torch.int64, device="cuda"), 1.0, 5).shape == (0, 2, 64)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert ops.window_attention(q, k, k, none.expand(0, 1).new_zeros(3, 1), cu, cu, 0, 1.0, 5, 2).shape == (0, 2, 64)
    none = torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    assert ops.window_decode(q, k, k, none, torch.zeros(0, dtype=torch.int64, device="cuda"), 1.0, 5).shape == (0, 2, 64)
    assert ops.window_attention(q, k, k, none, cu[:1], cu[:1], 0, 1.0, 5, 2).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [128, 72])
def test_pools_beyond_32_bits(D, dtype):
    """Pages behind 2^31 elements (2^32 bytes and more): the same bits as from a small pool of those pages."""
    from llm_from_scratch_b200 import ops
    page, Hq, Hkv, few = 16, 16, 8, 300
    blocks = 2 ** 31 // (page * Hkv * D) + few
    gen = torch.Generator("cuda").manual_seed(D)
    big = [torch.empty(blocks, page, Hkv, D, dtype=dtype, device="cuda") for _ in range(2)]
    small = [torch.randn(few, page, Hkv, D, generator=gen, device="cuda").to(dtype) for _ in range(2)]
    for b, s in zip(big, small):
        b[blocks - few:] = s
    lens = [700, 33, 1500, 16]
    ids = torch.randperm(few, generator=gen, device="cuda")[:4 * 75].int().view(4, 75)
    bt = torch.nn.functional.pad(ids, (0, 25), value=-1)
    bt[2] = torch.randint(0, few, (100,), generator=gen, device="cuda")
    far = torch.where(bt >= 0, bt + (blocks - few), bt)
    q = torch.randn(4, Hq, D, generator=gen, device="cuda").to(dtype)
    cl = torch.tensor(lens, device="cuda")
    decode = lambda pools, t: ops.window_decode(q, *pools, t, cl, 0.1, 200, 3)
    assert torch.equal(decode(big, far), decode(small, bt))
    new = [100, 33, 129, 1]
    cu = lambda x: torch.tensor([0] + x, device="cuda").cumsum(0).int()
    x = torch.randn(sum(new), Hq, D, generator=gen, device="cuda").to(dtype)
    prompts = lambda pools, t: ops.window_attention(x, *pools, t, cu(new), cu(lens), max(new), 0.1, 200, 3)
    assert torch.equal(prompts(big, far), prompts(small, bt))
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_token_strides_and_alignment(D, dtype):
    """Queries inside a wider tensor, one row for all tokens, rows and pools at odd addresses."""
    from llm_from_scratch_b200 import ops
    gen = torch.Generator().manual_seed(D)
    n, before, Hq, Hkv, page, window, first = 70, 50, 4, 2, 16, 33, 5
    k, v, bt, rows = paged([n + before], page, window, first, [max(0, before + 1 - window)], gen, dtype, Hkv, D, D)
    row = torch.randn(1, Hq, D, generator=gen).to(dtype)
    cu = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")
    shift = lambda t: torch.cat([torch.zeros(1, dtype=dtype), t.flatten()]).cuda()[1:].view(t.shape)
    def call(q, kk, vv):
        return ops.window_attention(q, kk, vv, bt.cuda(), cu(n), cu(n + before), n, D ** -0.5, window, first)
    want = formula(row.expand(n, Hq, D), *rows[0], before, D ** -0.5, window, first)
    check_close(call(row.cuda().expand(n, Hq, D), k.cuda(), v.cuda()), *want, dtype)
    x = torch.randn(n, Hq, D, generator=gen).to(dtype)
    want = formula(x, *rows[0], before, D ** -0.5, window, first)
    for extra, at in ((0, 0), (8, 0), (8, 8), (3, 1), (1, 0)):
        wide = torch.zeros(n, Hq * D + extra, dtype=dtype)
        wide[:, at:at + Hq * D] = x.flatten(1)
        check_close(call(wide.cuda()[:, at:at + Hq * D].unflatten(1, (Hq, D)), k.cuda(), v.cuda()), *want, dtype)
    check_close(call(x.cuda(), shift(k), shift(v)), *want, dtype)
    one = torch.tensor([n + before], device="cuda")
    want = formula(x[-1:], *rows[0], n + before - 1, D ** -0.5, window, first)
    check_close(ops.window_decode(shift(x[-1:]), shift(k), shift(v), bt.cuda(), one, D ** -0.5, window, first), *want, dtype)
    ops.check_status()
