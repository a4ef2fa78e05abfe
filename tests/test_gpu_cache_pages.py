"""Copies and compaction of cache pages (``ops.copy_pages``, ``ops.compact_pages``): exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cache(shapes, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda shape, dtype: torch.randint(0, 100, (pages, *shape), generator=g).to(dtype).cuda()
    return [make(shape, dtype) for shape, dtype in shapes]


SHAPES = [
    [((16, 4, 64), torch.bfloat16)],
    [((16, 8, 128), torch.bfloat16), ((16, 8, 128), torch.float32), ((16, 576), torch.bfloat16)],       # pages of unlike sizes
    [((3, 1, 5), torch.bfloat16), ((7,), torch.int8), ((256, 8, 128), torch.bfloat16), ((1, 1), torch.float32)],
]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("pages,n", [(4, 1), (50, 20), (400, 190), (5000, 2400)])
def test_copy(shapes, pages, n):
    from llm_from_scratch_b200 import ops
    if pages > 1000 and any(s[0][0] == 256 for s in shapes):
        pages, n = pages // 4, n // 4
    pools = cache(shapes, pages)
    g = torch.Generator().manual_seed(n)
    perm = torch.randperm(pages, generator=g)
    target = perm[:n].int()
    source = perm[n:][torch.randint(0, pages - n, (n,), generator=g)].int()              # some more than once
    source[n // 2] = -1
    target[n // 3] = -3
    want = [p.clone() for p in pools]
    for a, b in zip(source.tolist(), target.tolist()):
        if a >= 0 and b >= 0:
            for w, p in zip(want, pools):
                w[b] = p[a]
    ops.copy_pages(ops.PagePools(pools), source.cuda(), target.cuda())
    assert all(torch.equal(w, p) for w, p in zip(want, pools))
    ops.check_status()


@pytest.mark.parametrize("filler", [0, 1500])
def test_conflicting_pairs_are_left_out_and_reported(filler):
    """A page that is copied elsewhere is no target, and no page is a target twice; the other pairs are carried out."""
    from llm_from_scratch_b200 import ops
    pools = cache(SHAPES[0], 10 + 2 * filler)
    handle = ops.PagePools(pools)
    extra = torch.arange(10, 10 + filler), torch.arange(10 + filler, 10 + 2 * filler)
    pairs = lambda *x: [torch.cat([torch.tensor(v), e]).int().cuda() for v, e in zip(zip(*x), extra)]
    old = pools[0].clone()
    ops.copy_pages(handle, *pairs((0, 1), (1, 2), (3, 4), (5, 4), (6, 6), (7, 8)))
    assert ops.read_status_code() == -1
    want = old.clone()
    for a, b in ((1, 2), (3, 4), (7, 8)):
        want[b] = old[a]
    want[10 + filler:] = old[10:10 + filler]
    assert torch.equal(pools[0], want)
    ops.copy_pages(handle, *pairs((0, 0), (0, 9)))                                          # onto itself: nothing to do, no conflict
    ops.check_status()
    assert torch.equal(pools[0][9], pools[0][0])


def test_ids_outside_the_pool_are_left_out_and_reported():
    from llm_from_scratch_b200 import _lib, ops
    pools = cache(SHAPES[1], 8)
    old = [p.clone() for p in pools]
    ids = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    ops.copy_pages(ops.PagePools(pools), ids(0, 8, 1, 2), ids(4, 5, 2 ** 31 - 1, 6))
    assert ops.read_status_code() == _lib.ERR_BOUNDS
    for o, p in zip(old, pools):
        o[4], o[6] = o[0], o[2]
        assert torch.equal(o, p)


def plain_compact(tables, pages):
    used = sorted(set(x for x in tables.flatten().tolist() if 0 <= x < pages))
    named = set(used)
    holes = [p for p in range(len(used)) if p not in named]
    names = {p: p for p in used if p < len(used)}
    moves = list(zip([p for p in used if p >= len(used)], holes))
    names.update(moves)
    page_map = torch.tensor([names.get(p, -1) for p in range(pages)], dtype=torch.int32)
    renamed = torch.tensor([[names.get(x, -1) for x in row] for row in tables.tolist()], dtype=torch.int32).view(tables.shape)
    return renamed, page_map, [len(used), len(moves)], moves


@pytest.mark.parametrize("shapes", SHAPES[:2])
@pytest.mark.parametrize("pages,rows,width,share", [(1, 1, 1, 0.5), (10, 3, 2, 0.6), (100, 7, 20, 0.5), (2000, 64, 30, 0.3), (5000, 10, 300, 0.9),
                                                    (3000, 2, 1, 0.0), (1025, 300, 9, 0.7)])
def test_compact(shapes, pages, rows, width, share):
    from llm_from_scratch_b200 import ops
    pools = cache(shapes, pages)
    g = torch.Generator().manual_seed(pages)
    ids = torch.randint(0, pages, (rows, width), generator=g)                              # pages in several tables among them
    wide = torch.where(torch.rand(rows, width, generator=g) < share, -1 - ids, ids).int()
    tables = torch.cat([torch.full((rows, 3), 99999, dtype=torch.int32), wide, torch.full((rows, 1), 99999, dtype=torch.int32)], 1).cuda()[:, 3:3 + width]
    renamed, page_map, counts, moves = plain_compact(wide, pages)
    want = [p.clone() for p in pools]
    for a, b in moves:
        for w in want:
            w[b] = w[a]
    handle = ops.PagePools(pools)
    before = tables.clone()
    for _ in range(2):                                                                     # the tables given are left as they are
        r = ops.compact_pages(handle, tables)
        assert torch.equal(r.block_tables.cpu(), renamed) and torch.equal(r.page_map.cpu(), page_map) and r.counts.tolist() == counts
        assert all(torch.equal(w, p) for w, p in zip(want, pools))
    assert torch.equal(tables, before)
    ops.check_status()
    again = ops.compact_pages(handle, r.block_tables)                                      # nothing is left to move
    assert again.counts.tolist() == [counts[0], 0] and torch.equal(again.block_tables, r.block_tables)


def test_compact_reports_ids_outside_the_pool():
    from llm_from_scratch_b200 import _lib, ops
    pools = cache(SHAPES[0], 6)
    r = ops.compact_pages(ops.PagePools(pools), torch.tensor([[5, 6, -1], [2, 700, 5]], dtype=torch.int32).cuda())
    assert ops.read_status_code() == _lib.ERR_BOUNDS
    assert r.block_tables.tolist() == [[1, -1, -1], [0, -1, 1]] or r.block_tables.tolist() == [[0, -1, -1], [1, -1, 0]]
    assert r.block_tables.tolist() == plain_compact(torch.tensor([[5, 6, -1], [2, 700, 5]]), 6)[0].tolist()


def test_compact_without_tables():
    from llm_from_scratch_b200 import ops
    pools = cache(SHAPES[0], 6)
    for shape in ((0, 4), (3, 0)):
        r = ops.compact_pages(ops.PagePools(pools), torch.zeros(shape, dtype=torch.int32).cuda())
        assert r.counts.tolist() == [0, 0] and (r.page_map == -1).all() and r.block_tables.shape == shape
    ops.copy_pages(ops.PagePools(pools), *(torch.zeros(0, dtype=torch.int32).cuda() for _ in range(2)))


def test_captured_and_on_two_streams():
    """Forks and compactions captured into graphs, two pools on two streams."""
    from llm_from_scratch_b200 import ops
    caches = [cache(SHAPES[0], 600, seed=s) for s in (1, 2)]
    g = torch.Generator().manual_seed(9)
    perms = [torch.randperm(600, generator=g).int().cuda() for _ in caches]
    tables = [p[:120].view(6, 20) for p in perms]
    olds = [p[0].clone() for p in caches]
    handles = [ops.PagePools(p) for p in caches]
    graphs = []
    for handle, perm, table in zip(handles, perms, tables):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = ops.compact_pages(handle, table)
            ops.copy_pages(handle, r.block_tables[:, 19].contiguous(), perm[200:206] % 100 + 400)
        graphs.append((graph, r, torch.cuda.Stream()))
    for _ in range(2):
        for (pools, old, (graph, _, stream)) in zip(caches, olds, graphs):
            with torch.cuda.stream(stream):
                pools[0].copy_(old)
                graph.replay()
    torch.cuda.synchronize()
    for pools, old, perm, table, (_, r, _) in zip(caches, olds, perms, tables, graphs):
        renamed, page_map, counts, moves = plain_compact(table.cpu(), 600)
        want = old.clone()
        for a, b in moves:
            want[b] = want[a]
        for a, b in zip(renamed[:, 19].tolist(), (perm[200:206] % 100 + 400).tolist()):
            want[b] = want[a]
        assert torch.equal(r.block_tables.cpu(), renamed) and torch.equal(pools[0], want)


@pytest.mark.parametrize("pages,rows,width", [(70000, 300, 10), (3000, 300, 300), (65000, 300, 300), (66000, 1, 66000)])
def test_compact_of_many_pages_or_entries(pages, rows, width):
    from llm_from_scratch_b200 import ops
    pools = cache([((2, 1, 4), torch.int8), ((3,), torch.float32)], pages)
    g = torch.Generator().manual_seed(pages)
    tables = torch.randint(-pages // 2, pages, (rows, width), generator=g).int()
    renamed, page_map, counts, moves = plain_compact(tables, pages)
    want = [p.clone() for p in pools]
    at = torch.tensor(moves, dtype=torch.int64).view(-1, 2).cuda()
    for w, p in zip(want, pools):
        w[at[:, 1]] = p[at[:, 0]]
    r = ops.compact_pages(ops.PagePools(pools), tables.cuda())
    assert torch.equal(r.block_tables.cpu(), renamed) and torch.equal(r.page_map.cpu(), page_map) and r.counts.tolist() == counts
    assert all(torch.equal(w, p) for w, p in zip(want, pools))
    ops.check_status()


def test_pools_beyond_32_bits():
    from llm_from_scratch_b200 import ops
    pool = torch.empty(70000, 65536, dtype=torch.int8, device="cuda")                       # 4.6 GB
    page = lambda x: torch.full((65536,), x, dtype=torch.int8, device="cuda")
    for i, x in ((69999, 1), (69998, 2), (3, 3), (0, 4)):
        pool[i] = page(x)
    handle = ops.PagePools([pool])
    ids = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ops.copy_pages(handle, ids(69999, 3), ids(5, 69997))
    assert torch.equal(pool[5], page(1)) and torch.equal(pool[69997], page(3))
    r = ops.compact_pages(handle, ids(69998, 0, 69997, -1, 69999).view(1, 5))
    assert r.block_tables.tolist() == [[2, 0, 1, -1, 3]] and r.counts.tolist() == [4, 3]
    assert all(torch.equal(pool[i], page(x)) for i, x in ((0, 4), (1, 3), (2, 2), (3, 1)))
    ops.check_status()


def test_the_largest_pool():
    """2^31 - 1 pages of a byte: the last run of the plan ends at the last page."""
    from llm_from_scratch_b200 import ops
    n = 2 ** 31 - 1
    pool = torch.zeros(n, dtype=torch.uint8, device="cuda")
    used = [n - 1, 3, n - 2, n - 1500, 2 ** 30 + 7, n - 3000000, 0]
    for i, page in enumerate(used):
        pool[page] = i + 1
    tables = torch.tensor(used + [-1], dtype=torch.int32, device="cuda").view(2, 4)
    r = ops.compact_pages(ops.PagePools([pool]), tables)
    assert r.counts.tolist() == [7, 5]
    want = {0: 0, 3: 3, 2 ** 30 + 7: 1, n - 3000000: 2, n - 1500: 4, n - 2: 5, n - 1: 6}
    assert r.block_tables.flatten().tolist() == [want[p] for p in used] + [-1]
    assert pool[:8].tolist() == [7, 5, 6, 2, 4, 3, 1, 0]
    assert r.page_map[torch.tensor(used, device="cuda")].tolist() == [want[p] for p in used]
    assert sum(int((part >= 0).sum()) for part in r.page_map.split(1 << 28)) == 7
    ops.check_status()
