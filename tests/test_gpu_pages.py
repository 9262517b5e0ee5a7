"""GPU tests of forked and compacted pages (vib3_amd.pages) against the same done entry by entry on the host: copies are exact."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_caches(kinds, pages, ps, seed=0):
    """Caches of these kinds with bytes of any pattern (NaN among them), and their pools as [pages, tokens, ...] views."""
    from vib3_amd import gqa, mla
    g = torch.Generator(device="cuda").manual_seed(seed)

    def noise(*shape):
        return torch.randint(-32768, 32768, shape, generator=g, device="cuda", dtype=torch.int16).view(torch.bfloat16)
    caches, pools = [], []
    for kind in kinds:
        if kind == "mla":
            pool = noise(pages, ps, 576)
            caches.append(mla.MlaCache(pool, 512))
            pools.append(pool)
            continue
        if kind == "mla_rows":
            pool = noise(pages, ps, 640)[..., 8:584]
            caches.append(mla.MlaCache(pool, 512))
            pools.append(pool)
            continue
        if kind == "tokens":
            k, v = noise(pages, ps, 2, 64), noise(pages, ps, 2, 64)
        elif kind == "heads":
            k, v = (noise(pages, 3, ps, 128).transpose(1, 2) for _ in range(2))
        elif kind == "one":
            k, v = noise(pages, ps, 1, 256), noise(pages, ps, 1, 256)
        else:  # tokens in wider rows, keys and values of a page together
            both = noise(pages, 2, ps, 2, 72)[..., :64]
            k, v = both[:, 0], both[:, 1]
        caches.append(gqa.GqaCache(k, v))
        pools += [k, v]
    return caches, pools


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def bits(pools):
    return [p.clone() for p in pools]


ALL = ["tokens", "mla", "heads", "wide", "one", "mla_rows"]


def fork_host(table, lens, parents, children, new, pools, ps, width):
    pages = pools[0].shape[0] if pools else 0
    for p, c, n in zip(parents, children, new):
        if not (0 <= p < len(table) and 0 <= c < len(table)):
            continue
        full, rest = divmod(min(max(lens[p], 0), width * ps), ps)
        if rest and 0 <= table[p][full] < pages and 0 <= n < pages:
            for t in pools:
                t[n, :rest] = t[table[p][full], :rest].clone()
        table[c] = (table[p][:full] + [n] + [-1] * width)[:width]


@pytest.mark.parametrize("kinds", [["tokens"], ["mla"], ALL, ["heads"] * 40])
@pytest.mark.parametrize("ps", [1, 16, 48, 257])
def test_fork(kinds, ps):
    from vib3_amd import pages
    caches, pools = make_caches(kinds, 12, ps, seed=ps)
    table = [[3, 7, 1, -1], [9, 0, 5, 2], [8, 8, 8, 8], [4, -1, 4, 4], [-1] * 4, [6, 6, 6, 6], [-1] * 4]
    lens = [2 * ps + ps // 2, 3 * ps, 5, 1, 0, 4 * ps, 0]
    parents, children, new = [0, 1, 0, 4], [2, 3, 4, 6], [10, 11, 8, 6]
    parents[3] = 5  # full to the last entry: no room for a new page
    dev = ints(table)
    want = bits(pools)
    fork_host(table, lens, parents, children, new, want, ps, 4)
    pages.fork_pages(caches, dev, ints(lens), ints(parents), ints(children), ints(new))
    assert dev.tolist() == table
    assert all(same(a, b) for a, b in zip(pools, want))


def test_fork_out_of_range():
    from vib3_amd import pages
    caches, pools = make_caches(ALL, 4, 16)
    table = [[3, -1, 9], [0, 1, 2], [1, 1, 1], [2, 2, 2], [7, 7, 7], [2 ** 31 - 1] * 3, [5, 5, 5]]
    lens = [20, 2 ** 31 - 1, -7, 40, 17, 33, 0]
    # a missing page, past the table, no tokens, pairs outside, a new page that is none
    parents, children, new = [0, 1, 2, -1, 7, 3, 5], [6, 4, 3, 4, 2, 7, 2], [1, 2, 0, 0, 0, 0, 400]
    dev, want = ints(table), bits(pools)
    fork_host(table, lens, parents, children, new, want, 16, 3)
    pages.fork_pages(caches, dev, ints(lens), ints(parents), ints(children), ints(new))
    assert dev.tolist() == table and all(same(a, b) for a, b in zip(pools, want))
    pages.fork_pages(caches, dev, ints(lens), ints([]), ints([]), ints([]))
    assert dev.tolist() == table


def compact_host(table, lens, pools, ps, pages):
    used = [[row[k] for k in range(min(-(-max(n, 0) // ps), len(row)))] for row, n in zip(table, lens)]
    live = sorted({p for row in used for p in row if 0 <= p < pages})
    holes = [p for p in range(len(live)) if p not in set(live)]
    to = dict(zip([p for p in live if p >= len(live)], holes))
    for t in pools:
        for a, b in to.items():
            t[b] = t[a]
    return len(live), [[to.get(p, p) for p in row] + [-1] * (len(table[0]) - len(row)) for row in used]


def random_tables(pages, seqs, width, ps, seed, shared=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).tolist()
    table, lens = [], []
    for s in range(seqs):
        n = int(torch.randint(0, width + 1, (1,), generator=g))
        row = [ids.pop() if ids else -1 for _ in range(n)]
        if table and table[-1] and row and torch.rand(1, generator=g) < shared:
            row[0] = table[-1][0]
        table.append(row + [int(torch.randint(-1, pages, (1,), generator=g)) for _ in range(width - n)])
        lens.append(max(0, n * ps - int(torch.randint(0, ps, (1,), generator=g))))
    return table, lens


@pytest.mark.parametrize("pages,seqs,width", [(1, 1, 1), (2, 1, 1), (31, 3, 4), (32, 5, 6), (33, 40, 2), (100, 7, 9), (1000, 30, 20), (70, 1, 70)])
@pytest.mark.parametrize("kinds,ps", [(["tokens"], 16), (ALL, 5), (["heads"] * 40, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(kinds, ps, pages, seqs, width, in_place):
    from vib3_amd import pages as P
    caches, pools = make_caches(kinds, pages, ps, seed=pages)
    op = P.PageCompaction(caches)
    for seed in range(3):
        table, lens = random_tables(pages, seqs, width, ps, seed)
        dev, want = ints(table), bits(pools)
        live, moved = compact_host(table, lens, want, ps, pages)
        out = dev if in_place else torch.full_like(dev, 77)
        got = op.launch(dev, ints(lens), out_table=None if in_place else out)
        assert got.tolist() == [live] and out.tolist() == moved
        assert in_place or dev.tolist() == table
        assert all(same(a, b) for a, b in zip(pools, want))


def test_compact_all_none_and_entries_that_are_no_pages():
    from vib3_amd import pages as P
    caches, pools = make_caches(["tokens", "mla"], 64, 4)
    op, want = P.PageCompaction(caches), bits(pools)
    table = ints([list(range(64))[::-1]])
    assert op.launch(table, ints([256])).tolist() == [64] and table.tolist() == [list(range(64))[::-1]]  # all in use: nothing moves
    assert op.launch(table, ints([0])).tolist() == [0] and table.tolist() == [[-1] * 64]
    assert op.launch(torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([])).tolist() == [0]
    assert all(same(a, b) for a, b in zip(pools, want))
    table = ints([[-5, 63, 64, 2 ** 31 - 1], [63, 40, -1, 3]])
    assert op.launch(table, ints([16, 10 ** 9])).tolist() == [3]
    # in use: 3, 40, 63; free below 3: 0, 1, 2
    assert table.tolist() == [[-5, 2, 64, 2 ** 31 - 1], [2, 1, -1, 0]]
    caches, pools = make_caches(["tokens"], 64, 4, seed=9)
    first = bits(pools)
    table = ints([[63, 40, 3, -1]])
    P.PageCompaction(caches).launch(table, ints([12]))
    assert table.tolist() == [[2, 1, 0, -1]]
    for a, b in zip(pools, first):
        assert same(a[0], b[3]) and same(a[1], b[40]) and same(a[2], b[63]) and same(a[3:], b[3:])


def test_compact_many_pages():
    """The most pages a call takes: 2^20 of one token, of which a few thousand are in use."""
    from vib3_amd import gqa, pages as P
    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(n, 1, 1, 64, generator=g, device="cuda").half() for _ in range(2))
    ids = torch.randperm(n, generator=g, device="cuda")[:5000]
    table = ids.int().view(5, 1000).clone()
    want = k[ids].clone(), v[ids].clone()
    op = P.PageCompaction([gqa.GqaCache(k, v)])
    assert op.launch(table, ints([1000] * 5)).tolist() == [5000]
    at = table.flatten().long()
    assert sorted(at.tolist()) == list(range(5000)) and torch.equal(k[at], want[0]) and torch.equal(v[at], want[1])
    low = ids < 5000
    assert torch.equal(at[low], ids[low])
    with pytest.raises(ValueError):
        P.PageCompaction([gqa.GqaCache(torch.zeros(n + 1, 1, 1, 64, dtype=torch.half, device="cuda"),
                                       torch.zeros(n + 1, 1, 1, 64, dtype=torch.half, device="cuda"))])


@pytest.mark.parametrize("ps", [65535, 65536])
@pytest.mark.parametrize("kinds", [["heads"], ["wide", "mla"]])
def test_largest_pages(kinds, ps):
    from vib3_amd import pages as P
    caches, pools = make_caches(kinds, 6, ps, seed=ps)
    table, lens = [[5, 2, -1], [-1, -1, -1], [4, -1, -1]], [ps + 12345, 0, ps]
    dev, want = ints(table), bits(pools)
    fork_host(table, lens, [0], [1], [3], want, ps, 3)
    P.fork_pages(caches, dev, ints(lens), ints([0]), ints([1]), ints([3]))
    lens[1] = lens[0]
    assert dev.tolist() == table and all(same(a, b) for a, b in zip(pools, want))
    live, moved = compact_host(table, lens, want, ps, 6)
    assert P.PageCompaction(caches).launch(dev, ints(lens)).tolist() == [live] and dev.tolist() == moved
    assert all(same(a, b) for a, b in zip(pools, want))


def test_host_refusals():
    from vib3_amd import pages as P
    (a,), _ = make_caches(["tokens"], 4, 16)
    (b,), _ = make_caches(["mla"], 5, 16)
    (c,), _ = make_caches(["tokens"], 4, 8)
    table, lens, one = ints([[0, 1], [2, 3]]), ints([20, 0]), ints([0])
    for caches in ([], [a, b], [a, c], [a.keys], [None]):
        with pytest.raises((TypeError, ValueError)):
            P.fork_pages(caches, table, lens, one, one, one)
        with pytest.raises((TypeError, ValueError)):
            P.PageCompaction(caches)
    for args in ((table.t(), lens, one, one, one), (table, lens[:1], one, one, one), (table, lens, one, ints([0, 1]), one),
                 (table, lens, one, one, one.long()), (table.cpu(), lens, one, one, one), (table, lens, one[None], one, one)):
        with pytest.raises((TypeError, ValueError)):
            P.fork_pages([a], *args)
    op = P.PageCompaction([a])
    for args in ((table.t(), lens), (table, lens[:1]), (table.long(), lens), (table, lens, table[:1])):
        with pytest.raises((TypeError, ValueError)):
            op.launch(*args)


def test_captured_fork_and_compact():
    """One graph whose tables and lengths change between replays, checked against the host each time."""
    from vib3_amd import pages as P
    caches, pools = make_caches(["tokens", "mla"], 40, 8)
    op = P.PageCompaction(caches)
    table, lens = ints([[-1] * 6] * 5), ints([0] * 5)
    parents, children, new = ints([0, 0]), ints([3, 4]), ints([0, 0])

    def step():
        P.fork_pages(caches, table, lens, parents, children, new)
        op.launch(table, lens)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(5):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randperm(40, generator=g).tolist()
        rows = [[ids.pop() for _ in range(6)] for _ in range(5)]
        n = torch.randint(0, 48, (5,), generator=g).tolist()
        n[0] = min(n[0], 40)
        n[3] = n[4] = n[0]
        fresh = [ids.pop(), ids.pop()]
        table.copy_(ints(rows)), lens.copy_(ints(n)), new.copy_(ints(fresh))
        want = bits(pools)
        fork_host(rows, n, [0, 0], [3, 4], fresh, want, 8, 6)
        live, moved = compact_host(rows, n, want, 8, 40)
        graph.replay()
        torch.cuda.synchronize()
        assert op.live.tolist() == [live] and table.tolist() == moved and all(same(a, b) for a, b in zip(pools, want))


def test_forked_and_compacted_sequences_attend_alike():
    """A fork sees its parent's tokens, before and after the pages were compacted."""
    from vib3_amd import gqa, pages as P
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(30, 16, 2, 64, generator=g, device="cuda").half() for _ in range(2))
    c = gqa.GqaCache(k, v)
    table = ints([[7, 29, 12, 5], [-1] * 4, [-1] * 4])
    lens = ints([55, 55, 55])
    P.fork_pages([c], table, lens, ints([0, 0]), ints([1, 2]), ints([20, 3]))
    op = gqa.GqaDecode(c, 8, 3)
    q = torch.randn(1, 8, 64, generator=g, device="cuda").half().expand(3, 8, 64)
    first = op.launch(q, table, lens, 0.125).clone()
    assert torch.equal(first[1], first[0]) and torch.equal(first[2], first[0])
    lens[0] = 0  # the parent is freed
    assert P.PageCompaction([c]).launch(table, lens).tolist() == [5]
    assert int(table.max()) == 4 and table[0].tolist() == [-1] * 4
    again = op.launch(q, table, lens, 0.125)
    assert torch.equal(again[1:], first[1:]) and bool((again[0] == 0).all())
