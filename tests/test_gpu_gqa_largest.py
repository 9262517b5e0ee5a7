"""GPU tests of the grouped-query attention and page launchers with so many workgroups that one dimension of a grid (fewer than 2^32
threads) does not hold them. Large inputs are one row seen many times (strides of 0)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_gqa import BF16, F16, ints, rnd  # noqa: E402


def test_append_of_2_24_tokens():
    """All but a few tokens are padding."""
    from vib3_amd import gqa
    n = (1 << 24) + 3
    keys, values = (torch.zeros(2, 16, 1, 64, dtype=BF16, device="cuda") for _ in range(2))
    k, v = rnd(1, 1, 64, seed=1), rnd(1, 1, 64, seed=2)
    seqs = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    pos = torch.zeros_like(seqs)
    for i, t in enumerate((0, 1 << 21, (1 << 24) - 1, 1 << 24, n - 1)):
        seqs[t], pos[t] = 0, 4 * i
    gqa.gqa_append(gqa.GqaCache(keys, values), ints([[1, 0]]), seqs, pos, None, k.expand(n, 1, 64), v.expand(n, 1, 64))
    for i in range(32):
        page, row = (1, i) if i < 16 else (0, i - 16)
        there = i in (0, 4, 8, 12, 16)
        assert torch.equal(keys[page, row], k[0] if there else torch.zeros_like(k[0])), i
        assert torch.equal(values[page, row], v[0] if there else torch.zeros_like(v[0])), i


def test_decode_of_the_most_rows_and_heads():
    """65536 rows of 1024 heads: a few see one token, whose value is their result, the others none."""
    from vib3_amd import gqa
    rows, heads = 65536, 1024
    k, v = rnd(1, 16, 1, 64, dtype=F16, seed=1), rnd(1, 16, 1, 64, dtype=F16, seed=2)
    op = gqa.GqaDecode(gqa.GqaCache(k, v), heads, rows)
    op.out.fill_(5.0)
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    some = [0, 1, 4095, 4096, 32767, 32768, 65534, 65535]
    lens[some] = 1
    q = rnd(1, heads, 64, dtype=F16, seed=3).expand(rows, heads, 64)
    got = op.launch(q, ints([[0]]), lens, 0.1, seqs=torch.zeros_like(lens))
    assert torch.equal(got[some], v[0, 0].expand(len(some), heads, 64))
    got[some] = 0
    assert not bool(got.view(torch.int32).any())


def test_chunk_of_many_sequences_and_heads():
    """8200 sequences of one query, 1024 key/value heads: each sees one token, whose value is its result."""
    from vib3_amd import gqa
    seqs, heads = 8200, 1024
    k, v = rnd(2, 1, heads, 64, seed=1), rnd(2, 1, heads, 64, seed=2)
    op = gqa.GqaChunk(gqa.GqaCache(k, v), heads, seqs, seqs)
    op.out.fill_(5.0)
    q = rnd(1, heads, 64, seed=3).expand(seqs, heads, 64)
    which = torch.arange(seqs, device="cuda", dtype=torch.int32) % 2
    got = op.launch(q, which[:, None].contiguous(), torch.arange(seqs + 1, device="cuda", dtype=torch.int32), torch.ones_like(which), 0.1)
    assert torch.equal(got[0::2], v[0].expand(seqs // 2, heads, 64)) and torch.equal(got[1::2], v[1].expand(seqs // 2, heads, 64))


def test_fork_of_many_children():
    """2^18 children in 64 pools (32 times one cache's two)."""
    from vib3_amd import gqa, pages
    n = 1 << 18
    k, v = (torch.zeros(n + 1, 2, 1, 64, dtype=F16, device="cuda") for _ in range(2))
    k[0], v[0] = rnd(2, 1, 64, dtype=F16, seed=1), rnd(2, 1, 64, dtype=F16, seed=2)
    first = k[0].clone(), v[0].clone()
    table = torch.full((n + 1, 1), -1, dtype=torch.int32, device="cuda")
    table[0] = 0
    children = torch.arange(1, n + 1, device="cuda", dtype=torch.int32)
    lens = torch.ones(n + 1, dtype=torch.int32, device="cuda")
    pages.fork_pages([gqa.GqaCache(k, v)] * 32, table, lens, torch.zeros_like(children), children, children.flip(0).contiguous())
    assert table[0].tolist() == [0] and torch.equal(table[1:, 0], children.flip(0))
    for t, f in zip((k, v), first):
        assert torch.equal(t[0], f) and torch.equal(t[1:, 0], f[0].expand(n, 1, 64)) and not bool(t[1:, 1].any())
