"""GPU tests of attention objects that serve calls of different kinds in turn, and of captured calls against the definition in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import gqa_reference as R  # noqa: E402
from test_gpu_gqa import BF16, F16, NAN, Paged, check_chunk, check_decode, chunk, close, decode, ints, inv_freq, rnd  # noqa: E402


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (12, 4, 64, F16), (16, 2, 256, BF16)])
def test_chunks_of_other_batches_between(heads, kv_heads, dim, dtype):
    """A call's result does not depend on what the object did before: fewer and more sequences, more and fewer pieces, whole blocks."""
    from vib3_amd import gqa
    nk = [4000, 333, 130, 9000, 70] + [5] * 1100
    c = Paged(nk, kv_heads, dim, dtype, 16, seed=90)
    op = gqa.GqaChunk(c.cache, heads, 2000, len(nk))

    def call(nq):
        n = len(nq)
        q = rnd(sum(nq), heads, dim, dtype=dtype, scale=2.0, seed=sum(nq))
        return q, op.launch(q, c.table[:n].contiguous(), ints([sum(nq[:i]) for i in range(n + 1)]), ints(nk[:n]), dim ** -0.5).clone()
    batches = [[40, 3, 130], [40, 3, 130, 700, 70], [1], [600], [0, 0, 1, 9], [3, 1, 2, 0, 70] + [1] * 1100, [0, 0, 0, 4, 4]]
    first = []
    for nq in batches:
        q, got = call(nq)
        some = sum(nq[:20])
        check_chunk(c, q[:some], got[:some], nq[:20], nk[:len(nq[:20])])
        first.append(got)
    for i in (0, 3, 1, 5, 0, 6, 2, 4, 1):
        assert torch.equal(call(batches[i])[1], first[i]), f"batch {i} again"


def test_a_sequence_alone_and_among_others():
    nq, nk = [40, 3, 130], [4000, 333, 130]
    c = Paged(nk, 2, 128, BF16, 16, seed=91)
    q, got = chunk(c, 8, nq)
    check_chunk(c, q, got, nq)
    for s, a in ((0, 0), (1, 40), (2, 43)):
        alone = [n if i == s else 0 for i, n in enumerate(nq)]
        part, mine = chunk(c, 8, alone, q=q[a:a + nq[s]])
        check_chunk(c, part, mine, alone)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (12, 4, 64, F16), (16, 2, 256, BF16)])
def test_decodes_of_other_batches_between(heads, kv_heads, dim, dtype):
    from vib3_amd import gqa
    lens = [4000, 333, 130, 9000, 70, 1]
    c = Paged(lens, kv_heads, dim, dtype, 16, seed=92)
    op = gqa.GqaDecode(c.cache, heads, 400)
    batches = [[(0, 4000)], [(i, n) for i, n in enumerate(lens)], [(5, 1)] * 300, [(3, 9000 - i) for i in range(50)], [(2, 0)] * 7, [(4, 70)] * 400]
    first = []
    for rows in batches:
        q, got = decode(c, heads, rows, op=op)
        check_decode(c, q, got, rows[:20])
        first.append(got.clone())
    for i in (1, 0, 3, 2, 1, 5, 0, 4, 3):
        assert torch.equal(decode(c, heads, batches[i], op=op)[1], first[i]), f"batch {i} again"


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (12, 4, 64, F16), (16, 2, 256, F16)])
def test_captured_step_against_the_definition(heads, kv_heads, dim, dtype):
    """Append, decode and chunk in two graphs with objects of their own, replayed in turn with other lengths each time."""
    from vib3_amd import gqa
    c = Paged([900, 900], kv_heads, dim, dtype, 16, seed=93)
    j = torch.arange(900, device="cuda")
    at = [(c.table[s].long()[j // 16], j % 16) for s in range(2)]
    f, scale, u = inv_freq(dim), dim ** -0.5, R.half_step(dtype)
    seqs, cu = ints([0, 1]), ints([0, 30, 40])
    graphs = []
    for i in range(2):
        g = dict(k=rnd(2, kv_heads, dim, dtype=dtype, seed=94 + i), v=rnd(2, kv_heads, dim, dtype=dtype, seed=96 + i),
                 q=rnd(2, heads, dim, dtype=dtype, scale=2.0, seed=98 + i), qc=rnd(40, heads, dim, dtype=dtype, scale=2.0, seed=100 + i),
                 pos=ints([0, 0]), lens=ints([1, 1]), turned=torch.empty(2, heads, dim, dtype=dtype, device="cuda"),
                 dec=gqa.GqaDecode(c.cache, heads, 2), chk=gqa.GqaChunk(c.cache, heads, 40, 2))

        def step(g=g):
            gqa.gqa_append(c.cache, c.table, seqs, g["pos"], g["q"], g["k"], g["v"], f, q_out=g["turned"])
            g["dec"].launch(g["turned"], c.table, g["lens"], scale, window=300, sinks=2)
            g["chk"].launch(g["qc"], c.table, cu, g["lens"], scale)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        g["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g["graph"]):
            step()
        graphs.append(g)
    for i, n in enumerate((1, 40, 333, 899, 64, 700, 2, 900)):
        g, lens = graphs[i % 2], [n, n // 2 + 1]
        g["pos"].copy_(ints([x - 1 for x in lens]))
        g["lens"].copy_(ints(lens))
        for t in (g["turned"], g["dec"].out, g["chk"].out):
            t.fill_(NAN)
        g["graph"].replay()
        torch.cuda.synchronize()
        for s, x in enumerate(lens):
            keys, values = c.keys[at[s]], c.values[at[s]]
            assert torch.equal(values[x - 1], g["v"][s])
            want, tol = R.attend(g["turned"][s:s + 1], keys[:x], values[:x], j[x - 1:x], scale, u, 300, 2)
            close(g["dec"].out[s:s + 1], want, tol, f"replay {i}: single token of sequence {s}")
            a, b = ((0, 30), (30, 40))[s]
            pos = torch.arange(x - (b - a), x, device="cuda")
            want, tol = R.attend(g["qc"][a:b], keys[:x], values[:x], pos, scale, u)
            close(g["chk"].out[a:b], want, tol, f"replay {i}: chunk of sequence {s}")
