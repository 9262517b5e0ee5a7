"""GPU tests of the grouped-query attention operators (vib3_amd.gqa) against their definition in 64 bits (tests/gqa_reference.py,
which derives the tolerances)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import gqa_reference as R  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def rnd(*shape, dtype=BF16, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000003 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def close(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(9e9).max()):.3g} x tolerance"


def inv_freq(rot, base=1e6):
    return (base ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)).float()


class Paged:
    """Sequences of these many tokens in a cache of random pages; slots that no token has hold NaN."""

    def __init__(self, lens, kv_heads, dim, dtype=BF16, ps=16, seed=0, layout="tokens", spare=2, max_pages=None):
        from vib3_amd import gqa
        need = [(n + ps - 1) // ps for n in lens]
        pages = sum(need) + spare
        g = torch.Generator().manual_seed(seed)
        ids = torch.randperm(pages, generator=g).tolist()
        table = torch.full((len(need), max_pages or max(need + [1])), -1, dtype=torch.int32)
        for i, n in enumerate(need):
            for j in range(n):
                table[i, j] = ids.pop()
        if layout == "tokens":
            keys, values = (torch.full((pages, ps, kv_heads, dim), NAN, dtype=dtype, device="cuda") for _ in range(2))
        elif layout == "heads":
            keys, values = (torch.full((pages, kv_heads, ps, dim), NAN, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
        else:  # keys and values of a page together, tokens in wider rows
            both = torch.full((pages, 2, ps, kv_heads, dim + 8), NAN, dtype=dtype, device="cuda")[..., :dim]
            keys, values = both[:, 0], both[:, 1]
        self.lens, self.ps, self.table, self.keys, self.values = lens, ps, table.cuda(), keys, values
        self.k = [rnd(n, kv_heads, dim, dtype=dtype, seed=seed + 10 + i) for i, n in enumerate(lens)]
        self.v = [rnd(n, kv_heads, dim, dtype=dtype, seed=seed + 5000 + i) for i, n in enumerate(lens)]
        self.store()
        self.cache = gqa.GqaCache(keys, values)
        self.kv_heads, self.dim, self.dtype = kv_heads, dim, dtype

    def store(self):
        for i, n in enumerate(self.lens):
            if n:
                j = torch.arange(n, device="cuda")
                at = self.table[i].long()[j // self.ps], j % self.ps
                self.keys[at], self.values[at] = self.k[i], self.v[i]


# ------------------------------------------------------------------------------- append


@pytest.mark.parametrize("dim,dtype,src,interleaved,ps,heads,kv_heads,rot,norm", [
    (128, BF16, BF16, False, 64, 32, 8, 128, None), (128, F16, F32, True, 16, 40, 8, 64, F32), (64, BF16, F32, False, 1, 1, 1, 64, BF16),
    (64, F16, F16, True, 48, 7, 7, 16, F16), (256, BF16, F16, False, 7, 16, 2, 64, F16), (256, F16, BF16, True, 128, 33, 3, 256, F32),
    (128, BF16, BF16, False, 5, 128, 1, 0, BF16), (64, BF16, BF16, False, 16, 64, 8, 48, None),
])
@pytest.mark.parametrize("tokens", [1, 6, 131])
def test_append(dim, dtype, src, interleaved, ps, heads, kv_heads, rot, norm, tokens):
    from vib3_amd import gqa
    starts = [0, 130001, 5, 77]
    seqs = [i % 4 for i in range(tokens)]
    pos = [starts[s] + i // 4 for i, s in enumerate(seqs)]
    used = sorted({(s, p // ps) for s, p in zip(seqs, pos)})
    table = torch.full((4, (130001 + tokens) // ps + 1), -1, dtype=torch.int32, device="cuda")
    for i, (s, p) in enumerate(used):
        table[s, p] = len(used) - i
    keys, values = (rnd(len(used) + 1, ps, kv_heads, dim, dtype=dtype, seed=i) for i in (3, 4))
    before = keys.clone(), values.clone()
    qkv = rnd(tokens, heads + 2 * kv_heads, dim + 16, dtype=src, scale=1.5, seed=1)[..., 8:8 + dim]  # one projection, wider rows
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    wq, wk = ((1 + rnd(dim, dtype=F32, scale=0.2, seed=i)).to(norm) if norm else None for i in (5, 6))
    f, g = (inv_freq(rot) if rot else None), 1.25
    out = gqa.gqa_append(gqa.GqaCache(keys, values), table, ints(seqs), ints(pos), q, k, v, f, q_norm=wq, k_norm=wk, eps=1e-5,
                         rope_scale=g, interleaved=interleaved)
    s, p = torch.tensor(seqs, device="cuda"), torch.tensor(pos, device="cuda")
    at = table[s, p // ps].long(), p % ps
    u = R.half_step(dtype)
    for got, x, w, what in ((out, q, wq, "queries"), (keys[at], k, wk, "keys")):
        x = x.double()
        if norm:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        if rot:
            want = R.rotate(x[..., :rot], p[:, None], f, g, interleaved)
            # the norm's f32 work adds 2^-20 of each of the two elements, as in the part that is not turned
            close(got[..., :rot], want, R.rotate_tol(2 * g * x[..., :rot], u, want, interleaved), what)
        close(got[..., rot:], x[..., rot:], u * x[..., rot:].abs() * (1 + 2 ** -9) + 2.0 ** -20 * x[..., rot:].abs() + R.tiny(u), what)
    assert torch.equal(values[at], v.to(dtype))
    before[0][at], before[1][at] = keys[at], values[at]
    assert torch.equal(keys, before[0]) and torch.equal(values, before[1]), "slots that no token belongs to were written"


@pytest.mark.parametrize("layout", ["tokens", "heads", "joint"])
def test_append_padding_missing_pages_and_in_place(layout):
    from vib3_amd import gqa
    c = Paged([48, 48], 2, 64, ps=16, layout=layout, spare=0)
    before = c.keys.clone(), c.values.clone()
    ids = c.table[0, 0].item(), c.table[1, 0].item()
    table = ints([[ids[0], -1, 7], [ids[1], 6, 2 ** 31 - 1]])  # -1, 6, 7 and the last are not pages of the pool
    seqs, pos = ints([0, 0, 0, 0, 1, 1, 1, -1, 2, 0]), ints([3, 16, 32, 48, 5, 17, 47, 0, 0, -1])
    cached = [(0, ids[0], 3), (4, ids[1], 5)]  # 48 is past the table; the last three tokens are padding
    k, v, q = rnd(10, 2, 64, seed=5), rnd(10, 2, 64, seed=6), rnd(10, 6, 72, seed=7)
    first = q.clone()
    args = (c.cache, table, seqs, pos)
    want = torch.full((10, 6, 64), 7.0, dtype=BF16, device="cuda")
    assert gqa.gqa_append(*args, q[..., :64], k, v, inv_freq(64), q_out=want) is want
    gqa.gqa_append(*args, q[..., :64], k, v, inv_freq(64), q_out=q[..., :64])  # in place
    assert torch.equal(q[:7, :, :64], want[:7]) and torch.equal(q[7:], first[7:]) and torch.equal(q[..., 64:], first[..., 64:])
    assert bool((want[7:] == 7.0).all()) and not torch.equal(want[:7], first[:7, :, :64])
    ref = gqa.GqaCache(torch.zeros(1, 16, 2, 64, dtype=BF16, device="cuda"), torch.zeros(1, 16, 2, 64, dtype=BF16, device="cuda"))
    gqa.gqa_append(ref, ints([[0]]), ints([0, 0]), ints([3, 5]), None, k[[0, 4]], v[[0, 4]], inv_freq(64))
    for i, (t, page, row) in enumerate(cached):
        before[0][page, row], before[1][page, row] = ref.keys[0, (3, 5)[i]], v[t]
    assert torch.equal(c.keys.nan_to_num(9), before[0].nan_to_num(9)) and torch.equal(c.values.nan_to_num(9), before[1].nan_to_num(9))
    gqa.gqa_append(c.cache, table, seqs[:0], pos[:0], q[:0, :, :64], k[:0], v[:0], inv_freq(64))
    assert torch.equal(c.keys.nan_to_num(9), before[0].nan_to_num(9))


# ------------------------------------------------------------------------------- decode


def decode(c, heads, rows, op=None, scale=None, window=0, sinks=0, q=None, seqs=True, out=None, q_scale=2.0):
    """rows: (sequence, visible tokens) of each query. Returns (q, output)."""
    from vib3_amd import gqa
    q = rnd(len(rows), heads, c.dim, dtype=c.dtype, scale=q_scale, seed=1) if q is None else q
    op = op or gqa.GqaDecode(c.cache, heads, len(rows))
    return q, op.launch(q, c.table, ints([n for _, n in rows]), c.dim ** -0.5 if scale is None else scale,
                        seqs=ints([s for s, _ in rows]) if seqs else None, window=window, sinks=sinks, out=out)


def check_decode(c, q, got, rows, scale=None, window=0, sinks=0, hole=None):
    u = R.half_step(got.dtype)
    for r, (s, n) in enumerate(rows):
        n = min(n, c.lens[s]) if 0 <= s < len(c.lens) else 0
        if n <= 0:
            assert bool((got[r] == 0).all()), f"row {r} sees nothing and is not zero"
            continue
        pos = torch.tensor([n - 1], device="cuda")
        want, tol = R.attend(q[r:r + 1], c.k[s][:n], c.v[s][:n], pos, c.dim ** -0.5 if scale is None else scale, u, window, sinks,
                             None if hole is None else hole(s, torch.arange(n, device="cuda")))
        close(got[r:r + 1], want, tol, f"row {r}: sequence {s}, {n} tokens")


SHORT = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 300]


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 8), (28, 4), (16, 1), (17, 1), (48, 2), (5, 5), (12, 3), (33, 1)])
@pytest.mark.parametrize("dim,dtype,ps", [(128, BF16, 64), (64, F16, 48), (256, F16, 1), (256, BF16, 128), (64, BF16, 16), (128, F16, 7)])
def test_decode_heads_and_lengths(heads, kv_heads, dim, dtype, ps):
    c = Paged(SHORT, kv_heads, dim, dtype, ps, seed=heads)
    rows = [(i, n) for i, n in enumerate(SHORT)] + [(13, 0), (0, 0), (13, -5), (-1, 9), (14, 9), (13, 100)]
    check_decode(c, *decode(c, heads, rows), rows)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 0), (64, 16), (65, 1), (100, 100), (1000, 3), (7, 2 ** 31 - 1),
                                          (2 ** 31 - 1, 5)])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (256, BF16)])
def test_decode_windows(window, sinks, dim, dtype):
    lens = SHORT + [777, 3000]
    c = Paged(lens, 2, dim, dtype, 16, seed=2)
    rows = [(i, n) for i, n in enumerate(lens)] + [(15, 0), (15, 64), (15, 65), (14, 101)]
    check_decode(c, *decode(c, 8, rows, window=window, sinks=sinks), rows, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(32, 8, 128, BF16), (16, 2, 256, F16), (40, 8, 64, BF16), (32, 1, 128, F16)])
@pytest.mark.parametrize("lens", [[20011], [5000, 1, 9000, 64], [3001] * 20])
def test_decode_long_rows(heads, kv_heads, dim, dtype, lens):
    """Rows that many workgroups share, and workgroups that share many rows."""
    c = Paged(lens, kv_heads, dim, dtype, 64, seed=5)
    rows = list(enumerate(lens))
    check_decode(c, *decode(c, heads, rows), rows)
    check_decode(c, *decode(c, heads, rows, window=1500, sinks=4), rows, window=1500, sinks=4)


@pytest.mark.parametrize("n", [2, 255, 256, 257, 700, 1025, 5000])
def test_decode_row_counts(n):
    lens = [(i * 37) % 90 for i in range(n)]
    c = Paged(lens, 2, 64, BF16, 16, seed=6)
    rows = list(enumerate(lens))
    q, got = decode(c, 8, rows)
    some = sorted({*range(0, n, max(1, n // 60)), n - 1, *range(min(n, 20))})
    check_decode(c, q[some], got[some], [rows[i] for i in some])


def test_decode_missing_pages_are_not_seen():
    c = Paged([500, 70, 33], 2, 128, BF16, 16, seed=7)
    c.table[0, 3:7], c.table[1, 0], c.table[2, 2] = -1, 1000, -2
    c.table[1, 1:] = -1
    gone = [set(range(48, 112)), set(range(70)), {32}]

    def hole(s, j):
        return torch.tensor([int(x) in gone[s] for x in j], device="cuda")
    rows = [(0, 500), (0, 60), (0, 112), (2, 33), (2, 32)]
    check_decode(c, *decode(c, 8, rows), rows, hole=hole)
    check_decode(c, *decode(c, 8, rows, window=64, sinks=50), rows, window=64, sinks=50, hole=hole)
    _, got = decode(c, 8, [(1, 70), (1, 16), (1, 1)])
    assert bool((got == 0).all())


def test_decode_length_past_the_table():
    c = Paged([64, 64], 2, 64, F16, 16, seed=8)
    rows = [(0, 64), (0, 65), (1, 10 ** 9), (1, 2 ** 31 - 1)]
    check_decode(c, *decode(c, 4, rows), rows)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_nan_and_inf_stay_in_their_rows(dtype):
    c = Paged([300, 300, 40], 2, 128, dtype, 16, seed=9)
    for t in (c.k[0], c.v[0]):
        t[200:] = NAN
        t[199:201, :, ::2] = INF
    c.store()
    c.keys[c.table[2, 2].long(), 8:], c.values[c.table[2, 2].long(), 8:] = INF, NAN  # behind sequence 2, in its last page
    rows = [(0, 199), (1, 300), (2, 40), (0, 17), (0, 300)]
    q, got = decode(c, 8, rows)
    check_decode(c, q, got, rows[:4])
    assert bool(got[4].isnan().all())
    rows = [(0, 100), (0, 199)]
    check_decode(c, *decode(c, 8, rows, window=50, sinks=10), rows, window=50, sinks=10)


def test_decode_windows_hide_nan():
    c = Paged([1000], 2, 64, BF16, 16, seed=10)
    c.k[0][8:900], c.v[0][8:900] = NAN, INF
    c.store()
    rows = [(0, 1000), (0, 950)]
    check_decode(c, *decode(c, 8, rows, window=50, sinks=8), rows, window=50, sinks=8)
    check_decode(c, *decode(c, 8, rows[:1], window=100), rows[:1], window=100)


def far_pages(dim=128, kv_heads=2, ps=16):
    """A cache whose pages lie 2^30 elements and more apart."""
    from vib3_amd import gqa
    stride = 2 ** 30 + 4096
    space = torch.empty(2 * stride + 2 * ps * kv_heads * dim, dtype=BF16, device="cuda")
    at = (3, ps, kv_heads, dim), (stride, kv_heads * dim, dim, 1)
    keys, values = torch.as_strided(space, *at), torch.as_strided(space, *at, ps * kv_heads * dim)
    c = Paged([40], kv_heads, dim, BF16, ps, spare=0)
    c.keys, c.values, c.cache = keys, values, gqa.GqaCache(keys, values)
    c.store()
    return c


def test_far_pages():
    from vib3_amd import gqa
    c = far_pages()
    check_decode(c, *decode(c, 8, [(0, 40)]), [(0, 40)])
    q = rnd(30, 8, 128, scale=2.0, seed=3)
    got = gqa.GqaChunk(c.cache, 8, 30, 1).launch(q, c.table, ints([0, 30]), ints([40]), 0.09)
    want, tol = R.attend(q, c.k[0], c.v[0], torch.arange(10, 40, device="cuda"), 0.09, 2.0 ** -9 * 2)
    close(got, want, tol)
    gqa.gqa_append(c.cache, c.table, ints([0]), ints([40]), None, c.k[0][:1], c.v[0][:1])
    page = c.table[0, 2].long()
    assert torch.equal(c.keys[page, 8], c.k[0][0]) and torch.equal(c.values[page, 8], c.v[0][0])


@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_layouts_and_strided_outputs(layout, dim):
    c = Paged([100, 333, 7], 4, dim, F16, 16, seed=11, layout=layout)
    rows = [(0, 100), (1, 333), (2, 7), (1, 50)]
    q = rnd(4, 24, dim + 8, dtype=F16, scale=2.0, seed=12)[:, ::2, :dim]
    room = torch.full((4, 12, dim + 16), 5.0, dtype=F16, device="cuda")
    q, got = decode(c, 12, rows, q=q, out=room[..., 8:8 + dim])
    check_decode(c, q, got, rows)
    assert bool((room[..., :8] == 5.0).all()) and bool((room[..., 8 + dim:] == 5.0).all())


def test_decode_default_sequences_fewer_rows_and_repeats():
    from vib3_amd import gqa
    lens = [100, 2000, 7, 64]
    c = Paged(lens, 2, 128, BF16, 16, seed=13)
    op = gqa.GqaDecode(c.cache, 8, 9)
    rows = list(enumerate(lens))
    q, got = decode(c, 8, rows, op=op, seqs=False)
    check_decode(c, q, got, rows)
    assert got.data_ptr() == op.out.data_ptr() and got.shape[0] == 4
    first = got.clone()
    for _ in range(3):
        op.workspace.fill_(255)
        assert torch.equal(decode(c, 8, rows, op=op, q=q, seqs=False)[1], first)
    check_decode(c, *decode(c, 8, rows[:1], op=op), rows[:1])
    assert op.launch(q[:0], c.table, ints([]), 1.0, seqs=ints([])).shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 3.0, -50.0])
def test_scales(scale, dtype):
    """Scores far apart, equal and of the other sign."""
    from vib3_amd import gqa
    c = Paged([500, 70], 2, 64, dtype, 16, seed=14)
    rows = [(0, 500), (1, 70), (0, 129)]
    check_decode(c, *decode(c, 4, rows, scale=scale), rows, scale=scale)
    q = rnd(90, 4, 64, dtype=dtype, scale=2.0, seed=15)
    got = gqa.GqaChunk(c.cache, 4, 90, 2).launch(q, c.table, ints([0, 80, 90]), ints([500, 70]), scale)
    u = R.half_step(dtype)
    for s, a, b in ((0, 0, 80), (1, 80, 90)):
        want, tol = R.attend(q[a:b], c.k[s], c.v[s], torch.arange(c.lens[s] - (b - a), c.lens[s], device="cuda"), scale, u)
        close(got[a:b], want, tol, f"sequence {s}")


def test_scale_extremes():
    """A scale near f32's end: the largest score takes all (ties share)."""
    from vib3_amd import gqa
    c = Paged([300], 1, 64, BF16, 16, seed=16)
    q = rnd(100, 4, 64, scale=2.0, seed=17)
    s = q.float() @ c.k[0][:, 0].float().t()
    for scale in (3e38, -3e38):
        best = (s if scale > 0 else -s).masked_fill(~R.visible(torch.arange(200, 300, device="cuda"), 300)[:, None], -INF)
        top = best.topk(2).values
        clear = (top[..., 0] - top[..., 1]) > 1e-3  # f32 sums in another order differ by less
        want = c.v[0][best.argmax(-1), 0]
        got = gqa.GqaChunk(c.cache, 4, 100, 1).launch(q, c.table, ints([0, 100]), ints([300]), scale)
        assert torch.equal(got[clear], want[clear]) and bool(clear.any())
        got = decode(c, 4, [(0, 300)], scale=scale, q=q[99:])[1]
        assert torch.equal(got[clear[99:]], want[99:][clear[99:]])


@pytest.mark.parametrize("dtype,gap", [(F16, 12.0), (F16, 18.0), (BF16, 18.0), (F16, 24.0)])
def test_one_key_above_a_long_tail(dtype, gap):
    """One key whose value is 0 lies gap nats above 8192 others that hold all of the values."""
    from vib3_amd import gqa
    n = 8193
    c = Paged([n], 1, 64, dtype, 64, seed=18)
    c.k[0].zero_()
    c.k[0][4000, 0, 0] = 1.0
    c.v[0].fill_(1.0)
    c.v[0][4000] = 0.0
    c.store()
    q = torch.zeros(4, 4, 64, dtype=dtype, device="cuda")
    q[..., 0] = gap
    w = (n - 1) * math.exp(-gap)
    u = R.half_step(dtype)
    # the tail's equal probabilities round alike: u of the result, twice with its own rounding
    for want, got in ((w / (1 + w), decode(c, 4, [(0, n)], scale=1.0, q=q[:1])[1][0]),
                      (None, gqa.GqaChunk(c.cache, 4, 4, 1).launch(q, c.table, ints([0, 4]), ints([n]), 1.0))):
        if want is None:
            m = torch.tensor([(n - 4 + i) * math.exp(-gap) for i in range(4)], device="cuda", dtype=torch.float64)
            want = (m / (1 + m))[:, None, None]
        close(got, torch.zeros_like(got, dtype=torch.float64) + want, (2.5 * u + 2.0 ** -15) * want + 2.0 ** -25)


# ------------------------------------------------------------------------------- chunk


def chunk(c, heads, nq, nk=None, op=None, scale=None, window=0, sinks=0, q=None, out=None):
    from vib3_amd import gqa
    nk = nk or c.lens
    q = rnd(sum(nq), heads, c.dim, dtype=c.dtype, scale=2.0, seed=1) if q is None else q
    op = op or gqa.GqaChunk(c.cache, heads, len(q), len(nq))
    return q, op.launch(q, c.table, ints([sum(nq[:i]) for i in range(len(nq) + 1)]), ints(nk),
                        c.dim ** -0.5 if scale is None else scale, window=window, sinks=sinks, out=out)


def check_chunk(c, q, got, nq, nk=None, scale=None, window=0, sinks=0, hole=None):
    u, at = R.half_step(got.dtype), 0
    for s, (a, n) in enumerate(zip(nq, nk or c.lens)):
        pos = torch.arange(n - a, n, device="cuda")
        want, tol = R.attend(q[at:at + a], c.k[s][:max(n, 0)], c.v[s][:max(n, 0)], pos, c.dim ** -0.5 if scale is None else scale, u,
                             window, sinks, None if hole is None else hole(s, torch.arange(max(n, 0), device="cuda")))
        close(got[at:at + a], want, tol, f"sequence {s}: {a} queries over {n} tokens")
        none = pos < 0
        assert bool((got[at:at + a][none] == 0).all())
        at += a


@pytest.mark.parametrize("n", [1, 2, 17, 31, 32, 33, 63, 64, 65, 100, 129, 257, 300])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,ps", [(32, 8, 128, BF16, 64), (6, 2, 64, F16, 16), (16, 2, 256, BF16, 48),
                                                         (5, 5, 128, F16, 1), (7, 1, 64, BF16, 5), (24, 1, 256, F16, 128)])
def test_chunk_one_prompt(heads, kv_heads, dim, dtype, ps, n):
    c = Paged([n], kv_heads, dim, dtype, ps, seed=n)
    check_chunk(c, *chunk(c, heads, [n]), [n])


RAGGED = [([5, 1, 130, 0, 64, 1, 300], [5, 70, 130, 9, 200, 1, 1000]), ([1] * 9, [1, 64, 65, 500, 3, 2, 128, 127, 33]),
          ([4] * 5, [4, 100, 1001, 63, 68]), ([0, 0, 3], [0, 7, 3]), ([700], [2500]), ([10, 3, 40], [4, 0, 39])]


@pytest.mark.parametrize("nq,nk", RAGGED)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(32, 8, 128, BF16), (9, 3, 64, F16), (16, 2, 256, F16), (17, 1, 128, F16)])
def test_chunk_ragged(nq, nk, heads, kv_heads, dim, dtype):
    c = Paged(nk, kv_heads, dim, dtype, 16, seed=20)
    check_chunk(c, *chunk(c, heads, nq), nq)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 0), (64, 70), (65, 1), (100, 200), (500, 3), (7, 2 ** 31 - 1),
                                          (2 ** 31 - 1, 5)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(32, 8, 128, BF16), (10, 2, 64, F16), (16, 2, 256, BF16)])
def test_chunk_windows(window, sinks, heads, kv_heads, dim, dtype):
    nq, nk = [5, 1, 330, 64, 1, 300, 3], [5, 70, 330, 200, 1, 1500, 900]
    c = Paged(nk, kv_heads, dim, dtype, 16, seed=21)
    check_chunk(c, *chunk(c, heads, nq, window=window, sinks=sinks), nq, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,nq,nk", [
    (32, 8, 128, BF16, [3000], [3000]), (64, 8, 64, F16, [1500, 1000], [1500, 3000]), (32, 8, 128, F16, [40], [9000]),
    (32, 2, 256, BF16, [600, 600], [600, 2600]), (64, 64, 64, BF16, [300] * 3, [300, 400, 1300]), (8, 1, 128, BF16, [1, 2048], [4096, 2048]),
])
def test_chunk_long(heads, kv_heads, dim, dtype, nq, nk):
    c = Paged(nk, kv_heads, dim, dtype, 64, seed=22)
    check_chunk(c, *chunk(c, heads, nq), nq)
    check_chunk(c, *chunk(c, heads, nq, window=700, sinks=4), nq, window=700, sinks=4)


@pytest.mark.parametrize("seqs", [63, 64, 65, 300, 1100])
def test_chunk_sequence_counts(seqs):
    nk = [1 + (i * 29) % 80 for i in range(seqs)]
    nq = [(i * 7) % (n + 1) for i, n in enumerate(nk)]
    c = Paged(nk, 2, 64, BF16, 16, seed=23)
    check_chunk(c, *chunk(c, 4, nq), nq)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,nq,nk", [
    (32, 8, 128, BF16, [70] + [5] * 40, [9000] + [9] * 40), (8, 1, 256, F16, [1] * 300 + [20] + [1] * 300, [3] * 300 + [6000] + [130] * 300),
    (6, 2, 64, F16, [300, 2, 300] + [2] * 500, [301, 7000, 5000] + [2] * 500), (4, 1, 128, F16, [1] * 20, [64 * i + 1 for i in range(20)]),
    (16, 16, 64, BF16, [0, 3, 0, 400, 0], [0, 20000, 5, 400, 64]), (8, 1, 128, BF16, [2] * 1024, [70] * 1024),
])
def test_chunk_long_sequences_beside_short_ones(heads, kv_heads, dim, dtype, nq, nk):
    """Blocks that are cut into pieces beside whole ones, and counts of them around those that one launch plans for."""
    c = Paged(nk, kv_heads, dim, dtype, 64)
    check_chunk(c, *chunk(c, heads, nq), nq)
    check_chunk(c, *chunk(c, heads, nq, window=900, sinks=70), nq, window=900, sinks=70)


def test_chunk_missing_pages_are_not_seen():
    c = Paged([500, 70], 2, 128, BF16, 16, seed=24)
    c.table[0, 3:7], c.table[1, 0] = -1, 1000
    gone = [set(range(48, 112)), set(range(16))]

    def hole(s, j):
        return torch.tensor([int(x) in gone[s] for x in j], device="cuda")
    for nq in ([300, 70], [500, 3]):
        q, got = chunk(c, 8, nq)
        check_chunk(c, q, got, nq, hole=hole)
        q, got = chunk(c, 8, nq, window=40, sinks=60)
        check_chunk(c, q, got, nq, hole=hole, window=40, sinks=60)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 8, 64), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chunk_nan_and_inf_where_they_are_not_seen(dtype, heads, kv_heads, dim):
    """Every other token from 150 on is not finite: queries before see none of them; behind the newest token lies NaN."""
    n = 400
    c = Paged([n, 90], kv_heads, dim, dtype, 16, seed=25)
    clean = c.k[0].clone(), c.v[0].clone()
    c.k[0][151::2], c.v[0][151::2] = NAN, INF
    c.v[0][150::4], c.v[0][152::4, :, ::2] = -INF, NAN
    c.store()
    q, got = chunk(c, heads, [n, 90])
    c.k[0], c.v[0] = clean
    want, tol = R.attend(q[:150], c.k[0][:150], c.v[0][:150], torch.arange(150, device="cuda"), dim ** -0.5, R.half_step(dtype))
    close(got[:150], want, tol, "queries before")
    want, tol = R.attend(q[n:], c.k[1], c.v[1], torch.arange(90, device="cuda"), dim ** -0.5, R.half_step(dtype))
    close(got[n:], want, tol, "the other sequence")
    assert bool(got[152:n].isnan().all())


@pytest.mark.parametrize("window,sinks", [(30, 5), (64, 0), (200, 70)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (8, 1, 64, F16)])
def test_chunk_windows_hide_nan(window, sinks, heads, kv_heads, dim, dtype):
    """Tokens 75..79 are not finite: only the queries whose window holds one of them are touched."""
    n = 500
    c = Paged([n], kv_heads, dim, dtype, 16, seed=26)
    clean = c.k[0].clone(), c.v[0].clone()
    c.k[0][75:80], c.v[0][75:80] = NAN, INF
    c.store()
    q, got = chunk(c, heads, [n], window=window, sinks=sinks)
    c.k[0], c.v[0] = clean
    want, tol = R.attend(q, c.k[0], c.v[0], torch.arange(n, device="cuda"), dim ** -0.5, R.half_step(dtype), window, sinks)
    touched = R.visible(torch.arange(n, device="cuda"), n, window, sinks)[:, 75:80].any(-1)
    close(got[~touched], want[~touched], tol[~touched], "untouched queries")
    assert bool(got[touched].isnan().all()) and bool(touched.any()) and not bool(touched.all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("at", [0, 40, 70, 99])
def test_infinite_values_that_are_seen(dtype, at):
    """An infinite value that counts gives an infinity, both signs NaN, and one whose probability is 0 in f32 NaN."""
    from vib3_amd import gqa
    n = 100
    c = Paged([n], 1, 64, dtype, 16, seed=27)
    c.v[0][at, 0, 0], c.v[0][at, 0, 1] = INF, -INF
    c.v[0][at, 0, 2], c.v[0][(at + 1) % n, 0, 2] = INF, -INF
    c.store()
    q = rnd(n, 4, 64, dtype=dtype, seed=28)
    clean = torch.where(torch.isfinite(c.v[0]), c.v[0], torch.zeros_like(c.v[0]))
    for got, pos in ((chunk(c, 4, [n], q=q)[1], torch.arange(n, device="cuda")),
                     (chunk(c, 4, [7], q=q[:7])[1], torch.arange(n - 7, n, device="cuda")),
                     (decode(c, 4, [(0, n)], q=q[:1])[1], torch.tensor([n - 1], device="cuda"))):
        see, other = pos >= at, pos >= (at + 1) % n
        assert bool((got[see][..., 0] == INF).all()) and bool((got[see][..., 1] == -INF).all())
        assert bool(got[see & other][..., 2].isnan().all())
        want, tol = R.attend(q[:len(pos)], c.k[0], clean, pos, 0.125, R.half_step(dtype))
        close(got[..., 3:], want[..., 3:], tol[..., 3:], "other elements")
        close(got[~see][..., :2], want[~see][..., :2], tol[~see][..., :2], "queries before")
    # probability 0: the key lies 200 nats below the others
    c.k[0].zero_()
    c.k[0][at, 0, 0] = -200.0
    c.store()
    q = torch.zeros(n, 4, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    got = chunk(c, 4, [n], q=q, scale=1.0)[1]
    see = torch.arange(n, device="cuda") >= max(at, 1)
    assert bool(got[see][..., 0].isnan().all()) and bool(got[: at, :, 0].isfinite().all())
    assert bool(decode(c, 4, [(0, n)], q=q[:1], scale=1.0)[1][..., 0].isnan().all())


def test_infinite_scores():
    """Scores of +infinity give NaN, of -infinity a probability of 0, all of them -infinity zeros."""
    c = Paged([100], 1, 64, BF16, 16, seed=29)
    c.k[0].zero_()
    c.k[0][30, 0, 0] = INF
    c.store()
    q = torch.zeros(100, 4, 64, dtype=BF16, device="cuda")
    q[..., 0] = -1.0
    mean = c.v[0][:, 0].double()
    got = chunk(c, 4, [100], q=q)[1]
    for p in (29, 30, 64, 99):
        keep = [j for j in range(p + 1) if j != 30]
        close(got[p], mean[keep].mean(0).expand(4, 64), 2.0 ** -8 * mean[keep].abs().mean(0) + 2.0 ** -8 * mean[keep].mean(0).abs())
    keep = [j for j in range(100) if j != 30]
    close(decode(c, 4, [(0, 100)], q=q[:1])[1][0], mean[keep].mean(0).expand(4, 64),
          2.0 ** -8 * mean[keep].abs().mean(0) + 2.0 ** -8 * mean[keep].mean(0).abs())
    assert bool(chunk(c, 4, [100], q=-q)[1][30:].isnan().all()) and bool(decode(c, 4, [(0, 100)], q=-q[:1])[1].isnan().all())
    c.k[0][..., 0] = INF
    c.store()
    assert bool((chunk(c, 4, [100], q=q)[1] == 0).all()) and bool((decode(c, 4, [(0, 100)], q=q[:1])[1] == 0).all())


@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunk_layouts_views_and_rows_behind_the_last_sequence(layout, dim):
    nq, nk = [50, 7, 130], [100, 333, 130]
    c = Paged(nk, 4, dim, F16, 16, seed=30, layout=layout)
    q = rnd(200, 24, dim + 8, dtype=F16, scale=2.0, seed=12)[:, ::2, :dim]
    room = torch.full((200, 12, dim + 16), 5.0, dtype=F16, device="cuda")
    q, got = chunk(c, 12, nq, q=q, out=room[..., 8:8 + dim])
    check_chunk(c, q, got, nq)
    assert bool((room[..., :8] == 5.0).all()) and bool((room[..., 8 + dim:] == 5.0).all()) and bool((got[187:] == 5.0).all())


def test_chunk_offsets_are_cut_to_the_tensors():
    from vib3_amd import gqa
    c = Paged([64, 64, 64], 2, 64, BF16, 16, seed=31)
    q = rnd(20, 4, 64, scale=2.0, seed=32)
    op = gqa.GqaChunk(c.cache, 4, 20, 3)
    got = op.launch(q, c.table, ints([-5, 10, 15, 2 ** 31 - 1]), ints([64, 2 ** 31 - 1, 30]), 0.125)
    u, see = R.half_step(BF16), torch.arange(64, device="cuda")
    for s, a, b, n in ((0, 0, 10, 64), (1, 10, 15, 64), (2, 15, 20, 30)):
        want, tol = R.attend(q[a:b], c.k[s][:n], c.v[s][:n], see[n - (b - a):n], 0.125, u)
        close(got[a:b], want, tol, f"sequence {s}")
    op.out.fill_(3.0)
    got = op.launch(q, c.table, ints([10, 5, 5, 2]), ints([64, 64, 64]), 0.125)  # no sequence has queries
    assert bool((got == 3.0).all())


def test_chunk_repeats_bit_for_bit_and_alone():
    """A query's result does not depend on the workspace, nor a sequence's on the launch before."""
    from vib3_amd import gqa
    nq, nk = [40, 3, 130], [4000, 333, 130]
    c = Paged(nk, 2, 128, BF16, 16, seed=33)
    op = gqa.GqaChunk(c.cache, 8, 300, 5)
    q, got = chunk(c, 8, nq, op=op)
    first = got.clone()
    for _ in range(3):
        op.workspace.fill_(255)
        op.out.fill_(NAN)
        assert torch.equal(chunk(c, 8, nq, op=op, q=q)[1], first)
    assert op.launch(q[:0], c.table, ints([0, 0, 0, 0]), ints(nk), 1.0).shape == (0, 8, 128)


# ------------------------------------------------------------------------------- together


@pytest.mark.parametrize("ps", [2, 3, 1000, 4097, 65535, 65536])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_sizes(ps, dim):
    lens = [min(3 * ps // 2, 3000 + ps) + 7, 5, 2 * ps if ps > 1000 else 0]
    c = Paged(lens, 2, dim, F16, ps, spare=1)
    rows = [(s, n) for s in range(3) for n in (lens[s], lens[s] - 1, min(lens[s], ps), min(lens[s], ps + 1))]
    check_decode(c, *decode(c, 6, rows), rows)
    check_decode(c, *decode(c, 6, rows, window=100, sinks=3), rows, window=100, sinks=3)
    nq = [min(n, 9) for n in lens]
    check_chunk(c, *chunk(c, 6, nq), nq)


def test_longest_sequence():
    """2^31 - 2^12 tokens, the most that count: a table whose entries all name page 0, but for the last one. Keys are 0 but for token 777
    of page 0 (score 24) and the last token (score 50), whose values are the only ones that are not 0: what the others have in the sums is
    below 2^16 e^-24 and 2^31 e^-26, less than half a step."""
    from vib3_amd import gqa
    ps, most = 65536, 2 ** 31 - 2 ** 12
    k, v = (torch.zeros(2, ps, 1, 64, dtype=F16, device="cuda") for _ in range(2))
    last = (most - 1) % ps
    k[0, 777], k[1, last] = 24 / 64, 50 / 64
    v[0, 777], v[1, last] = rnd(1, 64, dtype=F16, seed=1), rnd(1, 64, dtype=F16, seed=2)
    first, second = v[0, 777, 0].float(), v[1, last, 0].float()
    c = gqa.GqaCache(k, v)
    table = ints([[0] * 32767 + [1]])
    q = torch.ones(6, 2, 64, dtype=F16, device="cuda")
    zero = torch.zeros_like(first)

    def check(got, want):
        assert bool(((got.float() - torch.stack(want)[:, None]).abs() <= 2 * R.half_step(F16) * torch.stack(want)[:, None].abs()).all())
    op = gqa.GqaDecode(c, 2, 6)
    lens = ints([2 ** 31 - 1, most, most - 1, 3 * ps + 778, 3 * ps, 777])
    check(op.launch(q, table, lens, 1.0, seqs=ints([0] * 6)), [second, second, first, first, first, zero])
    for sinks, low in ((0, zero), (778, first), (777, zero)):
        check(op.launch(q, table, lens, 1.0, seqs=ints([0] * 6), window=4096, sinks=sinks),
              [second, second, low, first, zero if sinks < 778 else first, zero])
    op = gqa.GqaChunk(c, 2, 6, 1)
    check(op.launch(q[:3], table, ints([0, 3]), ints([most]), 1.0), [first, first, second])
    check(op.launch(q[:3], table, ints([0, 3]), ints([2 ** 31 - 1]), 1.0, window=4096, sinks=0), [zero, zero, second])
    check(op.launch(q[:3], table, ints([0, 3]), ints([most - 1]), 1.0, window=4096, sinks=778), [first, first, first])


def test_host_refusals():
    from vib3_amd import gqa
    k = torch.zeros(4, 16, 2, 128, dtype=BF16, device="cuda")
    c = gqa.GqaCache(k, k.clone())
    table, one = ints([[0, 1], [2, 3]]), ints([0, 1])
    for bad in ((k[..., :96], k), (k, k[:3]), (k, k.half()), (k, k.transpose(2, 3).contiguous().transpose(2, 3)), (k[0], k[0]),
                (k.float(), k.float()), (k, torch.zeros(4, 16, 2, 256, dtype=BF16, device="cuda")[..., :128])):
        with pytest.raises((TypeError, ValueError)):
            gqa.GqaCache(*bad)
    q, kv, f = rnd(2, 8, 128), rnd(2, 2, 128), inv_freq(128)
    for kw in (dict(q=rnd(2, 7, 128)), dict(q=q.half()), dict(k=kv.float()), dict(v=kv[:1]), dict(inv_freq=f[:7]), dict(inv_freq=f.double()),
               dict(inv_freq=inv_freq(256)), dict(q_out=q.half()), dict(q_out=q[:, :4]), dict(q_norm=torch.ones(64, device="cuda")),
               dict(q_norm=torch.ones(128, device="cuda"), k_norm=torch.ones(128, device="cuda").half()), dict(seqs=ints([0])),
               dict(positions=one.long()), dict(block_table=table.t()), dict(q=rnd(2, 8, 256)[..., ::2])):
        a = dict(block_table=table, seqs=one, positions=one, q=q, k=kv, v=kv, inv_freq=f)
        with pytest.raises((TypeError, ValueError)):
            gqa.gqa_append(c, **{**a, **kw})
    for make in (lambda: gqa.GqaDecode(c, 7, 4), lambda: gqa.GqaDecode(c, 8, 70000), lambda: gqa.GqaDecode(c, 0, 4),
                 lambda: gqa.GqaChunk(c, 9, 4, 2), lambda: gqa.GqaChunk(c, 8, -1, 2), lambda: gqa.GqaChunk(c, 8, 4, -1)):
        with pytest.raises(ValueError):
            make()
    op, ch = gqa.GqaDecode(c, 8, 2), gqa.GqaChunk(c, 8, 2, 2)
    lens = ints([3, 4])
    for kw in (dict(q=rnd(3, 8, 128)), dict(q=rnd(2, 4, 128)), dict(lens=ints([1])), dict(out=q.half()), dict(scale=NAN), dict(window=-1),
               dict(sinks=-1), dict(seqs=ints([0])), dict(block_table=table[:1])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            op.launch(**{**dict(q=q, block_table=table, lens=lens, scale=0.1), **kw})
    for kw in (dict(q=rnd(3, 8, 128)), dict(q=rnd(2, 4, 128)), dict(cu_q=ints([0, 2])), dict(lens=ints([1])), dict(out=q.half()),
               dict(scale=INF), dict(window=-1), dict(sinks=-1), dict(block_table=ints([[0]] * 3))):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            ch.launch(**{**dict(q=q, block_table=table, cu_q=ints([0, 1, 2]), lens=lens, scale=0.1), **kw})


def test_other_streams():
    from vib3_amd import gqa
    lens = [3000, 17, 900]
    c = Paged(lens, 2, 128, BF16, 16, seed=40)
    rows = list(enumerate(lens))
    q, want = decode(c, 8, rows)
    qc, want_c = chunk(c, 8, [50, 3, 200])
    want, want_c = want.clone(), want_c.clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    ops = [(gqa.GqaDecode(c.cache, 8, 3), gqa.GqaChunk(c.cache, 8, 253, 3)) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (d, ch) in zip(streams, ops):
            with torch.cuda.stream(s):
                decode(c, 8, rows, op=d, q=q)
                chunk(c, 8, [50, 3, 200], op=ch, q=qc)
    torch.cuda.synchronize()
    for d, ch in ops:
        assert torch.equal(d.out, want) and torch.equal(ch.out, want_c)


def test_captured_step():
    """Append, decode and chunk in one graph whose lengths and positions change between replays."""
    from vib3_amd import gqa
    c = Paged([600, 600], 2, 128, BF16, 16, seed=41)
    k, v, q = rnd(2, 2, 128, seed=42), rnd(2, 2, 128, seed=43), rnd(2, 8, 128, scale=2.0, seed=44)
    qc, cu = rnd(40, 8, 128, scale=2.0, seed=45), ints([0, 30, 40])
    seqs, pos, lens = ints([0, 1]), ints([0, 0]), ints([1, 1])
    f, turned = inv_freq(128), torch.empty_like(q)
    dec, chk = gqa.GqaDecode(c.cache, 8, 2), gqa.GqaChunk(c.cache, 8, 40, 2)

    def step():
        gqa.gqa_append(c.cache, c.table, seqs, pos, q, k, v, f, q_out=turned)
        dec.launch(turned, c.table, lens, 0.1, window=300, sinks=2)
        chk.launch(qc, c.table, cu, lens, 0.1)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in (1, 40, 333, 599, 64):
        pos.copy_(ints([n - 1, n // 2]))
        lens.copy_(ints([n, n // 2 + 1]))
        graph.replay()
        torch.cuda.synchronize()
        got = turned.clone(), dec.out.clone(), chk.out.clone()
        for t in (turned, dec.out, chk.out):
            t.fill_(NAN)
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (turned, dec.out, chk.out)):
            assert torch.equal(a, b)
        chk.out.fill_(NAN)


def test_layer_together():
    """A prompt in two chunks, then single tokens and a drafted pair, as a layer runs them, against attention over all tokens."""
    from vib3_amd import gqa
    heads, kv_heads, dim, ps, n = 12, 3, 64, 16, 150
    keys, values = (torch.full((12, ps, kv_heads, dim), NAN, dtype=F16, device="cuda") for _ in range(2))
    c = gqa.GqaCache(keys, values)
    table = ints([[3, 9, 0, 11, 5, 2, 7, 10, 1, 4]])
    q, k, v = (rnd(n, h, dim, dtype=F32, seed=50 + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    wq, wk = (1 + rnd(dim, dtype=F32, scale=0.2, seed=i) for i in (53, 54))
    f = inv_freq(dim)
    dec, chk = gqa.GqaDecode(c, heads, 1), gqa.GqaChunk(c, heads, 100, 1)
    out, turned = [], []
    for a, b in ((0, 100), (100, 140), (140, 141), (141, 142), (142, 144), (144, 150)):
        pos = torch.arange(a, b, device="cuda", dtype=torch.int32)
        t = gqa.gqa_append(c, table, torch.zeros_like(pos), pos, q[a:b], k[a:b], v[a:b], f, q_norm=wq, k_norm=wk)
        got = dec.launch(t, table, ints([b]), dim ** -0.5, window=60, sinks=4) if b == a + 1 else \
            chk.launch(t, table, ints([0, b - a]), ints([b]), dim ** -0.5, window=60, sinks=4)
        out.append(got.clone())
        turned.append(t)
    j = torch.arange(n, device="cuda")
    at = table[0].long()[j // ps], j % ps
    want, tol = R.attend(torch.cat(turned), keys[at], values[at], j, dim ** -0.5, R.half_step(F16), 60, 4)
    close(torch.cat(out), want, tol)
    x = k.double()
    x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wk.double()
    want = R.rotate(x, j[:, None], f, 1.0, False)
    close(keys[at], want, R.rotate_tol(2 * x, R.half_step(F16), want, False))
