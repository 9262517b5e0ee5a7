"""GPU tests of the latent-attention operators (vib3_amd.mla) against their definition in 64 bits
(tests/mla_reference.py, which derives the tolerances)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import mla_reference as R  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
WIDE, NARROW = (512, 64, 128, 128), (256, 32, 64, 64)  # rank, rope, nope, v


def rnd(*shape, dtype=BF16, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000003 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def close(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(9e9).max()):.3g} x tolerance"


def inv_freq(rope):
    return (50000.0 ** (-torch.arange(0, rope, 2, device="cuda").double() / rope)).float()


def paged(rows_per_seq, ps, width, dtype, spare=2, fill=None, seed=0, max_pages=None):
    """A pool with a page table for sequences of these many tokens: (pool, table)."""
    need = [(n + ps - 1) // ps for n in rows_per_seq]
    pages = sum(need) + spare
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(need), max_pages or max(need + [1])), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        for j in range(n):
            table[i, j] = ids.pop()
    pool = torch.full((pages, ps, width), float("nan"), dtype=dtype, device="cuda") if fill is None else \
        torch.full((pages, ps, width), fill, dtype=dtype, device="cuda")
    return pool, table.cuda()


def fill_cache(pool, table, seq, rows):
    ps = pool.shape[1]
    j = torch.arange(len(rows), device="cuda")
    pool[table[seq].long()[j // ps], j % ps] = rows


# ------------------------------------------------------------------------------- append


@pytest.mark.parametrize("dims,dtype,kv_dtype,interleaved,ps,heads,norm", [
    (WIDE, BF16, BF16, True, 64, 64, True), (WIDE, F16, F32, False, 16, 5, True), (NARROW, BF16, F32, True, 1, 1, True),
    (NARROW, F16, F16, False, 48, 40, False), (WIDE, BF16, F16, False, 7, 128, False), (WIDE, F16, BF16, True, 128, 33, True),
])
@pytest.mark.parametrize("tokens", [1, 6, 131])
def test_append(dims, dtype, kv_dtype, interleaved, ps, heads, norm, tokens):
    from vib3_amd import mla
    rank, rope, nope, _ = dims
    starts = [0, 130001, 5, 77]
    seqs = [i % 4 for i in range(tokens)]
    pos = [starts[s] + i // 4 for i, s in enumerate(seqs)]
    pool, table = paged([0, 0, 0, 0], ps, rank + rope, dtype, spare=0, max_pages=(130001 + tokens) // ps + 1)
    used = sorted({(s, p // ps) for s, p in zip(seqs, pos)})
    pool = rnd(len(used) + 1, ps, rank + rope, dtype=dtype, seed=3)
    for i, (s, p) in enumerate(used):
        table[s, p] = len(used) - i
    before = pool.clone()
    kv = rnd(tokens, rank + rope + 64, dtype=kv_dtype, scale=1.5, seed=1)[:, 32:32 + rank + rope]  # rows inside wider ones
    q = rnd(tokens, heads, nope + rope, dtype=dtype, seed=2)
    w = (1 + rnd(rank, dtype=F32, scale=0.2)).to(F16) if norm else None
    f, g = inv_freq(rope), 1.25
    q_out = torch.empty(tokens, heads, rope, dtype=dtype, device="cuda")
    kv_out = torch.empty(tokens, rank + rope, dtype=dtype, device="cuda")
    mla.mla_append(mla.MlaCache(pool, rank), table, ints(seqs), ints(pos), kv, f, norm_weight=w, eps=1e-5, rope_scale=g,
                   interleaved=interleaved, q_rope=q[..., nope:], q_out=q_out, kv_out=kv_out)
    u, x, p = R.half_step(dtype), kv.double(), torch.tensor(pos, device="cuda")
    c = x[:, :rank]
    if norm:
        c = c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    close(kv_out[:, :rank], c, u * c.abs() * (1 + 2 ** -9) + 2.0 ** -20 * c.abs() + R.tiny(u), "latent")
    want = R.rotate(x[:, rank:], p, f, g, interleaved)
    close(kv_out[:, rank:], want, R.rotate_tol(g * x[:, rank:], u, want, interleaved), "shared key")
    want = R.rotate(q[..., nope:].double(), p[:, None], f, g, interleaved)
    close(q_out, want, R.rotate_tol(g * q[..., nope:].double(), u, want, interleaved), "queries")
    s, at = torch.tensor(seqs, device="cuda"), p
    assert torch.equal(pool[table[s, at // ps].long(), at % ps], kv_out)
    before[table[s, at // ps].long(), at % ps] = kv_out
    assert torch.equal(pool, before), "rows of the cache that no token belongs to were written"


def test_append_padding_missing_pages_and_in_place():
    from vib3_amd import mla
    rank, rope, ps = 512, 64, 16
    pool = rnd(3, ps, 576, seed=4)
    before = pool.clone()
    table = ints([[2, -1, 7], [1, 3, 0]])  # -1, 7 and 3 are not pages of the pool
    seqs = ints([0, 0, 0, 0, 1, 1, 1, -1, 2, 0])
    pos = ints([3, 16, 32, 48, 5, 17, 47, 0, 0, -1])  # 48 is past the table; the last three tokens are padding
    kept, cached = [0, 1, 2, 3, 4, 5, 6], [(0, 2, 3), (4, 1, 5), (6, 0, 15)]
    kv = rnd(10, 576, seed=5)
    q = rnd(10, 6, 192, seed=6)
    ref_q = torch.empty(10, 6, 64, dtype=BF16, device="cuda")
    kv_out = torch.full((10, 576), 7.0, dtype=BF16, device="cuda")
    args = (mla.MlaCache(pool, rank), table, seqs, pos, kv, inv_freq(rope))
    mla.mla_append(*args, q_rope=q[..., 128:], q_out=ref_q)
    first = q.clone()
    mla.mla_append(*args, q_rope=q[..., 128:], q_out=q[..., 128:], kv_out=kv_out)
    assert torch.equal(q[kept][..., 128:], ref_q[kept])
    assert torch.equal(q[7:], first[7:]) and torch.equal(q[..., :128], first[..., :128])
    assert bool((kv_out[7:] == 7.0).all()) and not bool((kv_out[:7] == 7.0).all(-1).any())
    for t, page, row in cached:
        before[page, row] = kv_out[t]
    assert torch.equal(pool, before)
    mla.mla_append(args[0], table, seqs[:0], pos[:0], kv[:0], args[5])
    assert torch.equal(pool, before)


# ------------------------------------------------------------------------------- decode


def decode_case(dims, dtype, heads, ps, seq_lens, rows, scale=None, q_scale=2.0, latent=False, seed=0):
    """rows: (sequence, visible tokens) of each query token. Returns what launch() takes, and the sequences' rows."""
    rank, rope, nope, v = dims
    pool, table = paged(seq_lens, ps, rank + rope, dtype, seed=seed)
    data = [rnd(n, rank + rope, dtype=dtype, seed=seed + 10 + i) for i, n in enumerate(seq_lens)]
    for i, d in enumerate(data):
        fill_cache(pool, table, i, d)
    n = len(rows)
    q = rnd(n, heads, (rank if latent else nope) + rope, dtype=dtype, scale=q_scale, seed=seed + 1)
    kv_b = None if latent else rnd(heads, nope + v, rank, dtype=dtype, scale=rank ** -0.5, seed=seed + 2)
    return dict(pool=pool, table=table, data=data, q=q, kv_b=kv_b, rows=rows, heads=heads, dims=dims,
                scale=scale or (nope + rope) ** -0.5, latent=latent)


def run_decode(c, op=None, max_rows=None):
    from vib3_amd import mla
    rank, rope, nope, v = c["dims"]
    op = op or mla.MlaDecode(mla.MlaCache(c["pool"], rank), c["heads"], nope, v, max_rows or len(c["rows"]))
    split = rank if c["latent"] else nope
    return op.launch(c["q"][..., :split], c["q"][..., split:], c["kv_b"], c["table"], ints([n for _, n in c["rows"]]),
                     c["scale"], seqs=ints([s for s, _ in c["rows"]]))


def check_decode(c, got, hole=None):
    rank, rope, nope, v = c["dims"]
    u, split = R.half_step(got.dtype), rank if c["latent"] else nope
    for r, (s, n) in enumerate(c["rows"]):
        rows = c["data"][s][:max(n, 0)] if 0 <= s < len(c["data"]) else c["data"][0][:0]
        if hole and len(rows):
            rows = rows[[j for j in range(len(rows)) if not hole(s, j)]]
        if len(rows) == 0:
            assert bool((got[r] == 0).all()), f"row {r} sees nothing and is not zero"
            continue
        want, tol = R.decode_row(c["q"][r, :, :split], c["q"][r, :, split:], c["kv_b"], nope, rows[:, :rank], rows[:, rank:],
                                 c["scale"], u)
        close(got[r], want, tol, f"row {r}: sequence {s}, {n} tokens")


@pytest.mark.parametrize("heads", [1, 8, 16, 17, 40, 64, 100, 128])
@pytest.mark.parametrize("dims,dtype,ps", [(WIDE, BF16, 64), (NARROW, F16, 48), (WIDE, F16, 1), (NARROW, BF16, 128)])
def test_decode_heads_and_lengths(heads, dims, dtype, ps):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 300]
    rows = [(i, n) for i, n in enumerate(lens)] + [(13, 0), (0, 0), (13, -5), (-1, 9), (14, 9), (13, 100)]
    c = decode_case(dims, dtype, heads, ps, lens, rows, seed=heads)
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("dims", [(512, 32, 96, 160), (256, 64, 32, 256), (512, 64, 256, 32)])
def test_decode_other_widths(dims):
    c = decode_case(dims, BF16, 20, 16, [100, 333], [(0, 100), (1, 333), (1, 50)])
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("heads,dims,dtype", [(64, WIDE, BF16), (16, WIDE, F16), (40, NARROW, BF16), (128, WIDE, BF16), (4, NARROW, F16)])
@pytest.mark.parametrize("lens", [[20011], [5000, 1, 9000, 64], [3001] * 20])
def test_decode_long_rows(heads, dims, dtype, lens):
    """Rows that many workgroups share, and workgroups that share many rows."""
    c = decode_case(dims, dtype, heads, 64, lens, [(i, n) for i, n in enumerate(lens)], seed=5)
    check_decode(c, run_decode(c))


def test_decode_many_rows():
    lens = [(i * 37) % 90 for i in range(700)]
    c = decode_case(NARROW, BF16, 8, 16, lens, [(i, n) for i, n in enumerate(lens)], seed=6)
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("latent", [False, True])
def test_decode_latent_form_and_drafts(latent, heads):
    rows = [(s, n - 3 + j) for s, n in ((0, 500), (1, 70), (2, 3)) for j in range(4)]
    c = decode_case(WIDE, BF16, heads, 32, [500, 70, 3], rows, latent=latent, seed=7)
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_large_scores(dtype):
    """Scores of several hundred: one token takes everything, and exp of the others underflows."""
    c = decode_case(WIDE, dtype, 16, 16, [400, 70], [(0, 400), (1, 70)], latent=True, q_scale=20.0, seed=8)
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("scale", [0.0, -0.05, 1e-30])
def test_decode_other_scales(scale):
    """A scale of 0 (plain averages), a negative one, and one that leaves nothing of the scores; with a masked whole part."""
    c = decode_case(WIDE, BF16, 20, 16, [900, 50], [(0, 900), (1, 50), (0, 0), (0, 333)], seed=17)
    c["scale"] = scale
    c["table"][0, 4:30] = -1
    check_decode(c, run_decode(c), hole=lambda s, j: s == 0 and 64 <= j < 480)


@pytest.mark.parametrize("heads,n", [(8, 1300), (128, 700)])
def test_decode_more_rows_than_the_plan_keeps_at_hand(heads, n):
    lens = [(i * 29) % 70 if i % 3 else 0 for i in range(n)]
    lens[n // 2] = 6000
    c = decode_case(NARROW, BF16, heads, 16, lens, [(i, m) for i, m in enumerate(lens)], seed=18)
    check_decode(c, run_decode(c))


@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 9, 17, 33])
def test_decode_row_counts(n):
    """Rows that share a finishing workgroup, each in many parts."""
    lens = [700 + 13 * i for i in range(n)]
    c = decode_case(WIDE, F16, 9, 32, lens, [(i, m) for i, m in enumerate(lens)], seed=19)
    check_decode(c, run_decode(c))


def test_decode_missing_pages_are_not_seen():
    """Pages that are not resident (in the middle, at the end, all of them) count as masked."""
    ps = 16
    c = decode_case(WIDE, BF16, 24, ps, [200, 200, 40], [(0, 200), (1, 200), (2, 40)], seed=9)
    holes = {(0, 0), (0, 3), (0, 4), (0, 5), (0, 6), (0, 12), (1, 11), (2, 0), (2, 1), (2, 2)}
    for k, (s, p) in enumerate(sorted(holes)):
        c["table"][s, p] = (-1, c["pool"].shape[0], 2 ** 31 - 1, -2 ** 31)[k % 4]
    check_decode(c, run_decode(c), hole=lambda s, j: (s, j // ps) in holes)


def test_decode_length_past_the_table():
    c = decode_case(WIDE, BF16, 8, 16, [64], [(0, 2 ** 31 - 1)], seed=10)
    got = run_decode(c)
    c["rows"] = [(0, 64)]
    check_decode(c, got)


def test_decode_nan_and_inf_stay_in_their_rows():
    c = decode_case(WIDE, BF16, 64, 64, [100, 100, 100], [(0, 100), (1, 90), (2, 100)], seed=11)
    c["data"][1][95] = float("inf")  # behind what row 1 sees
    c["data"][2][99, 3] = float("nan")  # seen by row 2
    for i in (1, 2):
        fill_cache(c["pool"], c["table"], i, c["data"][i])
    got = run_decode(c)
    assert bool(got[2].isnan().all())
    c["rows"] = c["rows"][:2]
    check_decode(c, got[:2])


def test_decode_far_pages():
    """A pool of more than 2^32 bytes and 2^31 elements: pages at its end."""
    ps, width = 128, 576
    pages = 2 ** 31 // (ps * width) + 64
    pool = torch.empty(pages, ps, width, dtype=BF16, device="cuda")
    small = decode_case(WIDE, BF16, 16, ps, [300], [(0, 300)], seed=12)
    table = ints([[pages - 1, 0, pages - 2]])
    fill_cache(pool, table, 0, small["data"][0])
    small["pool"], small["table"] = pool, table
    check_decode(small, run_decode(small))


def test_decode_strided_pool_and_outputs():
    from vib3_amd import mla
    big = rnd(6, 3, 16, 640, seed=13)
    pool = big[:, 1, :, 32:32 + 576]  # rows and pages inside wider ones
    c = decode_case(WIDE, BF16, 10, 16, [70], [(0, 70), (0, 33)], seed=13)
    for j in range(5):
        pool[j + 1] = c["pool"][int(c["table"][0, j])]
        c["table"][0, j] = j + 1
    c["pool"] = pool
    keep = torch.full((2, 12, 160), 3.0, dtype=BF16, device="cuda")
    op = mla.MlaDecode(mla.MlaCache(pool, 512), 10, 128, 128, 2)
    got = op.launch(c["q"][..., :128], c["q"][..., 128:], c["kv_b"], c["table"], ints([70, 33]), c["scale"], seqs=ints([0, 0]),
                    out=keep[:, 1:11, 16:144])
    check_decode(c, got)
    rest = keep.clone()
    rest[:, 1:11, 16:144] = 3.0
    assert bool((rest == 3.0).all())


def test_decode_default_sequences_and_fewer_rows():
    from vib3_amd import mla
    c = decode_case(WIDE, BF16, 8, 16, [40, 50, 60], [(0, 40), (1, 50), (2, 60)], seed=14)
    op = mla.MlaDecode(mla.MlaCache(c["pool"], 512), 8, 128, 128, 3)
    want = run_decode(c, op).clone()
    q = c["q"]
    assert torch.equal(op.launch(q[..., :128], q[..., 128:], c["kv_b"], c["table"], ints([40, 50, 60]), c["scale"]), want)
    assert torch.equal(op.launch(q[:2, :, :128], q[:2, :, 128:], c["kv_b"], c["table"], ints([40, 50]), c["scale"]), want[:2])
    assert op.launch(q[:0, :, :128], q[:0, :, 128:], c["kv_b"], c["table"], ints([]), c["scale"]).shape == (0, 8, 128)


def test_decode_repeats_bit_for_bit():
    c = decode_case(WIDE, BF16, 64, 64, [9000, 1200, 5], [(0, 9000), (1, 1200), (2, 5)], seed=15)
    first = run_decode(c).clone()
    for _ in range(3):
        assert torch.equal(run_decode(c), first)


def test_host_refusals():
    from vib3_amd import _lib, mla
    c = decode_case(WIDE, BF16, 8, 16, [40], [(0, 40)], seed=16)
    cache = mla.MlaCache(c["pool"], 512)
    op = mla.MlaDecode(cache, 8, 128, 128, 1)
    qn, qr, t, n = c["q"][..., :128], c["q"][..., 128:], c["table"], ints([40])
    with pytest.raises(ValueError):
        mla.MlaCache(c["pool"], 500)
    with pytest.raises(ValueError):
        mla.MlaDecode(cache, 129, 128, 128, 1)
    with pytest.raises(TypeError):
        op.launch(qn.half(), qr, c["kv_b"], t, n, 1.0)
    with pytest.raises(ValueError):
        op.launch(qn[:, :4], qr, c["kv_b"], t, n, 1.0)
    with pytest.raises(ValueError):
        op.launch(qn.repeat(2, 1, 1), qr.repeat(2, 1, 1), c["kv_b"], t, ints([40, 40]), 1.0)
    with pytest.raises(TypeError):
        op.launch(qn, qr, c["kv_b"], t, n.long(), 1.0)
    with pytest.raises(ValueError):
        op.launch(qn, qr, c["kv_b"].transpose(0, 1).contiguous().transpose(0, 1), t, n, 1.0)
    with pytest.raises(_lib.Vib3Error) as e:  # a view that starts off a 16-byte boundary
        wide = rnd(1, 8, 200)
        op.launch(wide[..., 1:129], qr, c["kv_b"], t, n, 1.0)
    assert e.value.code == -3
    with pytest.raises(ValueError):
        mla.mla_append(cache, t, ints([0, 0]), ints([0]), rnd(1, 576), inv_freq(64))
    with pytest.raises(TypeError):
        mla.mla_append(cache, t, ints([0]), ints([0]), rnd(1, 576), inv_freq(64), q_rope=rnd(1, 8, 64))
    with pytest.raises(ValueError):
        mla.mla_prefill(rnd(4, 8, 128), rnd(4, 8, 64), rnd(4, 8, 128), rnd(4, 64), ints([0, 4]), ints([0, 4]), 1.0)


# ------------------------------------------------------------------------------- prefill


def prefill_case(dims, dtype, heads, nq, nk, seed=0, q_scale=2.0):
    rank, rope, nope, v = dims
    return dict(q=rnd(sum(nq), heads, nope + rope, dtype=dtype, scale=q_scale, seed=seed), nq=nq, nk=nk, dims=dims,
                kv=rnd(sum(nk), heads, nope + v, dtype=dtype, seed=seed + 1), rows=rnd(sum(nk), rank + rope, dtype=dtype, seed=seed + 2))


def offsets(n):
    return ints([sum(n[:i]) for i in range(len(n) + 1)])


def run_prefill(c, **kw):
    from vib3_amd import mla
    rank, rope, nope, v = c["dims"]
    return mla.mla_prefill(c["q"][..., :nope], c["q"][..., nope:], c["kv"], c["rows"][:, rank:], offsets(c["nq"]), offsets(c["nk"]),
                           (nope + rope) ** -0.5, **kw)


def check_prefill(c, got):
    rank, rope, nope, v = c["dims"]
    want, tol = R.prefill(c["q"][..., :nope], c["q"][..., nope:], c["kv"], c["rows"][:, rank:], c["nq"], c["nk"], nope,
                          (nope + rope) ** -0.5, R.half_step(got.dtype))
    close(got[:sum(c["nq"])], want, tol)


@pytest.mark.parametrize("dims,dtype,heads", [(WIDE, BF16, 3), (NARROW, F16, 2), (WIDE, F16, 9), (NARROW, BF16, 1),
                                              ((512, 32, 128, 64), BF16, 2), ((512, 64, 64, 128), F16, 2)])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 100, 255, 257, 513])
def test_prefill_one_prompt(dims, dtype, heads, n):
    c = prefill_case(dims, dtype, heads, [n], [n], seed=n)
    check_prefill(c, run_prefill(c))


@pytest.mark.parametrize("nq,nk", [([5, 0, 300, 1, 64], [5, 0, 300, 1, 64]), ([1, 40, 129], [900, 41, 700]),
                                   ([0, 0, 7], [3, 0, 7]), ([10, 200, 3], [4, 100, 0]), ([1] * 90, list(range(90))),
                                   ([300] * 3, [333, 300, 10])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_ragged(nq, nk, dtype):
    """Empty sequences, chunks behind earlier tokens, and more queries than keys (the first see nothing)."""
    c = prefill_case(WIDE, dtype, 2, nq, nk, seed=3)
    check_prefill(c, run_prefill(c))


def test_prefill_longer_prompt():
    c = prefill_case(WIDE, BF16, 2, [2500], [2900], seed=4)
    check_prefill(c, run_prefill(c))


def test_prefill_large_scores():
    c = prefill_case(WIDE, F16, 2, [300], [300], seed=5, q_scale=60.0)
    check_prefill(c, run_prefill(c))


@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_prefill_other_scales(scale):
    from vib3_amd import mla
    c = prefill_case(WIDE, BF16, 2, [200, 9], [230, 4], seed=12)
    got = mla.mla_prefill(c["q"][..., :128], c["q"][..., 128:], c["kv"], c["rows"][:, 512:], offsets(c["nq"]), offsets(c["nk"]), scale)
    want, tol = R.prefill(c["q"][..., :128], c["q"][..., 128:], c["kv"], c["rows"][:, 512:], c["nq"], c["nk"], 128, scale,
                          R.half_step(BF16))
    close(got, want, tol)


@pytest.mark.parametrize("n", [2100, 4200])
def test_prefill_many_blocks(n):
    """Enough queries and heads for the wide workgroups."""
    c = prefill_case(NARROW, BF16, 64, [n], [n], seed=13)
    check_prefill(c, run_prefill(c))


def test_prefill_nan_behind_the_diagonal_and_in_neighbours():
    """Infinities and NaN in keys and values that a query does not see leave it as it is."""
    c = prefill_case(WIDE, BF16, 2, [150, 90, 20], [150, 90, 20], seed=6)
    c["kv"][100, 0, 128:] = float("nan")  # value of token 100 of the first prompt
    c["kv"][120, 1, 5] = float("inf")     # key of its token 120
    c["kv"][130, 1, 200] = float("-inf")  # value of its token 130
    c["kv"][150 + 90:] = float("nan")     # all of the last prompt
    c["rows"][150 + 90:] = float("nan")
    got = run_prefill(c)
    clean = prefill_case(WIDE, BF16, 2, [150, 90, 20], [150, 90, 20], seed=6)
    want = run_prefill(clean)
    assert torch.equal(got[:100, 0], want[:100, 0]) and bool(got[100:150, 0].isnan().all())
    assert torch.equal(got[:120, 1], want[:120, 1])
    assert torch.equal(got[150:240], want[150:240])
    assert bool(got[240:].isnan().all())


def test_prefill_views_and_rows_behind_the_last_sequence():
    c = prefill_case(WIDE, BF16, 3, [50, 21], [50, 21], seed=7)
    wide = rnd(100, 5, 328, seed=8)
    wide[:71, 1:4, 8:264] = c["kv"]
    c["kv"] = wide[:80, 1:4, 8:264]
    c["rows"] = torch.cat([c["rows"], rnd(9, 576, seed=9)])
    c["q"] = torch.cat([c["q"], rnd(14, 3, 192, seed=10)])
    out = torch.full((85, 3, 136), 5.0, dtype=BF16, device="cuda")
    got = run_prefill(c, out=out[..., 8:])
    c["kv"], c["rows"], c["q"] = c["kv"][:71], c["rows"][:71], c["q"][:71]
    check_prefill(c, got)
    assert bool((out[71:] == 5.0).all()) and bool((out[..., :8] == 5.0).all())


def test_prefill_offsets_are_cut_to_the_tensors():
    from vib3_amd import mla
    c = prefill_case(WIDE, BF16, 2, [40], [40], seed=11)
    args = (c["q"][..., :128], c["q"][..., 128:], c["kv"], c["rows"][:, 512:])
    want = mla.mla_prefill(*args, ints([0, 40]), ints([0, 40]), 0.1)
    assert torch.equal(mla.mla_prefill(*args, ints([0, 2 ** 30]), ints([-7, 2 ** 30]), 0.1), want)
    assert mla.mla_prefill(*(a[:0] for a in args), ints([0, 0]), ints([0, 0]), 0.1).shape == (0, 2, 128)
    none = mla.mla_prefill(args[0], args[1], c["kv"][:0], c["rows"][:0, 512:], ints([0, 40]), ints([0, 0]), 0.1)
    assert bool((none == 0).all())


# ------------------------------------------------------------------------------- streams, graphs, together


def test_other_streams():
    c = decode_case(WIDE, BF16, 64, 64, [3000, 50], [(0, 3000), (1, 50)], seed=20)
    p = prefill_case(WIDE, BF16, 2, [200], [200], seed=21)
    want_d, want_p = run_decode(c).clone(), run_prefill(p)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append((run_decode(c), run_prefill(p)))  # each with its own workspace
    torch.cuda.synchronize()
    for d, q in got:
        assert torch.equal(d, want_d) and torch.equal(q, want_p)


def test_captured_decode_step():
    """Append and decode captured as one graph; replays follow the inputs, the lengths and the pages."""
    from vib3_amd import mla
    rank, rope, heads, ps = 512, 64, 64, 16
    c = decode_case(WIDE, BF16, heads, ps, [900, 40, 17], [(0, 900), (1, 40), (2, 17)], seed=22)
    cache = mla.MlaCache(c["pool"], rank)
    op = mla.MlaDecode(cache, heads, 128, 128, 3)
    kv, q = rnd(3, 576, seed=23), c["q"].clone()
    seqs, pos, lens = ints([0, 1, 2]), ints([899, 39, 16]), ints([900, 40, 17])
    q_out, f = torch.empty(3, heads, 64, dtype=BF16, device="cuda"), inv_freq(rope)

    def step():
        mla.mla_append(cache, c["table"], seqs, pos, kv, f, q_rope=q[..., 128:], q_out=q_out)
        return op.launch(q[..., :128], q_out, c["kv_b"], c["table"], lens, c["scale"], seqs=seqs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for k in range(4):
        kv.copy_(rnd(3, 576, seed=30 + k))
        q.copy_(rnd(3, heads, 192, seed=40 + k))
        pos.copy_(ints([899 - 200 * k, 39 - k, 16 - 5 * k]))
        lens.copy_(pos + 1 if k < 3 else ints([0, 37, 0]))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = step().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want), k
        assert bool((got[0] == 0).all()) == (k == 3)


def test_layer_together():
    """A decoder layer as served: the prompt is appended and attended to in the expanded form, the next tokens by the
    absorbed form over the cache, whose result joins the residual stream that the MoE sublayer reads."""
    from vib3_amd import kernels, mla, moe
    from vib3_amd._lib import DT_BF16, ROUTER_SIGMOID
    hidden, heads, n, steps, ps = 1024, 16, 75, 3, 16
    rank, rope, nope, v = WIDE
    x = rnd(n + steps, hidden, dtype=F32, seed=50)
    w_in = rnd(hidden, dtype=F16, scale=0.1, seed=51) + 1
    w_q = rnd(hidden, heads * (nope + rope), dtype=F16, scale=hidden ** -0.5 * 2, seed=52)
    w_kv = rnd(hidden, rank + rope, dtype=F16, scale=hidden ** -0.5, seed=53)
    kv_b = rnd(heads, nope + v, rank, dtype=F16, scale=rank ** -0.5, seed=54)
    w_o = rnd(heads * v, hidden, dtype=F16, scale=(heads * v) ** -0.5, seed=55)
    f, scale = inv_freq(rope), (nope + rope) ** -0.5
    pool, table = paged([n + steps], ps, rank + rope, F16)
    cache = mla.MlaCache(pool, rank)
    op = mla.MlaDecode(cache, heads, nope, v, 1)

    def project(lo, hi):
        a = torch.empty(hi - lo, hidden, dtype=F16, device="cuda")
        for i in range(lo, hi):
            kernels.rms_norm_f32(x[i], a[i - lo], w_in, hidden, 1e-6)
        q, kv = (a @ w_q).view(hi - lo, heads, nope + rope), a @ w_kv
        rows = torch.empty(hi - lo, rank + rope, dtype=F16, device="cuda")
        mla.mla_append(cache, table, ints([0] * (hi - lo)), ints(list(range(lo, hi))), kv, f, norm_weight=torch.ones(rank, dtype=F16, device="cuda"),
                       q_rope=q[..., nope:], q_out=q[..., nope:], kv_out=rows)
        return q, rows

    q, rows = project(0, n)
    kv = (rows[:, :rank] @ kv_b.view(-1, rank).t()).view(n, heads, nope + v)
    prompt = mla.mla_prefill(q[..., :nope], q[..., nope:], kv, rows[:, rank:], ints([0, n]), ints([0, n]), scale)
    # the last prompt token again, from the cache: the two forms agree within both their tolerances
    again = op.launch(q[-1:, :, :nope], q[-1:, :, nope:], kv_b, table, ints([n]), scale)
    u = R.half_step(F16)
    want, tol = R.decode_row(q[-1, :, :nope], q[-1, :, nope:], kv_b, nope, rows[:, :rank], rows[:, rank:], scale, u)
    close(again[0], want, tol, "absorbed")
    y = torch.matmul(kv_b[:, nope:].double().flatten(0, 1), rows[:, :rank].double().t().contiguous()).abs().amax()
    # the expanded form has its keys and values rounded by the projection: another u of each
    k = (kv[..., :nope].double().abs().amax() * q[-1, :, :nope].double().abs().sum(-1).amax()) * scale
    close(prompt[-1], want, tol + u * (1 + 2 * float(k)) * float(y), "expanded")

    shape = moe.BankShape(hidden=hidden, inter=256, group_size=32, scale_dtype=DT_BF16, scale_sigma=0.02, num_experts=16, num_shared=1)
    bank = moe.Int4ExpertBank(shape, layer=0, seed=1)
    router, bias = moe.make_router(shape, 0, 1, 0.02, 0.1)
    layer = moe.MoeInt4Layer(bank, router, bias, top_k=4, scoring_mode=ROUTER_SIGMOID, norm_weight=w_in)
    cached = rows
    for i in range(n, n + steps):
        q, row = project(i, i + 1)
        cached = torch.cat([cached, row])
        got = op.launch(q[..., :nope], q[..., nope:], kv_b, table, ints([i + 1]), scale)
        want, tol = R.decode_row(q[0, :, :nope], q[0, :, nope:], kv_b, nope, cached[:, :rank], cached[:, rank:], scale, u)
        close(got[0], want, tol, f"step {i}")
        res = x[i] + (got.reshape(1, -1) @ w_o)[0].float()
        out = layer.launch(res, residual=res)
        assert bool(out.isfinite().all()) and float((out - res).norm()) > 0
