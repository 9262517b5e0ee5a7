"""GPU tests of latent attention (vib3_amd.mla) at the ends of the values' range: long tails behind one key, scales far above
1, infinities that are seen. Results are compared with the definition in 64 bits.

Where all of a row's probabilities are of one size, they are rounded alike, and the errors do not average out: the tolerances
here count a whole half step u of sum_j p_j |y_j| for them, u |result| for the result's own rounding, and 2^-16 sum_j p_j |y_j| for the
f32 work (mla_reference). In f16, steps end at 2^-24: a probability goes to the matrix cores as 2^11 times its ratio to a
reference that is no larger than the row's largest, so its error is at most 2^-25 / 2^11 = 2^-36 of the sum of all, whatever
its size."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import mla_reference as R  # noqa: E402

BF16, F16 = torch.bfloat16, torch.float16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def whole(shape, top, dtype, seed):
    """Whole numbers of -top..top: their products' sums are exact in f32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(dtype)


def normal(*shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def close(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(9e9).max()):.3g} x tolerance"


def flat_tol(p, y, out, u):
    """p [..., n] (64 bits) over the seen tokens, y [n, columns]."""
    size = p @ y.abs()
    least = 2.0 ** -36 * y.abs().sum(0) if u < 2 ** -9 else 0.0
    return u * out.abs() + (u + 2.0 ** -16) * size + least + R.tiny(u)


def pages(rows, ps=64):
    """A pool with the rows [n, width] of one sequence in reversed order of pages, and its block table."""
    n, width = rows.shape
    count = (n + ps - 1) // ps
    pool = torch.full((count, ps, width), float("nan"), dtype=rows.dtype, device="cuda")
    table = torch.arange(count - 1, -1, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    j = torch.arange(n, device="cuda")
    pool[table[0].long()[j // ps], j % ps] = rows
    return pool, table


def decode(rows, q, lens, scale, rank=512, kv_b=None, nope=128, v=128):
    """All of lens are query tokens of one sequence [n, rank + rope]."""
    from vib3_amd import mla
    pool, table = pages(rows)
    op = mla.MlaDecode(mla.MlaCache(pool, rank), q.shape[1], nope, v, len(lens))
    split = rank if kv_b is None else nope
    return op.launch(q[..., :split], q[..., split:], kv_b, table, ints(lens), scale, seqs=ints([0] * len(lens)))


def prefill(q, kv, kr, nope, scale, nq=None, nk=None):
    from vib3_amd import mla
    nq, nk = nq or [len(q)], nk or [len(kv)]
    offsets = lambda n: ints([sum(n[:i]) for i in range(len(n) + 1)])  # noqa: E731
    return mla.mla_prefill(q[..., :nope], q[..., nope:], kv, kr, offsets(nq), offsets(nk), scale)


# ------------------------------------------------------------------------------- one key far above a long tail


@pytest.mark.parametrize("gap", [9, 14, 16, 18, 20, 23])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_one_key_above_a_long_tail(dtype, gap):
    """64 query tokens of one sequence, so that a workgroup walks over thousands of tokens. The key at place 5000 scores gap
    above all others (in units of e) and holds nothing; the others make up the result."""
    n, heads, at = 8192, 16, 5000
    rows = torch.zeros(n, 576, device="cuda", dtype=dtype)
    rows[:, 1:256] = 1.0
    rows[:, 256:512] = normal(n, 256, dtype=dtype, seed=1)
    rows[at] = 0.0
    rows[at, 0] = gap
    q = torch.zeros(64, heads, 576, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    lens = [n - 7 * i for i in range(64)]
    got = decode(rows, q, lens, 1.0)
    y = rows[:, :512].double()
    for r in (0, 17, 63):
        p = R.softmax(y[:lens[r], 0])
        want = p @ y[:lens[r]]
        close(got[r], want, flat_tol(p, y[:lens[r]], want, R.half_step(dtype)), f"row {r}")


@pytest.mark.parametrize("gap", [9, 14, 16, 18, 20, 23])
@pytest.mark.parametrize("heads", [2, 64])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_one_key_above_a_long_tail(dtype, heads, gap):
    nq, nk, at = 1030, 6000, 11
    kv = torch.zeros(nk, heads, 256, device="cuda", dtype=dtype)
    kv[..., 128:192] = 1.0
    kv[..., 192:] = normal(nk, 1, 64, dtype=dtype, seed=2)
    kv[at] = 0.0
    kv[at, :, 0] = gap
    q = torch.zeros(nq, heads, 192, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    got = prefill(q, kv, torch.zeros(nk, 64, device="cuda", dtype=dtype), 128, 1.0)
    for i in (0, 1, 700, nq - 1):
        see = i + 1 + nk - nq
        y = kv[:see, 0, 128:].double()
        p = R.softmax(kv[:see, 0, 0].double())
        want = p @ y
        close(got[i], want, flat_tol(p, y, want, R.half_step(dtype)), f"query {i}")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_largest_key_comes_last(dtype):
    """Scores that grow by less than what makes the reference value follow them, up to its end."""
    n, heads = 4096, 2
    step = torch.arange(n, device="cuda") // 64  # a new largest score every 64 keys
    kv = normal(n, heads, 256, dtype=dtype, seed=3)
    kv[..., :128] = 0.0
    kv[..., 0] = step[:, None].to(dtype)
    q = torch.zeros(130, heads, 192, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    for scale in (0.05, 1.0, 2.5, 3.9):
        got = prefill(q, kv, torch.zeros(n, 64, device="cuda", dtype=dtype), 128, scale)
        for i in (0, 65, 129):
            see = i + 1 + n - 130
            p = R.softmax(kv[:see, 0, 0].double() * scale)
            y = kv[:see, 1, 128:].double()
            close(got[i, 1], p @ y, flat_tol(p, y, p @ y, R.half_step(dtype)), f"scale {scale}, query {i}")
        rows = torch.zeros(n, 576, device="cuda", dtype=dtype)
        rows[:, 0] = step.to(dtype)
        rows[:, 1:512] = normal(n, 511, dtype=dtype, seed=4)
        ql = torch.zeros(40, heads, 576, device="cuda", dtype=dtype)
        ql[..., 0] = 1.0
        lens = [n - 3 * i for i in range(40)]
        got = decode(rows, ql, lens, scale)
        for r in (0, 39):
            y = rows[:lens[r], :512].double()
            p = R.softmax(y[:, 0] * scale)
            close(got[r, 0], p @ y, flat_tol(p, y, p @ y, R.half_step(dtype)), f"scale {scale}, row {r}")


# ------------------------------------------------------------------------------- large scales


def best(s, y):
    """The limit of large scales: the mean of y over the tokens with the highest (whole-numbered) score, in 64 bits."""
    p = (s == s.amax(-1, keepdim=True)).double()
    p = p / p.sum(-1, keepdim=True)
    return p @ y, p @ y.abs()


@pytest.mark.parametrize("scale", [1e7, 1e8, -1e9, 1e20, 1e37, 3.4e38, -3.4e38])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("latent", [False, True])
def test_decode_large_scales(dtype, scale, latent):
    """Scores are whole numbers, so that from a scale of some hundreds on only the highest ones count. (Without the latent form,
    W_uk and W_uv each pass 128 columns on as they are.)"""
    heads, n = 20, 3000
    rows = whole((n, 576), 3, dtype, 5)
    q = whole((3, heads, (512 if latent else 128) + 64), 3, dtype, 6)
    kv_b = None
    if not latent:
        kv_b = torch.zeros(heads, 256, 512, device="cuda", dtype=dtype)
        i = torch.arange(128, device="cuda")
        kv_b[:, i, i + 100] = 1.0
        kv_b[:, 128 + i, i + 300] = 1.0
    lens = [n, 50, 1]
    got = decode(rows, q, lens, scale, kv_b=kv_b)
    u = R.half_step(dtype)
    for r, m in enumerate(lens):
        x, c = q[r].double(), rows[:m].double()
        s = (x[:, :512] @ c[:, :512].t() if latent else x[:, :128] @ c[:, 100:228].t()) + x[:, -64:] @ c[:, 512:].t()
        want, size = best(s if scale > 0 else -s, c[:, :512] if latent else c[:, 300:428])
        close(got[r], want, u * want.abs() + 2.0 ** -16 * size, f"row {r}")


@pytest.mark.parametrize("scale", [1e7, 1e8, -1e9, 1e20, 1e37, 3.4e38, -3.4e38])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [3, 128])
def test_prefill_large_scales(dtype, scale, heads):
    nq, nk = 530, 700
    q, kv, kr = whole((nq, heads, 192), 3, dtype, 7), whole((nk, heads, 256), 3, dtype, 8), whole((nk, 64), 3, dtype, 9)
    got = prefill(q, kv, kr, 128, scale)
    seen = torch.arange(nk, device="cuda") <= torch.arange(nq, device="cuda")[:, None] + nk - nq
    for h in range(0, heads, max(1, heads // 4)):
        s = q[:, h, :128].double() @ kv[:, h, :128].double().t() + q[:, h, 128:].double() @ kr.double().t()
        want, size = best((s if scale > 0 else -s).masked_fill(~seen, -math.inf), kv[:, h, 128:].double())
        close(got[:, h], want, R.half_step(dtype) * want.abs() + 2.0 ** -16 * size, f"head {h}")


# ------------------------------------------------------------------------------- infinities that are seen


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,at", [(8, 40), (64, 700), (128, 3)])
def test_decode_infinite_latent_that_is_seen(dtype, heads, at):
    """Latent form: a seen token whose latent is -infinity in one column scores -infinity. That column is 0 * infinity, and all
    others are what the other tokens make them."""
    n, column = 900, 77
    rows = normal(n, 576, dtype=dtype, seed=10)
    rows[at, column] = -math.inf
    q = normal(2, heads, 576, dtype=dtype, seed=11)
    q[..., column] = 1.0
    scale, lens, u = 0.05, [n, at + 1], R.half_step(dtype)
    got = decode(rows, q, lens, scale)
    rest = [c for c in range(512) if c != column]
    for r, m in enumerate(lens):
        keep = torch.tensor([j for j in range(m) if j != at], device="cuda")
        want, tol = R.decode_row(q[r, :, :512], q[r, :, 512:], None, 128, rows[keep, :512], rows[keep, 512:], scale, u)
        close(got[r][:, rest], want[:, rest], tol[:, rest], f"row {r}")
        assert bool(got[r][:, column].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [2, 64])
@pytest.mark.parametrize("at,scale", [(10, 0.07), (70, 0.07), (127, -0.07), (300, 0.07), (900, -0.07), (1299, 0.07)])
def test_prefill_infinite_value_with_probability_zero(dtype, heads, at, scale):
    """A seen key that scores -infinity beside a value of infinity in one column is 0 * infinity there, in tiles that some queries
    do not see all of as in others; the queries before it, and the other columns, are as without that token."""
    n, column = 1300, 37
    q, kv, kr = (normal(*s, dtype=dtype, seed=12 + i) for i, s in enumerate([(n, heads, 192), (n, heads, 256), (n, 64)]))
    q[..., 128] = 1.0
    kr[at, 0] = math.copysign(math.inf, -scale)
    kv[at, :, 128 + column] = math.inf
    got = prefill(q, kv, kr, 128, scale)
    clean, sane = kv.clone(), kr.clone()
    sane[at] = 0.0
    clean[at] = 0.0
    seen = torch.arange(n, device="cuda") <= torch.arange(n, device="cuda")[:, None]
    seen[:, at] = False
    rest = [c for c in range(128) if c != column]
    u = R.half_step(dtype)
    for h in range(0, heads, max(1, heads // 2)):
        x, v = q[:, h].double(), clean[:, h, 128:].double()
        k = torch.cat([clean[:, h, :128], sane], -1).double()
        s = (scale * (x @ k.t())).masked_fill(~seen, -math.inf)
        p = R.softmax(s)
        want = p @ v
        f32 = R.f32_part(torch.where(seen, abs(scale) * (x.abs() @ k.abs().t()), torch.zeros_like(s)))
        tol = u * want.abs() + 6 * u / math.sqrt(3) * (p.square() @ v.square()).sqrt() + f32 * (p @ v.abs()) + R.tiny(u)
        close(got[:, h][:, rest], want[:, rest], tol[:, rest], f"head {h}")
        close(got[:at, h, column], want[:at, column], tol[:at, column], f"head {h}, before the token")
        assert bool(got[at:, h, column].isnan().all()), f"head {h}, from the token on"


@pytest.mark.parametrize("heads", [2, 64])
def test_prefill_infinite_value_that_counts(heads):
    """With ordinary scores: the column is infinite for the queries that see the value."""
    n, column = 900, 100
    q, kv, kr = (normal(*s, dtype=BF16, seed=20 + i) for i, s in enumerate([(n, heads, 192), (n, heads, 256), (n, 64)]))
    for at, value in ((130, math.inf), (650, -math.inf)):
        x = kv.clone()
        x[at, :, 128 + column] = value
        got = prefill(q, x, kr, 128, 0.01)
        assert bool((got[at:, :, column] == value).all())
        assert bool(got[:at].isfinite().all()) and bool(got[..., :column].isfinite().all())
