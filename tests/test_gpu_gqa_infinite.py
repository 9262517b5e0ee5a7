"""GPU tests of infinite values that a query sees with a small probability: as long as that is a normal f32 number they give an
infinity, whatever the 16-bit type's range, the tile and the form of the call."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import gqa_reference as R  # noqa: E402
from test_gpu_gqa import BF16, F16, INF, NAN, Paged, close, decode, ints  # noqa: E402
from test_gpu_gqa_forms import MANY, SHAPES, run  # noqa: E402


def below(n, kv_heads, dim, dtype, at, gap, ps=16):
    """n tokens with equal scores but for token `at`, whose key lies gap nats below and whose value holds infinities and NaN."""
    c = Paged([n], kv_heads, dim, dtype, ps, seed=70)
    c.k[0].zero_()
    c.k[0][at, :, 0] = -gap
    c.v[0][at, :, 0], c.v[0][at, :, 1], c.v[0][at, :, 2] = INF, -INF, NAN
    c.store()
    return c


def ones(n, heads, dim, dtype):
    q = torch.zeros(n, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    return q


def check(c, q, got, pos, at, gap, window=0, sinks=0):
    sees = R.visible(pos, c.lens[0], window, sinks)[:, at]
    assert bool(sees.any())
    if gap < 87:  # the probability is above 2^-126
        assert bool((got[sees][..., 0] == INF).all()) and bool((got[sees][..., 1] == -INF).all()), f"{gap} nats below"
    else:  # 0, but for the queries that see nothing else
        others = sees & (R.visible(pos, c.lens[0], window, sinks).sum(-1) > 1)
        assert bool(got[others][..., :2].isnan().all())
    assert bool(got[sees][..., 2].isnan().all())
    want, tol = R.attend(q, c.k[0], c.v[0], pos, 1.0, R.half_step(c.dtype), window, sinks)
    close(got[..., 3:], want[..., 3:], tol[..., 3:], "other columns")
    close(got[~sees], want[~sees], tol[~sees], "queries that do not see it")


@pytest.mark.parametrize("gap", [40.0, 84.0, 120.0])
@pytest.mark.parametrize("whole,at,window,sinks", [(True, 10, 0, 0), (True, 150, 200, 0), (False, 150, 0, 0), (False, 3, 100, 5)])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chunk(dtype, heads, kv_heads, dim, whole, at, window, sinks, gap):
    n = 400
    c = below(n, kv_heads, dim, dtype, at, gap)
    q, got = run(c, heads, [n], whole, many=MANY if whole else 1, scale=1.0, window=window, sinks=sinks, q=ones(n, heads, dim, dtype))
    check(c, q, got, torch.arange(n, device="cuda"), at, gap, window, sinks)


@pytest.mark.parametrize("gap", [40.0, 84.0, 120.0])
@pytest.mark.parametrize("n,at,ps", [(40, 7, 16), (400, 399, 7), (9000, 5000, 64)])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES + [(17, 1, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode(dtype, heads, kv_heads, dim, n, at, ps, gap):
    """Rows that one share holds and rows that many do, beside others that do not see the token."""
    c = below(n, kv_heads, dim, dtype, at, gap, ps)
    lens = [n, at + 1, max(at, 1), n]
    q = ones(4, heads, dim, dtype)
    _, got = decode(c, heads, [(0, x) for x in lens], scale=1.0, q=q)
    check(c, q, got, torch.tensor(lens, device="cuda") - 1, at, gap)
    _, got = decode(c, heads, [(0, x) for x in lens], scale=1.0, q=q, window=30, sinks=at + 1)
    check(c, q, got, torch.tensor(lens, device="cuda") - 1, at, gap, 30, at + 1)


@pytest.mark.parametrize("rows", [5, 600])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_are_all_minus_infinity(dtype, heads, kv_heads, dim, rows):
    """Nothing has a probability: zeros, also where values are not finite; NaN scores and +infinity give NaN."""
    n = 300
    c = Paged([n], kv_heads, dim, dtype, 16, seed=71)
    c.k[0].zero_()
    c.k[0][..., 0] = -INF
    c.v[0][5, :, 0], c.v[0][200, :, 1] = INF, NAN
    c.store()
    q = ones(n, heads, dim, dtype)
    lens = [n - i % n for i in range(rows)]
    for whole in (True, False):
        assert bool((run(c, heads, [n], whole, many=MANY if whole else 1, q=q)[1] == 0).all())
        assert bool(run(c, heads, [n], whole, many=MANY if whole else 1, q=-q)[1].isnan().all())
    one = q[:1].expand(rows, heads, dim)
    assert bool((decode(c, heads, [(0, x) for x in lens], q=one)[1] == 0).all())
    assert bool(decode(c, heads, [(0, x) for x in lens], q=-q[:1].expand(rows, heads, dim))[1].isnan().all())
    c.v[0].fill_(NAN)
    c.store()
    assert bool((decode(c, heads, [(0, x) for x in lens], q=one)[1] == 0).all())
    assert bool((run(c, heads, [n], True, q=q)[1] == 0).all()) and bool((run(c, heads, [n], False, many=1, q=q)[1] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,first", [(300, 299), (300, 150), (9000, 8999), (9000, 4000), (9000, 0)])
def test_values_that_are_nan_beside_infinities(dtype, n, first):
    """Tokens from `first` on hold NaN in two columns; an infinity in a third one counts little (40 nats below)."""
    c = Paged([n], 2, 128, dtype, 16, seed=73)
    c.k[0].zero_()
    c.k[0][7, :, 0] = -40.0
    c.v[0][first:, :, 4:6], c.v[0][7, :, 9] = NAN, INF
    c.store()
    q = ones(64, 8, 128, dtype)
    for got in (decode(c, 8, [(0, n)] * 3, scale=1.0, q=q[:3])[1], run(c, 8, [64], False, many=1, scale=1.0, q=q)[1][-1:],
                run(c, 8, [64], True, scale=1.0, q=q)[1][-1:]):
        assert bool(got[..., 4:6].isnan().all()) and bool((got[..., 9] == INF).all())
        others = [i for i in range(128) if i not in (4, 5, 9)]
        assert bool(got[..., others].isfinite().all())


def test_both_infinities_and_small_probabilities_together():
    """A column's infinities of both signs give NaN, also where one of them counts 2^-90 of the other."""
    from vib3_amd import gqa
    n = 200
    c = Paged([n], 1, 64, F16, 16, seed=72)
    c.k[0].zero_()
    c.k[0][20, 0, 0], c.k[0][90, 0, 0] = -62.0, -1.0
    c.v[0][20, 0, :2], c.v[0][90, 0, 0], c.v[0][90, 0, 2] = INF, -INF, INF
    c.store()
    q = ones(n, 4, 64, F16)
    for got in (gqa.GqaChunk(c.cache, 4, n, 1).launch(q, c.table, ints([0, n]), ints([n]), 1.0)[-1],
                decode(c, 4, [(0, n)], scale=1.0, q=q[:1])[1][0]):
        assert bool(got[:, 0].isnan().all()) and bool((got[:, 1] == INF).all()) and bool((got[:, 2] == INF).all())
        assert bool(got[:, 3:].isfinite().all())
