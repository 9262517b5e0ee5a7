"""GPU tests of the chunk operator's two forms: blocks that a workgroup takes whole (many blocks or sequences) and blocks that are cut into
pieces. Each test sees from the workspace, which only the second one writes, which form the call took."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import gqa_reference as R  # noqa: E402
from test_gpu_gqa import BF16, F16, INF, NAN, Paged, check_chunk, close, ints, rnd  # noqa: E402

MANY = 1030  # sequences: more than the form that cuts plans for
SHAPES = [(32, 8, 128), (9, 3, 64), (16, 2, 256)]


def run(c, heads, nq, whole, many=MANY, scale=None, window=0, sinks=0, q=None):
    """The queries nq of c's sequences among `many` sequences, of which the others have none. Returns (q, output)."""
    from vib3_amd import gqa
    q = rnd(sum(nq), heads, c.dim, dtype=c.dtype, scale=2.0, seed=1) if q is None else q
    places = [many * (2 * i + 1) // (2 * len(nq)) for i in range(len(nq))] if many > len(nq) else list(range(len(nq)))
    table = torch.full((max(many, len(nq)), c.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    count, lens = [0] * len(table), [7] * len(table)
    for i, p in enumerate(places):
        table[p], count[p], lens[p] = c.table[i], nq[i], c.lens[i]
    op = gqa.GqaChunk(c.cache, heads, len(q), len(table))
    op.workspace.fill_(255)
    cu = torch.tensor([0] + count).cumsum(0).int().cuda()
    got = op.launch(q, table, cu, ints(lens), c.dim ** -0.5 if scale is None else scale, window=window, sinks=sinks)
    at = op._space[0] - op.workspace.data_ptr()
    assert bool((op.workspace[at:at + 8] == 255).all()) == whole, "the call did not take the form that is meant to be tested"
    return q, got


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 70), (64, 3)])
@pytest.mark.parametrize("ps", [16, 5, 7])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_whole_blocks(dtype, heads, kv_heads, dim, ps, window, sinks):
    nq, nk = [300, 40, 1, 5, 64, 131, 9], [300, 700, 513, 130, 64, 400, 4]
    c = Paged(nk, kv_heads, dim, dtype, ps, seed=60)
    check_chunk(c, *run(c, heads, nq, True, window=window, sinks=sinks), nq, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,dim,n", [(64, 16, 128, 2100), (128, 16, 64, 2100), (48, 6, 256, 1400)])
@pytest.mark.parametrize("dtype,ps,window,sinks", [(BF16, 64, 0, 0), (F16, 7, 0, 0), (F16, 16, 500, 4), (BF16, 5, 300, 80)])
def test_one_long_prompt_of_whole_blocks(heads, kv_heads, dim, n, dtype, ps, window, sinks):
    c = Paged([n], kv_heads, dim, dtype, ps, seed=61)
    check_chunk(c, *run(c, heads, [n], True, many=1, window=window, sinks=sinks), [n], window=window, sinks=sinks)


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("ps", [16, 7])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_is_not_finite_reaches_only_who_sees_it(dtype, heads, kv_heads, dim, ps, whole):
    """NaN and infinities in keys and values, in the first tile (which is masked) and further ones: queries that see one become NaN, the
    others are as without."""
    nq, nk = [300, 40, 130, 64], [300, 700, 130, 64]
    c = Paged(nk, kv_heads, dim, dtype, ps, seed=62)
    clean = [t.clone() for t in c.v], [t.clone() for t in c.k]
    bad = [150, 680, 20, 63]
    for k, v, b in zip(c.k, c.v, bad):
        k[b], v[b] = NAN, INF
        v[b + 1:b + 2] = -INF
    c.store()
    many = MANY if whole else len(nq)
    q, got = run(c, heads, nq, whole, many=many)
    c.v, c.k = clean
    at = 0
    for s, (a, n, b) in enumerate(zip(nq, nk, bad)):
        pos = torch.arange(n - a, n, device="cuda")
        want, tol = R.attend(q[at:at + a], c.k[s], c.v[s], pos, dim ** -0.5, R.half_step(dtype))
        part, sees = got[at:at + a], pos >= b
        close(part[~sees], want[~sees], tol[~sees], f"sequence {s}: queries before")
        assert bool(part[sees].isnan().all()) and bool(sees.any())
        at += a


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 33)])
@pytest.mark.parametrize("at", [0, 63, 200])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinite_values_count_where_they_are_seen(dtype, heads, kv_heads, dim, at, window, sinks, whole):
    """One infinity (of each sign, in columns of their own): every query that sees it has it, whatever tile it lies in."""
    n = 260
    c = Paged([n], kv_heads, dim, dtype, 16, seed=63)
    c.v[0][at, :, 0], c.v[0][at, :, 1] = INF, -INF
    c.store()
    q, got = run(c, heads, [n], whole, many=MANY if whole else 1, window=window, sinks=sinks)
    pos = torch.arange(n, device="cuda")
    sees = R.visible(pos, n, window, sinks)[:, at]
    assert bool((got[sees][..., 0] == INF).all()) and bool((got[sees][..., 1] == -INF).all())
    want, tol = R.attend(q, c.k[0], c.v[0], pos, dim ** -0.5, R.half_step(dtype), window, sinks)
    close(got[..., 2:], want[..., 2:], tol[..., 2:], "other columns")
    close(got[~sees], want[~sees], tol[~sees], "queries that do not see it")
