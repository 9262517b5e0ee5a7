"""GPU tests of the expanded form with eight waves a workgroup (the form that calls with many queries and heads take), against the
definition in 64 bits and with the tolerances of mla_reference; and of few queries over many keys."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import mla_reference as R  # noqa: E402

BF16, F16 = torch.bfloat16, torch.float16


def rnd(*shape, dtype, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(9e9).max()):.3g} x tolerance"


def inputs(widths, dtype, heads, nq, nk, q_scale=2.0, seed=0):
    nope, rope, v = widths
    return (rnd(sum(nq), heads, nope + rope, dtype=dtype, scale=q_scale, seed=seed),
            rnd(sum(nk), heads, nope + v, dtype=dtype, seed=seed + 1), rnd(sum(nk), rope, dtype=dtype, seed=seed + 2))


def run(q, kv, kr, nope, nq, nk, scale):
    from vib3_amd import mla
    cu = [torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device="cuda") for n in (nq, nk)]
    return mla.mla_prefill(q[..., :nope], q[..., nope:], kv, kr, *cu, scale)


def check(got, q, kv, kr, nope, nq, nk, scale):
    want, tol = R.prefill(q[..., :nope], q[..., nope:], kv, kr, nq, nk, nope, scale, R.half_step(got.dtype))
    close(got, want, tol)


RAGGED = [300, 1, 0, 1513, 40, 256], [700, 1, 3, 1400, 41, 256]  # chunks, an empty sequence, more queries than keys


@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64), (128, 32, 64), (64, 64, 128), (128, 64, 64), (64, 32, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ragged(widths, dtype):
    q, kv, kr = inputs(widths, dtype, 64, *RAGGED, seed=1)
    scale = sum(widths[:2]) ** -0.5
    check(run(q, kv, kr, widths[0], *RAGGED, scale), q, kv, kr, widths[0], *RAGGED, scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.5])
def test_scales(scale, dtype):
    q, kv, kr = inputs((128, 64, 128), dtype, 64, *RAGGED, seed=2)
    check(run(q, kv, kr, 128, *RAGGED, scale), q, kv, kr, 128, *RAGGED, scale)


@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinities_and_nan_behind_the_diagonal(widths, dtype):
    """In keys, values and rotary keys, in each eighth of a tile's rows: a query that does not see them stays as it is."""
    nope, rope, v = widths
    heads, n = 64, 1500
    q, kv, kr = inputs(widths, dtype, heads, [n, 300], [n, 300], seed=3)
    want = run(q, kv, kr, nope, [n, 300], [n, 300], 0.08)
    odd, keys = kv.clone(), kr.clone()
    for i in range(8):
        at = 768 + 67 * i  # row 7 i of tile 12 + i or so
        odd[at, i::8, nope + (5 * i) % v] = (math.inf, -math.inf, math.nan)[i % 3]
    odd[1400, :, 3] = math.inf
    keys[1450, 1] = math.nan
    odd[n + 100:] = math.nan
    got = run(q, odd, keys, nope, [n, 300], [n, 300], 0.08)
    for h in range(heads):
        first = 768 + 67 * (h % 8)
        assert torch.equal(got[:first, h], want[:first, h]), h
        assert not bool(got[first:1400, h, (5 * (h % 8)) % v].isfinite().any()), h
        same = [c for c in range(v) if c != (5 * (h % 8)) % v]
        assert torch.equal(got[first:1400, h][:, same], want[first:1400, h][:, same]), h
    assert bool(got[1450:n].isnan().all())
    assert torch.equal(got[n:n + 100], want[n:n + 100]) and bool(got[n + 100:].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,nq,nk", [(2, [64], [30000]), (64, [3, 1], [20000, 17]), (5, [130, 2], [9000, 12000])])
def test_few_queries_over_many_keys(heads, nq, nk, dtype):
    q, kv, kr = inputs((128, 64, 128), dtype, heads, nq, nk, seed=4)
    scale = 192 ** -0.5
    check(run(q, kv, kr, 128, nq, nk, scale), q, kv, kr, 128, nq, nk, scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [8, 20])
def test_a_long_prompt_among_single_queries(heads, dtype):
    nq, nk = [1] * 15 + [4096] + [1] * 16 + [0], list(range(1, 16)) + [4096] + [100] * 16 + [5]
    q, kv, kr = inputs((128, 64, 128), dtype, heads, nq, nk, seed=5)
    scale = 192 ** -0.5
    check(run(q, kv, kr, 128, nq, nk, scale), q, kv, kr, 128, nq, nk, scale)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 130])
def test_sequence_counts(seqs):
    """Blocks are found 64 sequences at a time."""
    nq = [(37 * i) % 90 for i in range(seqs)]
    nq[-1] += 300
    nk = [a + 11 * (i % 4) for i, a in enumerate(nq)]
    q, kv, kr = inputs((64, 32, 64), F16, 128, nq, nk, seed=6)
    check(run(q, kv, kr, 64, nq, nk, 0.1), q, kv, kr, 64, nq, nk, 0.1)
