"""GPU test of the decode's rounding: probabilities go to the matrix cores in two summands, so that a result is rounded to 16 bits once."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import gqa_reference as R  # noqa: E402
from test_gpu_gqa import BF16, F16, Paged, close, decode  # noqa: E402


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (9, 3, 64), (16, 2, 256), (17, 1, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens", [[37, 300, 1], [4000, 65, 700]])
def test_results_are_rounded_once(lens, dtype, heads, kv_heads, dim):
    """u |ref| for the result, and of sum_j p_j |v_j| the two summands' 2^-15 (bf16: what is cut off is below 2^-7 of the number and rounded
    by 2^-8 of itself) or 2^-21 (f16: 2^-10 and 2^-11), f16's 2^-36 of the largest probability a token (the smallest numbers' spacing), and the
    work in f32 (mla_reference.f32_part)."""
    c = Paged(lens, kv_heads, dim, dtype, 16, seed=80)
    q, got = decode(c, heads, list(enumerate(lens)))
    u, scale = R.half_step(dtype), dim ** -0.5
    for s, n in enumerate(lens):
        want, tol = torch.zeros(heads, dim, dtype=torch.float64, device="cuda"), torch.zeros(heads, dim, dtype=torch.float64, device="cuda")
        for h in range(heads):
            x, y, v = q[s, h].double(), c.k[s][:, h * kv_heads // heads].double(), c.v[s][:, h * kv_heads // heads].double()
            p = R.softmax((scale * (y @ x))[None])
            f32 = R.f32_part((abs(scale) * (y.abs() @ x.abs()))[None])
            want[h] = (p @ v)[0]
            part = (2.0 ** -15 if dtype == BF16 else 2.0 ** -21) * (p @ v.abs())[0]
            if dtype == F16:
                part = part + 2.0 ** -36 * p.max() * v.abs().sum(0)
            tol[h] = u * want[h].abs() + (1 + u) * (part + (f32 * (p @ v.abs()))[0]) + R.tiny(u)
        close(got[s], want, tol, f"{n} tokens")
