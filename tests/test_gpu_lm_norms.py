"""Where the norms of pb_qk_rope end: the sum of a head's squares is held in fp32."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_rope import EPS, rope_params, table

pytestmark = pytest.mark.gpu


# few tokens and so many that a group takes several heads; sizes up to the range's end and behind it
@pytest.mark.parametrize("t", [3, 20000])
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("d,inside,outside", [(128, 1.6e18, 1.7e18), (64, 2.2e18, 3.3e38), (256, 1.1e18, 1e20)])
def test_sums_of_squares_up_to_the_range_of_fp32(ty, t, d, inside, outside):
    """A head of equal values is normed to ones (one half step each of the root, the quotient and the products, beside the output's) as long as the sum is finite;
    behind that it is zeros, and its neighbours are what they are."""
    q = torch.ones(t, 4, d, device="cuda", dtype=lu.TYPES[ty])
    q[:, 1], q[:, 2] = inside, outside
    assert d * float(q[0, 1, 0]) ** 2 < 3.4028234e38 < d * float(q[0, 2, 0]) ** 2
    out, w, tab, pos = torch.empty_like(q), torch.ones(d, device="cuda"), table(4, d), torch.zeros(t, device="cuda", dtype=torch.int32)
    lu.launch("qk_rope", rope_params(ty, q, q[:, :0], out, out[:, :0], w, None, tab, pos, d, 0))
    gu.sync()
    bound = lu.HALF_STEP[ty] + 32 * 2.0 ** -24
    one = (1.0 + EPS) ** -0.5
    assert bool(((out[:, [0, 3]].double() - one).abs() <= bound).all()) and bool(((out[:, 1].double() - 1.0).abs() <= bound).all())
    assert bool((out[:, 2] == 0).all()) and gu.error_flag() == 0
