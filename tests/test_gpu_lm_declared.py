"""What the norms around the residual declare of shared memory: dynamic and static bytes, as `pb_launch_info` says."""
import pytest

from paella_b200 import capi
from tests import lm_util as lu

pytestmark = pytest.mark.gpu
A = 1 << 20      # an address that stands for a buffer: nothing reads it


@pytest.mark.parametrize("dtype,es", [(capi.F32, 4), (capi.BF16, 2)])
@pytest.mark.parametrize("tokens,channels", [(1, 64), (3, 5001), (40, 4096), (16384, 1024), (16384, 4096), (16384, 8192)])
def test_residual_norm(tokens, channels, dtype, es):
    p = capi.ResidualNormParams(tokens=tokens, channels=channels, dtype=dtype, h_dtype=dtype, scale=1.0, eps=1e-6, x_stride=channels, residual_stride=channels, h_stride=channels, y_stride=channels, x=A, residual=A, h=A, y=A)
    li = lu.info("residual_norm", p)
    rows = 2 * 2 * channels * es if tokens == 16384 else 0           # two rows of x and residual, where they come through shared memory
    # besides them the partial sums of two reductions: at least a word a warp for each
    assert li.smem_per_block >= rows + 2 * 4 * (li.threads_per_block // 32) and li.smem_per_block <= rows + 1024
