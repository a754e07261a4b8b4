"""Log probabilities of fp32 logits that are large beside the differences between them (pb_logprobs), whose exponents x c - m c are differences of large products: against 64 bits, with the
tolerances of `test_gpu_lm_logprobs.py`."""
import math

import pytest
import torch

from tests import lm_util as lu
from tests.test_gpu_lm_logprobs import check, some

pytestmark = pytest.mark.gpu


def near(g, t, v, top, step):
    """Rows whose largest logit is `top`, with neighbours up to six steps below it and a third far below."""
    x = (top - step * torch.randint(0, 7, (t, v), generator=g, device="cuda").double()).float()
    x[:, v // 2] = top
    far = torch.rand(t, v, generator=g, device="cuda") < 0.3
    return torch.where(far, torch.full_like(x, top - 4000 * step), x)


# the largest logit times the scale; in fp32 its neighbours are 16 (2e8) to 2^40 apart
@pytest.mark.parametrize("size", [1e6, 3e7, 2e8, 2.7e8, 5.4e8, 1e9, 1.5e9, 2.2e9, 3161437440.0, 3.3e9, 4.2e9, 5.3e9, 9e9, 3e11, 1e19])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [1.0, 1e6, 0.7])
@pytest.mark.parametrize("t,v", [(3, 40001), (600, 2003)])
def test_large_logits(size, sign, scale, t, v):
    g = lu.gen(13)
    top = float(torch.tensor(sign * size / scale, dtype=torch.float32))
    step = 2.0 ** (math.frexp(abs(top))[1] - 24)                   # of fp32 there
    check(near(g, t, v, top, step), some(g, t, v), 4, scale)
    # differences that count: some steps of the exponentials' size, as far as fp32 has them there
    check(near(g, t, v, top, max(step, step * round(1.0 / (scale * step)))), some(g, t, v), 4, scale)


@pytest.mark.parametrize("size", [2.2e9, 3.3e9, 4.2e9])
def test_large_logits_behind_ordinary_ones(size):
    """The first vectors take the common way, with sums of their own, until the large ones come."""
    g, v = lu.gen(14), 60000
    x = 3.0 * lu.randn(g, 5, v)
    x[:, v - 20000:v - 1] = size - 256.0 * torch.randint(0, 3, (5, 19999), generator=g, device="cuda").float()
    x[4, :v // 2] = -size
    check(x, some(g, 5, v), 8)
