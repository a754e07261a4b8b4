"""The softmax of pb_prefix_attn where single keys of the prefix are odd."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_attn import Problem

pytestmark = pytest.mark.gpu


def formula(p, i, without):
    """Sequence i's result in 64 bits as if the prefix's key `without` were not there, and the bound that tests/test_gpu_lm_attn.py derives."""
    keep = torch.arange(p.prefix + p.lens[i], device="cuda") != without
    k, v = (p.tokens(c, i)[keep] for c in (p.kc, p.vc))
    q = p.q[i].double().view(p.hkv, p.group, p.d)
    s = torch.einsum("hgd,nhd->hgn", q, k) * p.scale
    size = torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()).max() * abs(p.scale)
    w = torch.softmax(s, -1)
    ref, mag = torch.einsum("hgn,nhd->hgd", w, v), torch.einsum("hgn,nhd->hgd", w, v.abs())
    half = lu.HALF_STEP[p.ty]
    small = (p.d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + s.abs().max() * 1.45) + (len(v) + 40) * 2.0 ** -23
    return ref.flatten(0, 1), ((half + small) * mag + half * ref.abs() + lu.TINY[p.ty] * 2).flatten(0, 1)


# one row tile, whose key tiles two groups share, and two; neighbouring keys take different paths; the first tile's halves and the last one's
@pytest.mark.parametrize("kernel", ["0", "1"])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("b", [3, 40])
@pytest.mark.parametrize("at", [*range(8), *range(64, 72), *range(192, 200)])
def test_a_nan_or_infinity_in_one_key_of_the_prefix(kernel, ty, b, at, monkeypatch):
    monkeypatch.setenv("PB_ATTN_PREFIX", kernel)
    p = Problem([4] * b, 1, 4, 64, 200, 16, ty)
    key = p.kc.view(-1, 64)[p.rows(p.prefix_pages, 200)[at]]
    key[5] = float("nan")
    assert bool(p.run().isnan().all())                           # all rows see it
    key[5] = float("inf")                                        # scores of +infinity make a row NaN, those of -infinity leave it to the other keys
    got, up = p.run(), p.q[:, :, 5] > 0
    assert bool((p.q[:, :, 5] != 0).all())
    assert bool(got[up].isnan().all()) and bool(got[~up].isfinite().all())
    for i in (0, 1, b - 1):
        ref, bound = formula(p, i, at)
        off = (got[i].double() - ref).abs() / bound
        assert bool((off[~up[i]] <= 1).all())
    assert gu.error_flag() == 0
