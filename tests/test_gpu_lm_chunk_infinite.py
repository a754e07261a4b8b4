"""Attention of chunks (pb_chunk_attn) where every key that a row sees scores -infinity: the softmax of nothing but -infinity is NaN, and only rows that see no token at all get zeros."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_chunk import Problem

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("seqs,window,upto", [([(1, 1)], 0, 1), ([(3, 3), (1, 40)], 0, 2), ([(5, 3)], 0, 1), ([(1, 700)], 0, 700), ([(1, 700)], 0, 699), ([(2, 4000)], 50, 3999), ([(60, 60)], 0, 17),
                                              ([(300, 300), (2, 9)], 0, 140), ([(300, 290)], 0, 3), ([(300, 2000)], 100, 1850), ([(300, 9000)], 0, 8800), ([(300, 9000)], 0, 8650)], ids=range(12))
@pytest.mark.parametrize("group,d,ty", [(4, 128, "bf16"), (1, 64, "f16"), (5, 80, "bf16")])
def test_rows_that_see_only_keys_of_minus_infinity(seqs, window, upto, group, d, ty):
    p = Problem(seqs, 2, group, d, 16, ty, window=window)
    n, l = seqs[0]
    p.q[:, :, 5] = p.q[:, :, 5].abs() + 0.1
    p.kc.view(-1, 2, d)[p.rows(0, l)[:upto], 1, 5] = -INF          # of key head 1
    got = p.run()
    assert gu.error_flag() == 0
    pos = torch.arange(l - n, l, device="cuda")
    at = torch.arange(l, device="cuda")
    seen = at <= pos[:, None]
    if window:
        seen &= at > pos[:, None] - window
    nothing = seen.any(1) & ~(seen & (at >= upto)).any(1)
    mine = got[:n].view(n, 2, group, d)
    assert bool(nothing.any()) == bool(mine.isnan().any()) and bool(mine[nothing, 1].isnan().all()) and not bool(mine[~nothing].isnan().any()) and not bool(mine[:, 0].isnan().any())
    assert bool((mine[pos < 0] == 0).all())
    # the other rows, in 64 bits: keys of -infinity have no part in them
    k, v, q = p.cached(p.kc, 0)[:, 1], p.cached(p.vc, 0)[:, 1], p.q[:n].view(n, 2, group, d)[:, 1].double()
    live = ~nothing & (pos >= 0)
    if bool(live.any()):
        k = k.clone()
        k[:upto] = 0.0
        use = (seen & (at >= upto))[live]
        s = torch.einsum("nhd,md->hnm", q[live], k) * p.scale
        w = torch.softmax(s.masked_fill(~use, -INF), -1)
        ref, mag = torch.einsum("hnm,md->nhd", w, v), torch.einsum("hnm,md->nhd", w, v.abs())
        size, half = float(torch.einsum("nhd,md->hnm", q[live].abs(), k.abs()).max() * p.scale), lu.HALF_STEP[ty]
        small = (d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + float(s.abs().max()) * 1.45) + (min(l, window or l) + 40) * 2.0 ** -23      # as `Problem.check`
        off = (mine[live, 1].double() - ref).abs()
        assert bool((off <= (half + small) * mag + half * ref.abs() + lu.TINY[ty] * 2).all())
