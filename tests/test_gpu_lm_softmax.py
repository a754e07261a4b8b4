"""The softmax of pb_prefix_attn, seen closer than its 16-bit results show it: odd keys of the prefix, and the exponentials themselves.

A row's sum of exponentials is held in fp32 beside the prefix's parts at the end of the scratch memory, [row tile][key head][part][128] pairs (maximum, sum)."""
import math

import numpy as np
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


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("b", [100, 250])
def test_exponentials(ty, b, monkeypatch):
    """A prefix of 128 keys of which two count: the first has score 0, which is each row's maximum so far, another in the second half of the tile has a score of the row's own,
    from far below to the 2^8 above the maximum that it may have before the maximum follows.  The exponent that the kernel forms in one rounding is known exactly; 2^x of it is
    off by 2^-22 (on either path), and the sum of the two by 2^-24."""
    monkeypatch.setenv("PB_ATTN_PREFIX", "1")
    shift = 5.0 if ty == "f16" else 0.0
    scale = np.float32(math.log(2.0))
    c = np.float32(scale * np.float32(1.4426950408889634))
    for at in range(64, 72):
        p = Problem([0] * b, 1, 1, 64, 128, 16, ty, most=0)
        p.scale = float(scale)
        k = torch.zeros(128, 64, device="cuda", dtype=lu.TYPES[ty])
        k[:, 2] = -30000.0
        k[0, 2] = k[at, 2] = 0.0
        k[at, 1] = 1.0
        p.kc.view(-1, 64)[p.rows(p.prefix_pages, 128)] = k
        score = (torch.rand(b, generator=lu.gen(at), device="cuda") * 28 - 20).to(lu.TYPES[ty])
        p.q.zero_()
        p.q[:, 0, 1], p.q[:, 0, 2] = score, 1.0
        p.run()
        n = len(p.scratch) - 16
        tiles = -(-b // 128)
        m, total = p.scratch[:n].view(torch.float32)[-tiles * 256:].view(-1, 2)[:b].double().cpu().numpy().T
        e = (score.double().cpu().numpy() * np.float64(c) + shift).astype(np.float32)
        one, other = 2.0 ** shift, np.exp2(np.float64(e))
        assert (m == 0).all()
        off = np.abs(total - one - other)
        bound = 2.0 ** -22 * (one + other) + 2.0 ** -24 * total
        assert (off <= bound).all(), (off / bound).max()
