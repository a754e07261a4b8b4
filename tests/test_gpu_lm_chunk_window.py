"""Attention of chunks (pb_chunk_attn) under a window whose cache has given up the pages in front of it: their entries in the block table are not read as pages, whatever they hold."""
import pytest

from tests import gpu_util as gu
from tests.test_gpu_lm_chunk import Problem

import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [[(1, 700)], [(1, 5000)], [(1, 700), (1, 20), (1, 3001)], [(4, 900), (2, 70)], [(30, 700), (3, 400)], [(400, 1700), (1, 200)], [(300, 2000)] * 3, [(1, 4100)] * 40],
                         ids=range(8))
@pytest.mark.parametrize("window", [1, 3, 100, 129, 500])
@pytest.mark.parametrize("hkv,group,d,page,ty,heads_first", [(2, 4, 128, 16, "bf16", False), (1, 5, 64, 8, "f16", True), (3, 2, 80, 24, "bf16", False), (1, 1, 96, 128, "f16", False), (1, 16, 128, 40, "bf16", False)])
def test_pages_in_front_of_the_window(seqs, window, hkv, group, d, page, ty, heads_first):
    p = Problem(seqs, hkv, group, d, page, ty, window=window, heads_first=heads_first)
    table = p.table.clone()
    for i, (n, l) in enumerate(seqs):
        gone = max(0, l - n - window + 1) // page                  # whole pages in front of what the first new token sees
        pages = table[i, :gone].long()
        p.kc[pages], p.vc[pages] = float("nan"), float("inf")
        p.table[i, :gone] = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31, p.kc.shape[0]], dtype=torch.int64).to(torch.int32).repeat(gone)[:gone].to("cuda")
    got = p.run()
    assert gu.error_flag() == 0
    p.table.copy_(table)
    p.check(got)
    # the page that the first row's window begins in is one that has to be there
    i = max(range(len(seqs)), key=lambda i: seqs[i][1])
    n, l = seqs[i]
    p.table[i, max(0, l - n - window + 1) // page] = -1
    p.run()
    assert gu.error_flag(reset=True) == 0x304
