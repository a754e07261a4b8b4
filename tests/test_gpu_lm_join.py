"""How pb_prefix_attn joins a row's parts: clusters of blocks that read one another's shared memory, heads that do not fill a row of it, groups of query heads that fill their blocks or do not."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_attn import Problem

pytestmark = pytest.mark.gpu


# two, four and eight blocks a sequence and key head; every size of head on either side of the two that rows have
@pytest.mark.parametrize("lens,hkv,group,prefix", [([300, 5], 2, 8, 0), ([1025, 0, 700], 1, 3, 0), ([2300], 2, 16, 0), ([900, 1], 1, 20, 513), ([300] * 130, 2, 4, 70)])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("kernel", ["0", "1"])
def test_parts_of_heads_of_any_size(kernel, d, lens, hkv, group, prefix, monkeypatch):
    monkeypatch.setenv("PB_ATTN_PREFIX", kernel)
    p = Problem(lens, hkv, group, d, prefix, 16, "f16" if d % 16 else "bf16")
    first = p.run().clone()
    p.check(first, only=range(3))
    params = p.params()
    for _ in range(10):                                          # block after block on the same SMs
        lu.launch("prefix_attn", params)
    gu.sync()
    assert torch.equal(p.out[:-1], first) and bool((p.out[-1] == 9.0).all())
    assert gu.error_flag() == 0


@pytest.mark.parametrize("group,fit", [(1, 3), (8, 3), (9, 2), (16, 2), (40, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_blocks_that_an_sm_holds(d, group, fit):
    """What the rule for own tokens' blocks says of them: 228 KB of shared memory and 65536 registers for blocks of 128 threads, 1 KB of each reserved."""
    li = lu.info("prefix_attn", Problem([5], 1, group, d, 0, 16).params())
    assert min(228 * 1024 // (li.smem_per_block + 1024), 65536 // (-(-li.regs_per_thread // 8) * 8 * 128)) == fit


@pytest.mark.parametrize("lens,hkv,group", [([70, 0, 31, 5] * 20, 4, 12), ([9] * 40, 8, 16), ([40, 3] * 41, 2, 20)])
def test_more_blocks_behind_a_prefix_than_fit_at_once(lens, hkv, group):
    """300 to 444 blocks of large groups: some come in only when others, which wait for the prefix, have left."""
    p = Problem(lens, hkv, group, 128, 3000, 32, most=100)
    p.check(p.run(), only=range(0, len(lens), 13))
    assert 296 < lu.info("prefix_attn", p.params()).num_blocks <= 444 and gu.error_flag() == 0
