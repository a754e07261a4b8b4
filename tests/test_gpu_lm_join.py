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
