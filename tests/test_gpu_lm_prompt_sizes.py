"""The operators of prompts at the sizes where they go other ways: many sequences, long caches whose ranges go round, rows through rings, selections that do not fit at first, one scratch memory for launches that follow one
another.  Tolerances are those of each operator's own tests."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests import test_gpu_lm_logprobs as lp
from tests import test_gpu_lm_residual as rn
from tests.test_gpu_lm_chunk import Problem

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


# more sequences than the plan has threads, more pairs of row tiles than it keeps in shared memory, sequences of few rows among them or not
@pytest.mark.parametrize("seqs", [[(10, 12)] * 2100, [(1, 5), (9, 30)] * 1100, [(0, 4), (70, 71), (2, 2)] * 700, [(600, 700)] * 30 + [(0, 0)] * 1500 + [(33, 40)]], ids=range(4))
def test_many_sequences(seqs):
    p = Problem(seqs, 1, 4, 64, 8)
    p.check(p.run())
    assert gu.error_flag() == 0


def test_long_caches_in_several_rounds():
    p = Problem([(2048, 40000)], 8, 4, 128, 64)
    p.check(p.run())
    assert gu.error_flag() == 0


# one sequence's next tokens behind a long cache: few rows that all blocks share out
@pytest.mark.parametrize("window", [0, 90000])
@pytest.mark.parametrize("seqs,hkv,group", [([(1, 100001)], 2, 4), ([(3, 90000)], 1, 5), ([(1, 110000), (1, 50), (0, 7)], 1, 8), ([(1, 70000), (1, 0), (2, 60001)], 2, 3)])
def test_few_rows_of_long_caches(seqs, hkv, group, window):
    p = Problem(seqs, hkv, group, 128, 64, window=window)
    p.check(p.run())
    assert gu.error_flag() == 0


def test_one_scratch_for_launches_that_follow_one_another():
    a, b = Problem([(300, 1500), (40, 900)], 2, 4, 128, 32), Problem([(20, 5000), (700, 900)], 2, 4, 128, 32, seed=3)
    pa, pb = a.params(), b.params()
    shared = torch.full((max(pa.scratch_bytes, pb.scratch_bytes),), 255, dtype=torch.uint8, device="cuda")
    pa.scratch = pb.scratch = lu.ptr(shared)
    for _ in range(20):
        lu.launch("chunk_attn", pa)
        lu.launch("chunk_attn", pb)
    gu.sync()
    a.check(a.out[:-1])
    b.check(b.out[:-1])


def test_too_little_scratch_is_refused():
    from paella_b200 import capi
    import ctypes as C
    p = Problem([(300, 1500)], 2, 4, 128, 32).params()
    p.scratch_bytes -= 1
    assert capi.load().pb_chunk_attn_launch(C.byref(p), torch.cuda.current_stream().cuda_stream, 0, None) == -2
    p.scratch_bytes, p.scratch = p.scratch_bytes + 1, None
    assert capi.load().pb_chunk_attn_launch(C.byref(p), torch.cuda.current_stream().cuda_stream, 0, None) == -2


@pytest.mark.parametrize("ty,hty", rn.TYPES)
@pytest.mark.parametrize("t,c", [(1500, 2048), (1200, 2056), (1000, 4096), (700, 8192), (400, 16384), (2000, 1024)])
@pytest.mark.parametrize("post,gate,residual,outs", [(True, "token", True, "hy"), (True, "channel", True, "hy"), (False, "none", False, "y"), (False, "token", True, "h"), (True, "none", False, "hy")])
def test_norms_of_many_rows(ty, hty, t, c, post, gate, residual, outs):
    g = lu.gen(c + t)
    x = rn.rows(g, t, c, ty, 16)
    r = rn.rows(g, t, c, hty, 8) if residual else None
    gt = {"none": None, "channel": rn.rows(g, 1, c, ty), "token": rn.rows(g, t, c, ty)}[gate]
    pw, w = lu.randn(g, c) if post else None, lu.randn(g, c)
    h = torch.full((t, c), 7.0, device="cuda", dtype=lu.TYPES[hty]) if "h" in outs else None
    y = torch.full((t, c), 7.0, device="cuda", dtype=lu.TYPES[ty]) if "y" in outs else None
    p = rn.params(ty, hty, x, pw, gt, r, h, w, y, -0.5)
    lu.launch("residual_norm", p)
    gu.sync()
    wh, wy, eh, ey = rn.ref(x, pw, gt, r, w, -0.5)
    if h is not None:
        rn.near(h, wh, eh, hty)
    if y is not None:
        rn.near(y, wy, ey, ty)
    li = lu.info("residual_norm", p)
    assert lu.records("residual_norm", p) == (li.num_blocks, li.num_blocks) and gu.error_flag() == 0


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v,top", [(600, 3001, 7), (1300, 70, 20), (700, 20001, 0), (2000, 1, 1), (601, 32, 32)])
def test_logits_of_many_rows(ty, t, v, top):
    g = lu.gen(t + v)
    lp.check(lp.logits(g, t, v, ty), lp.some(g, t, v), top, 1.3)


# the large logits with the vectors of a few threads (256 or 128 of them, 32 bytes a vector): more of them than there is room for
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("t", [150, 600])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed", "equal"])
@pytest.mark.parametrize("few", [3, 60])
def test_selections_that_do_not_fit_at_first(ty, t, order, few):
    threads, vector, v = 128 if t >= 592 else 256, 8 if ty == "f32" else 16, 65536
    g = lu.gen(few)
    x = lu.randn(g, t, v).clamp(-3, 3)
    at = torch.arange(v, device="cuda")
    mine = (at // vector) % threads < few
    n = int(mine.sum())
    values = {"rising": torch.linspace(10, 20, n), "falling": torch.linspace(20, 10, n), "mixed": torch.linspace(10, 20, n)[torch.randperm(n, generator=torch.Generator().manual_seed(1))], "equal": torch.full((n,), 12.0)}[order]
    x[:, mine] = values.cuda()
    lp.check(x.to(lu.TYPES[ty])[:8].repeat(t // 8 + 1, 1)[:t].contiguous(), lp.some(g, t, v), 32)


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [3, 160, 600])
def test_rows_of_nan_and_infinity(ty, t):
    g, v = lu.gen(2), 9001
    x = lp.logits(g, t, v, ty)
    x[0] = NAN
    x[1, 100:8000] = INF
    x[2, ::2] = NAN
    x[2, 1::2] = -INF
    lp.check(x, lp.some(g, t, v), 32)
