"""Rows in reverse order (negative strides) give the same results as in order, bit for bit."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_attn import Problem
from tests.test_gpu_lm_int8 import dense_params, operands
from tests.test_gpu_lm_rope import append_params, cache, heads, rope_params, table

pytestmark = pytest.mark.gpu


def last(t):
    """address of the last row"""
    return t.data_ptr() + (t.shape[0] - 1) * t.stride(0) * t.element_size()


@pytest.mark.parametrize("t,k,n", [(5, 300, 130), (300, 260, 600)])
def test_dense_and_quantiser(t, k, n):
    g = lu.gen(t)
    x, w, xs, ws = operands(g, t, k, n)
    y, z = torch.empty(t, n, device="cuda", dtype=torch.bfloat16), torch.full((t, n), 9.0, device="cuda", dtype=torch.bfloat16)
    lu.launch("int8_dense", dense_params(x, xs, w, ws, k, None, y, "bf16"))
    p = dense_params(x, xs, w, ws, k, None, z, "bf16")
    p.y, p.y_stride = last(z), -z.stride(0)
    lu.launch("int8_dense", p)
    f = lu.randn(g, t, k).bfloat16()
    q, r, s = torch.empty(t, 304, device="cuda", dtype=torch.int8), torch.empty(t, 304, device="cuda", dtype=torch.int8), torch.empty(2, t, device="cuda")
    p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=capi.BF16, x_stride=k, q_stride=304, x=lu.ptr(f), q=lu.ptr(q), scale=lu.ptr(s[0]))
    lu.launch("int8_quantize", p)
    p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=capi.BF16, x_stride=-k, q_stride=-304, x=last(f), q=last(r), scale=lu.ptr(s[1]))
    lu.launch("int8_quantize", p)
    gu.sync()
    assert torch.equal(y, z.flip(0)) and torch.equal(q[:, :k], r[:, :k]) and torch.equal(s[0], s[1].flip(0))


@pytest.mark.parametrize("t", [7, 20000])
def test_rope_and_append(t):
    g, d = lu.gen(t), 64
    x, tab = heads(g, t, 8, d, "bf16"), table(50, d)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    pos = torch.randint(0, 50, (t,), generator=g, device="cuda", dtype=torch.int32)
    back = pos.flip(0).contiguous()
    o = [torch.empty(t, 6, d, device="cuda", dtype=x.dtype) for _ in range(2)]
    lu.launch("qk_rope", rope_params("bf16", q, k, o[0][:, :4], o[0][:, 4:], None, None, tab, pos, d, 0))
    p = rope_params("bf16", q, k, o[1][:, :4], o[1][:, 4:], None, None, tab, back, d, 0)
    p.q, p.k, p.q_out, p.k_out = last(q), last(k), last(o[1][:, :4]), last(o[1][:, 4:])
    p.q_stride, p.k_stride, p.q_out_stride, p.k_out_stride = -p.q_stride, -p.k_stride, -p.q_out_stride, -p.k_out_stride
    lu.launch("qk_rope", p)
    pages = t // 16 + 2
    c = [[cache(pages, 16, 2, d, "bf16", False) for _ in range(2)] for _ in range(2)]
    slots = torch.randperm(pages * 16, generator=g, device="cuda")[:t].contiguous()
    lu.launch("kv_append", append_params("bf16", k, v, *c[0], slots, 16, tab, pos, d))
    p = append_params("bf16", k, v, *c[1], slots, 16, tab, pos, d)          # pages from the last to the first
    p.k_cache, p.v_cache, p.page_stride = last(c[1][0]), last(c[1][1]), -p.page_stride
    lu.launch("kv_append", p)
    gu.sync()
    assert torch.equal(o[0], o[1])                               # (each row where it was: input, output and position in reverse)
    assert torch.equal(c[0][0], c[1][0].flip(0)) and torch.equal(c[0][1], c[1][1].flip(0)) and gu.error_flag() == 0


@pytest.mark.parametrize("kernel", ["0", "1"])
@pytest.mark.parametrize("lens", [[5, 0, 40], [3] * 50])
def test_attention(kernel, lens, monkeypatch):
    monkeypatch.setenv("PB_ATTN_PREFIX", kernel)
    p = Problem(lens, 2, 4, 64, 200, 16)
    ref = p.run().clone()
    p.q = p.q.flip(0).contiguous()
    params, out = p.params(), p.out[:-1]
    out.fill_(9.0)
    params.q, params.q_stride, params.out, params.out_stride = last(p.q), -p.q.stride(0), last(out), -out.stride(0)
    lu.launch("prefix_attn", params)
    gu.sync()
    assert torch.equal(out.flip(0), ref) and bool((p.out[-1] == 9.0).all()) and gu.error_flag() == 0
