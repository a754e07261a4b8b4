"""A layer's prompt step and its continuation with the language-model operators together, as a serving program launches them, against the same in 64 bits from the operators' inputs as they were rounded:
norms around the residual, the fused projection in 8-bit integers, the append to the paged cache, attention of the chunk, the output projection, and at the end the log probabilities of the prompt's own
tokens.  Every step is checked on what the step before left, so that each has its own operator's tolerance."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_chunk import Problem
from tests.test_gpu_lm_logprobs import close, ref as logprobs_ref, run as run_logprobs
from tests.test_gpu_lm_residual import U, near, params as norm_params, ref as norm_ref
from tests.test_gpu_lm_rope import EPS, table

pytestmark = pytest.mark.gpu
HQ, HKV, D, WIDTH, PAGE, VOCAB = 8, 2, 64, 512, 16, 5000


class Layer:
    def __init__(self, g):
        f = lambda *s: lu.randn(g, *s)
        self.norm, self.post = 1.0 + 0.1 * f(WIDTH), 1.0 + 0.1 * f(WIDTH)
        self.qkv = torch.randint(-127, 128, ((HQ + 2 * HKV) * D, WIDTH), generator=g, device="cuda", dtype=torch.int8)
        self.qkv_scale = torch.rand((HQ + 2 * HKV) * D, generator=g, device="cuda") * 1e-3 + 5e-4
        self.out = torch.randint(-127, 128, (WIDTH, HQ * D), generator=g, device="cuda", dtype=torch.int8)
        self.out_scale = torch.rand(WIDTH, generator=g, device="cuda") * 1e-3 + 5e-4
        self.table = table(4096, D)


def dense(x, w, w_scale):
    """the launches of a quantised dense layer, and what they come to from the integers that they leave"""
    t, k, n = x.shape[0], x.shape[1], w.shape[0]
    q, scale, y = torch.empty(t, k, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda"), torch.empty(t, n, dtype=x.dtype, device="cuda")
    lu.launch("int8_quantize", capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=capi.BF16, x_stride=x.stride(0), q_stride=k, x=lu.ptr(x), q=lu.ptr(q), scale=lu.ptr(scale)))
    lu.launch("int8_dense", capi.Int8DenseParams(tokens=t, in_channels=k, out_channels=n, y_dtype=capi.BF16, x_stride=k, w_stride=k, y_stride=n, x=lu.ptr(q), x_scale=lu.ptr(scale), w=lu.ptr(w), w_scale=lu.ptr(w_scale),
                                                  y=lu.ptr(y)))
    return y


@pytest.mark.parametrize("window", [0, 60])
def test_prompt_and_next_tokens(window):
    g = lu.gen(window + 1)
    layer = Layer(g)
    # three sequences: two prompts and one in the middle of its answer; then one token more for each
    lens = [0, 0, 200]
    pages = torch.randperm(60, generator=g, device="cuda").to(torch.int32).view(3, 20).contiguous()
    kc, vc = (lu.randn(g, 60, PAGE, HKV, D).bfloat16() for _ in range(2))
    for new in ([150, 37, 1], [1, 1, 1]):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        t = starts[-1]
        before, lens = list(lens), [a + b for a, b in zip(lens, new)]
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(before, new)]).to(torch.int32).cuda()
        seq = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
        slots = pages[seq, (pos // PAGE).long()].long() * PAGE + pos % PAGE
        x = lu.randn(g, t, WIDTH).bfloat16()                       # the block before: its output, and the residual
        residual = (3.0 * lu.randn(g, t, WIDTH)).bfloat16()
        h, y = torch.empty_like(residual), torch.empty_like(x)
        lu.launch("residual_norm", norm_params("bf16", "bf16", x, None, None, residual, h, layer.norm, y, 1.0))
        qkv = dense(y, layer.qkv, layer.qkv_scale).view(t, HQ + 2 * HKV, D)
        q_out = torch.empty(t, HQ, D, dtype=torch.bfloat16, device="cuda")
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        p = capi.KvAppendParams(dtype=capi.BF16, tokens=t, q_heads=HQ, kv_heads=HKV, head_dim=D, rot_dim=D, max_position=4096, eps=EPS, page_size=PAGE, n_pages=60, k_stride=k.stride(0), k_head_stride=D,
                                v_stride=v.stride(0), v_head_stride=D, page_stride=kc.stride(0), token_stride=kc.stride(1), head_stride=kc.stride(2), k=lu.ptr(k), v=lu.ptr(v), cos_sin=lu.ptr(layer.table),
                                positions=lu.ptr(pos), slots=lu.ptr(slots), k_cache=lu.ptr(kc), v_cache=lu.ptr(vc), q_stride=q.stride(0), q_head_stride=D, q_out_stride=HQ * D, q_out_head_stride=D, q=lu.ptr(q),
                                q_out=lu.ptr(q_out))
        lu.launch("kv_append", p)
        # attention: a problem of the chunk's tests around this cache and these queries
        pr = Problem.__new__(Problem)
        pr.seqs, pr.hkv, pr.group, pr.d, pr.page, pr.ty, pr.window, pr.heads_first = list(zip(new, lens)), HKV, HQ // HKV, D, PAGE, "bf16", window, False
        pr.most_new, pr.most_len, pr.each, pr.tokens, pr.first, pr.scale = max(new), 320, 20, t, starts, D ** -0.5
        pr.table, pr.kc, pr.vc, pr.q, pr.out = pages, kc, vc, q_out, torch.full((t + 1, HQ, D), 9.0, dtype=torch.bfloat16, device="cuda")
        pr.starts, pr.lens = (torch.tensor(s, dtype=torch.int32, device="cuda") for s in (starts, lens))
        params = pr.params()
        lu.launch("chunk_attn", params)
        o = dense(pr.out[:-1].reshape(t, HQ * D), layer.out, layer.out_scale)
        h2, y2 = torch.empty_like(h), torch.empty_like(y)
        lu.launch("residual_norm", norm_params("bf16", "bf16", o, layer.post, None, h, h2, layer.norm, y2, 1.0))
        logits = (y2.float() @ lu.randn(lu.gen(7), WIDTH, VOCAB)).bfloat16()
        targets = torch.randint(0, VOCAB, (t,), generator=g, device="cuda").to(torch.int32)
        _, outs = run_logprobs(logits, targets, 4)
        gu.sync()
        assert gu.error_flag() == 0
        wh, wy, eh, ey = norm_ref(x, None, None, residual, layer.norm, 1.0)
        near(h, wh, eh, "bf16")
        near(y, wy, ey, "bf16")
        pr.check(pr.out[:-1])
        assert bool((pr.out[-1] == 9.0).all())
        wh, wy, eh, ey = norm_ref(o, layer.post, None, h, layer.norm, 1.0)
        near(h2, wh, eh, "bf16")
        near(y2, wy, ey, "bf16")
        want = logprobs_ref(logits, targets, 4, 1.0)
        assert torch.equal(outs["ranks"].cpu(), want["ranks"]) and torch.equal(outs["top_ids"].cpu(), want["top_ids"])
        close(outs["logprobs"], want["logprobs"], U * (320 + 8 * want["logprobs"].abs()))
