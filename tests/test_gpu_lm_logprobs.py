"""Log probabilities, ranks, entropies and likeliest tokens (pb_logprobs) against 64 bits; ranks and tokens have to be equal.

Tolerance, in u = 2^-24, a rounding of fp32.  d = (x - m) (s log2 e) has four roundings (the constant's two, the difference, the product), the exponential is off by
4 u, so that a term of S is off by (4 |d| + 4) u, relative; the mean of |d| over the terms is at most the entropy's 18 powers of two here.  A thread adds up
to 200 pairs, five shuffles, 16 warps, five shuffles and eight blocks follow: S is off by less than (72 + 4 + 240) u = 320 u.  log p = d - log S is off by
that and by 6 roundings of its own size; the entropy log S - E / S by 320 u for S, and 320 u + 2 u of E / S, which is at most the entropy and log S."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


def run(x, targets, top, scale=1.0, ty=None, stream=None, outs=None, only=None):
    t, v = x.shape
    ty = ty or {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[x.dtype]
    if outs is None:
        outs = dict(logprobs=torch.full((t,), 7.0, device="cuda"), ranks=torch.full((t,), 7, device="cuda", dtype=torch.int32), entropy=torch.full((t,), 7.0, device="cuda"),
                    top_ids=torch.full((t, max(top, 1)), 7, device="cuda", dtype=torch.int32), top_logprobs=torch.full((t, max(top, 1)), 7.0, device="cuda"))
    given = {n: lu.ptr(o) for n, o in outs.items() if (only is None or n in only) and (top or not n.startswith("top")) and (targets is not None or n not in ("logprobs", "ranks"))}
    p = capi.LogprobsParams(tokens=t, vocab=v, dtype=lu.CODES[ty], top=top, scale=scale, logits_stride=x.stride(0), top_stride=outs["top_ids"].stride(0), logits=lu.ptr(x), targets=lu.ptr(targets), **given)
    lu.launch("logprobs", p, stream=stream)
    return p, outs


def ref(x, targets, top, scale):
    """in 64 bits; the order by value and then by index, NaNs first"""
    z = x.double().cpu()
    s = float(torch.tensor(scale, dtype=torch.float32))
    odd = (z.isnan() | (z == INF)).any(1)
    nothing = (z == -INF).all(1)
    clean = torch.where(odd[:, None] | nothing[:, None], torch.zeros_like(z), z)
    lp = torch.log_softmax(clean * s, 1)
    h = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
    lp[odd], h[odd], lp[nothing], h[nothing] = NAN, NAN, -INF, 0.0
    order = torch.sort(torch.where(z.isnan(), torch.full_like(z, 1e300), torch.where(z == INF, torch.full_like(z, 1e299), z)) + 0.0, dim=1, descending=True, stable=True).indices
    at = torch.empty_like(order)
    at.scatter_(1, order, torch.arange(x.shape[1]).expand_as(order).contiguous())
    out = {"entropy": h, "top_ids": order[:, :top].int(), "top_logprobs": lp.gather(1, order[:, :top])}
    if targets is not None:
        tt = targets.cpu().long()
        real = (tt >= 0) & (tt < x.shape[1])
        safe = tt.clamp(0, x.shape[1] - 1)
        out["ranks"] = torch.where(real, at.gather(1, safe[:, None])[:, 0] + 1, 0).int()
        out["logprobs"] = torch.where(real, lp.gather(1, safe[:, None])[:, 0], torch.where(tt < 0, 0.0, NAN).double())
    return out


def close(got, want, bound):
    got, want = got.double().cpu(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    err = (got - want).abs()
    ok = same | (err <= bound)
    assert bool(ok.all()), (got[~ok][:5], want[~ok][:5])


def check(x, targets, top, scale=1.0, **kw):
    p, got = run(x, targets, top, scale, **kw)
    gu.sync()
    want = ref(x, targets, top, scale)
    h = want["entropy"].nan_to_num(0.0, 0.0, 0.0)
    close(got["entropy"], want["entropy"], U * (640 + 330 * h))
    if targets is not None:
        assert torch.equal(got["ranks"].cpu(), want["ranks"])
        close(got["logprobs"], want["logprobs"], U * (320 + 8 * want["logprobs"].abs().nan_to_num(0.0, 0.0, 0.0)))
    if top:
        assert torch.equal(got["top_ids"].cpu()[:, :top], want["top_ids"])
        close(got["top_logprobs"][:, :top], want["top_logprobs"], U * (320 + 8 * want["top_logprobs"].abs().nan_to_num(0.0, 0.0, 0.0)))
    return p, got


def logits(g, t, v, ty, size=3.0):
    x = size * lu.randn(g, t, v)
    x[:, :: max(1, v // 5)] += 6.0
    return x.to(lu.TYPES[ty])


def some(g, t, v):
    return torch.randint(0, v, (t,), generator=g, device="cuda").to(torch.int32)


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 5, 5), (4, 31, 31), (3, 33, 32), (2, 100, 5), (7, 1000, 20), (5, 4096, 32), (2, 8191, 1), (1, 131072, 20), (3, 50001, 5), (9, 32000, 0),
                                     (200, 9000, 3), (150, 40001, 8), (0, 10, 1)])
def test_sizes(ty, t, v, top):
    g = lu.gen(t * 3 + v)
    check(logits(g, t, v, ty), some(g, t, v), top, 0.8)


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [2, 160])
@pytest.mark.parametrize("shift,gap", [(1, 0), (0, 3), (3, 1), (5, 8), (7, 2)])
def test_strides_and_alignments(ty, t, shift, gap):
    g, v = lu.gen(4), 10007
    buf = torch.full((t * (v + gap) + shift + 16,), NAN, device="cuda", dtype=lu.TYPES[ty])
    x = buf[shift:shift + t * (v + gap)].view(t, v + gap)[:, :v]
    x.copy_(logits(g, t, v, ty))
    check(x, some(g, t, v), 7)


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v", [(3, 70001), (170, 5003)])
@pytest.mark.parametrize("kind", ["equal", "two values", "rising", "falling", "zeros of both signs", "masked", "one left", "nothing left", "lowest", "lowest and masked", "lowest but one", "huge", "infinity", "nan",
                                  "nan target", "one thread's"])
def test_values(ty, t, v, kind):
    g = lu.gen(11)
    x, targets = logits(g, t, v, ty), some(g, t, v)
    low = torch.finfo(lu.TYPES[ty]).min
    if kind == "equal":
        x[:] = 1.5
    elif kind == "two values":
        x[:] = (lu.randn(g, t, v) > 0).to(x.dtype)
    elif kind == "rising":
        x[:] = torch.linspace(-20, 20, v, device="cuda").to(x.dtype)
    elif kind == "falling":
        x[:] = torch.linspace(20, -20, v, device="cuda").to(x.dtype)
    elif kind == "zeros of both signs":
        x[:] = 0.0
        x[:, ::3] = -0.0
    elif kind == "masked":
        x[torch.rand(t, v, generator=g, device="cuda") < 0.95] = -INF
    elif kind == "one left":
        x[:] = -INF
        x[:, v // 3] = -2.0
        targets[0] = v // 3
    elif kind == "nothing left":
        x[1] = -INF
    elif kind == "lowest":
        x[:] = low
    elif kind == "lowest and masked":
        x[:] = low
        x[:, ::2] = -INF
    elif kind == "lowest but one":
        x[:] = low
        x[:, v // 2] = 4.0
    elif kind == "huge":
        x[:] = torch.where(lu.randn(g, t, v) > 0, 0.9, 0.8).to(x.dtype) * -low
    elif kind == "infinity":
        x[1, v // 2] = INF
    elif kind == "nan":
        x[1, v // 2], x[1, 3], x[2, v - 1], x[2, 0] = NAN, NAN, NAN, INF
    elif kind == "nan target":
        x[1, v // 2], x[1, 3] = NAN, NAN
        targets[1] = v // 2
    elif kind == "one thread's":
        x[:, 8 * 512 // (2 if ty == "f32" else 1):][:, :8] += 30.0
    check(x, targets, 16)


def test_targets_that_are_no_tokens():
    g = lu.gen(5)
    x, targets = logits(g, 6, 1000, "bf16"), some(g, 6, 1000)
    targets[1], targets[4] = -1, -2 ** 31
    check(x, targets, 3)
    assert gu.error_flag() == 0
    targets[2], targets[3] = 1000, 2 ** 31 - 1
    check(x, targets, 3)
    assert gu.error_flag(reset=True) == 0x305


@pytest.mark.parametrize("only", [("logprobs",), ("ranks",), ("entropy",), ("top_ids",), ("top_logprobs",)])
def test_outputs_one_at_a_time(only):
    g = lu.gen(6)
    x, targets = logits(g, 5, 3000, "f16"), some(g, 5, 3000)
    _, every = run(x, targets, 4)
    _, one = run(x, targets, 4, only=only)
    gu.sync()
    for n, o in one.items():
        assert torch.equal(o, every[n]) if n in only else bool((o == 7).all())
    check(x, None, 4)


@pytest.mark.parametrize("scale", [1e-6, 0.05, 1.0, 30.0, 1e6])
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
def test_scales(scale, ty):
    g = lu.gen(7)
    x = logits(g, 20, 6001, ty)
    p, got = run(x, some(g, 20, 6001), 5, scale)
    gu.sync()
    want = ref(x, None, 5, scale)
    # a difference of logits is rounded once, and counts times the scale
    d = (want["top_logprobs"].abs().amax(1) + x.double().cpu().abs().amax(1) * scale)[:, None]
    close(got["top_logprobs"], want["top_logprobs"], U * (320 + 8 * d))
    assert torch.equal(got["top_ids"].cpu(), want["top_ids"])


def test_rows_of_results_behind_one_another_and_from_the_last():
    g = lu.gen(8)
    x, targets = logits(g, 9, 2000, "bf16"), some(g, 9, 2000)
    _, plain = run(x, targets, 5)
    wide = torch.full((9, 11), 7, device="cuda", dtype=torch.int32), torch.full((9, 11), 7.0, device="cuda")
    outs = dict(plain, top_ids=wide[0], top_logprobs=wide[1])
    run(x, targets, 5, outs=outs)
    gu.sync()
    assert torch.equal(wide[0][:, :5], plain["top_ids"]) and torch.equal(wide[1][:, :5], plain["top_logprobs"]) and bool((wide[0][:, 5:] == 7).all()) and bool((wide[1][:, 5:] == 7).all())


def test_notifications_capture_and_the_same_bits_each_time():
    g = lu.gen(9)
    for t, v in ((3, 60000), (300, 3001)):
        x, targets = logits(g, t, v, "bf16"), some(g, t, v)
        p, outs = run(x, targets, 9)
        li = lu.info("logprobs", p)
        assert lu.records("logprobs", p) == (li.num_blocks, li.num_blocks)
        gu.sync()
        first = {n: o.clone() for n, o in outs.items()}
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lu.launch("logprobs", p, stream=side)
        for _ in range(20):
            graph.replay()
        gu.sync()
        assert all(torch.equal(o, first[n]) for n, o in outs.items())
        x.copy_(logits(g, t, v, "bf16"))
        graph.replay()
        gu.sync()
        assert torch.equal(outs["top_ids"].cpu(), ref(x, targets, 9, 1.0)["top_ids"])
