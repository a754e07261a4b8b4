"""Norms around the residual (pb_residual_norm) against the formulas in 64 bits.

Tolerance, in u = 2^-24, a rounding of fp32.  A sum of squares is of positive terms: a thread adds at most 64 of them, then five shuffles and
up to 32 warps, 101 u at most, which the root halves (51); the mean, the sum with eps (halved, too: 1), rsqrtf (2 ulp: 4) and the two products with the
weight make it 58 u of a.  The gate is one more, the product with scale and the sum with the residual one: h is off by 60 u of mag = |residual| +
|scale gate a|, beside its own rounding.  y's norm has the same 58 u, and what h's errors do to its sum of squares, which by Cauchy's inequality is at most
60 u of the root mean square of mag over that of h."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = pytest.mark.gpu
EPS, U = 1e-6, 2.0 ** -24


def params(ty, hty, x, post, gate, residual, h, weight, y, scale):
    p = capi.ResidualNormParams(tokens=x.shape[0], channels=x.shape[1], dtype=lu.CODES[ty], h_dtype=lu.CODES[hty], scale=scale, eps=EPS, x=lu.ptr(x), post_weight=lu.ptr(post), gate=lu.ptr(gate),
                                residual=lu.ptr(residual), h=lu.ptr(h), weight=lu.ptr(weight), y=lu.ptr(y))
    for name, t in (("x", x), ("residual", residual), ("h", h), ("y", y)):
        if t is not None:
            setattr(p, name + "_stride", t.stride(0))
    if gate is not None and gate.shape[0] == x.shape[0]:
        p.gate_stride = gate.stride(0)
    return p


def ref(x, post, gate, residual, weight, scale):
    """h, y and what their errors count of, in 64 bits"""
    a = x.double()
    if post is not None:
        a = a / (a.pow(2).mean(1, keepdim=True) + EPS).sqrt() * post.double()
    a = a * scale * (1.0 if gate is None else gate.double())
    r = torch.zeros_like(a) if residual is None else residual.double()
    h, mag = r + a, r.abs() + a.abs()
    f = 1.0 / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * (1.0 if weight is None else weight.double())
    ratio = mag.pow(2).mean(1, keepdim=True).sqrt() / h.pow(2).mean(1, keepdim=True).sqrt().clamp_min(1e-300)
    return h, h * f, 60 * U * mag, (60 * U * mag + (60 * ratio + 60) * U * h.abs()) * f.abs()


def near(got, want, off, ty):
    bound = lu.HALF_STEP[ty] * (want.abs() + off) + off + lu.TINY[ty]
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).nan_to_num(9e9).max())


def rows(g, t, c, ty, gap=0, shift=0):
    """[t][c] inside rows that are `gap` longer, `shift` elements into its buffer"""
    buf = lu.randn(g, t * (c + gap) + shift).to(lu.TYPES[ty])
    return buf[shift:].view(t, c + gap)[:, :c]


TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")]


@pytest.mark.parametrize("ty,hty", TYPES)
@pytest.mark.parametrize("t,c", [(1, 1), (3, 7), (5, 64), (2, 1000), (37, 1024), (1, 4096), (70, 4104), (9, 5001), (2, 16384), (3, 32768), (2, 32767), (1030, 256), (0, 64)])
def test_all_parts(ty, hty, t, c):
    g = lu.gen(t * 7 + c)
    x, r, gate = rows(g, t, c, ty), rows(g, t, c, hty), rows(g, t, c, ty)
    post, w = lu.randn(g, c), lu.randn(g, c)
    h, y = torch.full_like(r, 7.0), torch.full_like(x, 7.0)
    lu.launch("residual_norm", params(ty, hty, x, post, gate, r, h, w, y, 0.7))
    gu.sync()
    wh, wy, eh, ey = ref(x, post, gate, r, w, float(torch.tensor(0.7)))
    near(h, wh, eh, hty)
    near(y, wy, ey, ty)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("outs", ["hy", "h", "y"])
def test_parts_left_out(post, gate, residual, outs):
    g, t, c, ty = lu.gen(3), 19, 520, "bf16"
    x = rows(g, t, c, ty)
    r = rows(g, t, c, ty) if residual else None
    gt = {"none": None, "channel": rows(g, 1, c, ty), "token": rows(g, t, c, ty)}[gate]
    pw, w = (lu.randn(g, c), lu.randn(g, c)) if post else (None, None)
    h, y = torch.empty_like(x), torch.empty_like(x)
    lu.launch("residual_norm", params(ty, ty, x, pw, gt, r, h if "h" in outs else None, w, y if "y" in outs else None, -1.5))
    gu.sync()
    wh, wy, eh, ey = ref(x, pw, gt, r, w, -1.5)
    if "h" in outs:
        near(h, wh, eh, ty)
    if "y" in outs:
        near(y, wy, ey, ty)


@pytest.mark.parametrize("ty,hty", TYPES)
@pytest.mark.parametrize("gap,shift,c", [(3, 0, 512), (8, 0, 512), (0, 1, 512), (8, 8, 512), (1, 3, 77), (0, 0, 77)])
def test_strides_and_alignments(ty, hty, gap, shift, c):
    g, t = lu.gen(5), 11
    x, r = rows(g, t, c, ty, gap, shift), rows(g, t, c, hty, gap, shift)
    w = lu.randn(g, c + 1)[1:]
    h, y = rows(g, t, c, hty, gap, shift), rows(g, t, c, ty, gap + 2, shift)
    lu.launch("residual_norm", params(ty, hty, x, w, None, r, h, w, y, 1.0))
    gu.sync()
    wh, wy, eh, ey = ref(x, w, None, r, w, 1.0)
    near(h, wh, eh, hty)
    near(y, wy, ey, ty)
    base = y._base if y._base is not None else y
    assert base.isfinite().all()


@pytest.mark.parametrize("t", [3, 5000])
@pytest.mark.parametrize("c", [768, 4096])
def test_in_place_and_reversed_rows(t, c):
    g, ty = lu.gen(6), "bf16"
    x, r, w = rows(g, t, c, ty), rows(g, t, c, ty), lu.randn(g, c)
    wh, wy, eh, ey = ref(x, None, None, r, w, 1.0)
    x2, r2 = x.clone(), r.clone()
    lu.launch("residual_norm", params(ty, ty, x2, None, None, r2, r2, w, x2, 1.0))
    gu.sync()
    near(r2, wh, eh, ty)
    near(x2, wy, ey, ty)
    # results from the last row to the first
    h, y = torch.empty_like(x), torch.empty_like(x)
    p = params(ty, ty, x, None, None, r, h, w, y, 1.0)
    p.h_stride, p.h = -c, h.data_ptr() + (t - 1) * c * 2
    p.y_stride, p.y = -c, y.data_ptr() + (t - 1) * c * 2
    lu.launch("residual_norm", p)
    gu.sync()
    assert torch.equal(h.flip(0), r2) and torch.equal(y.flip(0), x2)


@pytest.mark.parametrize("t", [4, 3000])
def test_values_that_are_not_finite_stay_in_their_row(t):
    g, c, ty = lu.gen(8), 1024, "bf16"
    x, r, w = rows(g, t, c, ty), rows(g, t, c, ty), lu.randn(g, c)
    wh, wy, eh, ey = ref(x, w, None, r, w, 1.0)
    x[1, 5], r[2, 9] = float("nan"), float("inf")
    h, y = torch.empty_like(x), torch.empty_like(x)
    lu.launch("residual_norm", params(ty, ty, x, w, None, r, h, w, y, 1.0))
    gu.sync()
    good = [i for i in range(t) if i not in (1, 2)]
    near(h[good], wh[good], eh[good], ty)
    near(y[good], wy[good], ey[good], ty)
    assert h[1].isnan().all() and y[1].isnan().all() and h[2, 9] == float("inf") and bool((y[2, :9] == 0).all()) and y[2, 9].isnan()


@pytest.mark.parametrize("c,inside,outside", [(1024, 5.7e17, 5.8e17), (32768, 1.0e17, 1.1e17)])
def test_sums_of_squares_up_to_the_range_of_fp32(c, inside, outside):
    x = torch.ones(3, c, device="cuda")
    x[1], x[2] = inside, outside
    assert c * float(x[1, 0]) ** 2 < 3.4028234e38 < c * float(x[2, 0]) ** 2
    y = torch.empty_like(x)
    lu.launch("residual_norm", params("f32", "f32", x, None, None, None, None, None, y, 1.0))
    gu.sync()
    assert bool(((y[:2] - 1.0).abs() <= 64 * U + EPS).all()) and bool((y[2] == 0).all())


def test_notifications_streams_and_capture():
    g, t, c, ty = lu.gen(9), 700, 2048, "f16"
    x, r, w = rows(g, t, c, ty), rows(g, t, c, ty), lu.randn(g, c)
    h, y = torch.empty_like(x), torch.empty_like(x)
    p = params(ty, ty, x, w, None, r, h, w, y, 1.0)
    li = lu.info("residual_norm", p)
    assert lu.records("residual_norm", p) == (li.num_blocks, li.num_blocks)
    first = h.clone(), y.clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lu.launch("residual_norm", p, stream=side)
    x2 = lu.randn(g, t, c).half()
    for _ in range(3):
        x.copy_(x2)
        graph.replay()
        gu.sync()
        wh, wy, eh, ey = ref(x2, w, None, r, w, 1.0)
        near(h, wh, eh, ty)
        near(y, wy, ey, ty)
    assert not torch.equal(first[0], h)
