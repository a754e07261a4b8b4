"""Dense layers in 8-bit integers (pb_int8_quantize, pb_int8_dense).

The quantiser is defined in fp32 operations that are each correctly rounded, so torch's give the same integers and scales, bit
for bit.  The product's sum is exact; then the sum's conversion to fp32, the scales' product, the fused multiply-add and the
output's rounding are half a step each: 2^-24 x 3 of the product's magnitude, 2^-24 of the result, and the type's half step."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = pytest.mark.gpu


def plain_quantize(x):
    """each operation rounded to fp32 (torch takes a quotient by a plain number as a product: hence the tensor)"""
    most = x.float().abs().amax(1)
    return (x.float() * (most.reciprocal() * 127.0)[:, None]).round(), most / torch.full_like(most, 127.0)


def quantize(x, stride=None):
    t, k = x.shape
    q = torch.full((t + 1, stride or -(-k // 16) * 16), 77, device="cuda", dtype=torch.int8)
    s = torch.full((t + 1,), 9.0, device="cuda")
    ty = {v: n for n, v in lu.TYPES.items()}[x.dtype]
    p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=lu.CODES[ty], x_stride=x.stride(0), q_stride=q.stride(0), x=lu.ptr(x), q=lu.ptr(q), scale=lu.ptr(s))
    lu.launch("int8_quantize", p)
    gu.sync()
    assert float(s[t]) == 9.0 and bool((q[t] == 77).all()) and bool((q[:, k:] == 77).all())
    return q[:t, :k], s[:t], p


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,k,shift,gap", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 8, 0, 8), (2, 255, 1, 3), (4, 4096, 0, 0), (33, 1000, 0, 24), (300, 2056, 8, 0), (2, 40000, 0, 0), (1500, 72, 0, 0)])
def test_quantize(ty, t, k, shift, gap):
    g = lu.gen(k)
    base = (lu.randn(g, t * (k + gap) + shift) * 3).to(lu.TYPES[ty])
    x = base[shift:].view(t, k + gap)[:, :k]
    q, s, p = quantize(x)
    rq, rs = plain_quantize(x)
    assert torch.equal(q.float(), rq) and torch.equal(s, rs)


def test_quantize_odd_rows():
    x = torch.zeros(7, 300, device="cuda")
    x[1, 4], x[2, 299], x[3, 0] = float("nan"), float("inf"), -float("inf")
    x[4, 3], x[4, 4] = 2.0 ** -119, -2.0 ** -120
    x[5, 7] = 2.0 ** -120
    x[6] = 3.0e38
    q, s, _ = quantize(x)
    assert bool((q[:4] == 0).all()) and float(s[0]) == 0.0 and bool(s[1:4].isnan().all())
    assert q[4, 3] == 127 and q[4, 4] == -64 and float(s[4]) > 0               # -63.5: the half goes to even
    assert bool((q[5] == 0).all()) and float(s[5]) == 0.0
    assert bool((q[6] == 127).all())


def operands(g, t, k, n, gap=0):
    row = -(-k // 16) * 16 + gap
    x, w = (torch.full((r, row), 99, device="cuda", dtype=torch.int8) for r in (t, n))   # what lies behind a row's end is not read
    x[:, :k], w[:, :k] = (torch.randint(-128, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (t, n))
    return x, w, torch.rand(t, generator=g, device="cuda") + 0.1, (torch.rand(n, generator=g, device="cuda") + 0.1) / k


def dense_params(x, xs, w, ws, k, bias, y, ty, act=0):
    return capi.Int8DenseParams(tokens=x.shape[0], in_channels=k, out_channels=w.shape[0], y_dtype=lu.CODES[ty], act=act, x_stride=x.stride(0), w_stride=w.stride(0),
                                y_stride=y.stride(0), x=lu.ptr(x), x_scale=lu.ptr(xs), w=lu.ptr(w), w_scale=lu.ptr(ws), bias=lu.ptr(bias), y=lu.ptr(y))


def check_dense(y, x, xs, w, ws, k, bias, ty, act):
    main = (x[:, :k].double() @ w[:, :k].double().t()) * xs.double()[:, None] * ws.double()
    ref = main if bias is None else main + bias.double()
    ref = ref.clamp_min(0) if act else ref
    ref = ref.clamp_max(6) if act == 2 else ref
    bound = 3 * 2.0 ** -24 * main.abs() + (2.0 ** -24 + lu.HALF_STEP[ty]) * (ref.abs() + 3 * 2.0 ** -24 * main.abs()) + lu.TINY[ty]
    off = (y.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# rows and columns around the tiles' edges, reductions around the k-blocks' (16, 32, 128 bytes), few rows against many columns and the reverse
@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 4096, 4096), (2, 100, 129), (7, 512, 1000), (8, 128, 64), (9, 4097, 130), (16, 2000, 384), (17, 333, 2049), (24, 8192, 512), (31, 129, 95),
                                   (33, 1024, 777), (64, 2048, 2048), (65, 640, 300), (96, 16, 5000), (127, 127, 127), (128, 128, 128), (129, 257, 255), (200, 1000, 1000), (255, 31, 513),
                                   (256, 4096, 256), (300, 2049, 1025), (777, 2000, 5001), (1024, 512, 4096), (2049, 96, 65), (1, 131071, 3), (4096, 1024, 2048)])
@pytest.mark.parametrize("ty,bias,act,gap", [("bf16", False, 0, 0), ("f32", True, 1, 16), ("f16", True, 2, 0)])
def test_dense(ty, bias, act, gap, t, k, n):
    g = lu.gen(t * 3 + k * 5 + n)
    x, w, xs, ws = operands(g, t, k, n, gap)
    b = lu.randn(g, n) if bias else None
    y = torch.full((t + 1, n + gap), 9.0, device="cuda", dtype=lu.TYPES[ty])
    lu.launch("int8_dense", dense_params(x, xs, w, ws, k, b, y[:t], ty, act))
    gu.sync()
    check_dense(y[:t, :n], x, xs, w, ws, k, b, ty, act)
    assert bool((y[t] == 9.0).all()) and bool((y[:, n:] == 9.0).all())
    assert gu.error_flag() == 0


# more tiles than pairs of SMs, and a narrower last one: pairs that have a wide tile less than others take one or more of those, then all do
@pytest.mark.parametrize("t,k,n", [(257, 64, 20000), (519, 144, 40000), (777, 200, 5001), (777, 32, 9472), (1030, 272, 19001), (3000, 128, 2600), (333, 16, 30000), (290, 48, 37888), (1000, 96, 12345)])
def test_dense_of_many_tiles(t, k, n):
    g = lu.gen(t + n)
    x, w, xs, ws = operands(g, t, k, n)
    y = torch.full((t + 1, n), 9.0, device="cuda")
    for _ in range(2):
        lu.launch("int8_dense", dense_params(x, xs, w, ws, k, None, y[:t], "f32"))
    gu.sync()
    check_dense(y[:t], x, xs, w, ws, k, None, "f32", 0)
    assert bool((y[t] == 9.0).all()) and gu.error_flag() == 0


@pytest.mark.parametrize("t,k,n", [(1, 131071, 128), (40, 131071, 128), (200, 131071, 256)])
@pytest.mark.parametrize("a,b", [(-128, -128), (-128, 127), (127, 127)])
def test_dense_sums_reach_32_bits(t, k, n, a, b):
    x, w = torch.full((t, 131072), a, device="cuda", dtype=torch.int8), torch.full((n, 131072), b, device="cuda", dtype=torch.int8)
    xs, ws = torch.full((t,), 0.5, device="cuda"), torch.full((n,), 2.0, device="cuda")
    y = torch.empty(t, n, device="cuda")
    lu.launch("int8_dense", dense_params(x, xs, w, ws, k, None, y, "f32"))
    gu.sync()
    assert bool((y == torch.tensor(float(a * b * k), dtype=torch.float32)).all())


@pytest.mark.parametrize("t", [1, 20, 300])
def test_dense_rows_into_a_wider_tensor_and_nan_scales(t):
    """y's rows start anywhere; a token whose scale is NaN has NaN results, with relu too, and no other has."""
    g, k, n = lu.gen(t), 200, 130
    x, w, xs, ws = operands(g, t, k, n)
    xs[t // 2] = float("nan")
    big = torch.full((t * 150 + 8,), 9.0, device="cuda", dtype=torch.bfloat16)
    y = big[3:3 + t * 150].view(t, 150)[:, :n]
    p = dense_params(x, xs, w, ws, k, None, y, "bf16", act=1)
    lu.launch("int8_dense", p)
    gu.sync()
    rest = [i for i in range(t) if i != t // 2]
    assert bool(y[t // 2].isnan().all())
    check_dense(y[rest], x[rest], xs[rest], w, ws, k, None, "bf16", 1)
    assert bool((big[3:3 + t * 150].view(t, 150)[:, n:] == 9.0).all())


@pytest.mark.parametrize("t", [1, 12, 260])
def test_quantize_and_dense_together_captured(t):
    """The two launches as a program makes them, captured into a graph that is replayed on new activations."""
    g, k, n = lu.gen(9 + t), 520, 300
    _, w, _, ws = operands(g, t, k, n)
    x, q, s = torch.zeros(t, k, device="cuda", dtype=torch.bfloat16), torch.empty(t, 528, device="cuda", dtype=torch.int8), torch.empty(t, device="cuda")
    y, b = torch.empty(t, n, device="cuda"), lu.randn(g, n)
    p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=capi.BF16, x_stride=k, q_stride=528, x=lu.ptr(x), q=lu.ptr(q), scale=lu.ptr(s))
    d = dense_params(q, s, w, ws, k, b, y, "f32")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lu.launch("int8_quantize", p)
        lu.launch("int8_dense", d)
    first = None
    for i in range(3):
        x.copy_(lu.randn(g, t, k) if i < 2 else first)
        if i == 0:
            first = x.clone()
        graph.replay()
        gu.sync()
        rq, rs = plain_quantize(x)
        check_dense(y, rq, rs, w, ws, k, b, "f32", 0)
        if i == 0:
            kept = y.clone()
    assert torch.equal(y, kept)                                  # the same bits for the same inputs


@pytest.mark.parametrize("t", [0, 1, 30, 700])
def test_notifications_count_the_declared_blocks(t):
    g, k, n = lu.gen(t), 300, 600
    x, w, xs, ws = operands(g, max(t, 1), k, n)
    y = torch.full((max(t, 1), n), 9.0, device="cuda")
    p = dense_params(x, xs, w, ws, k, None, y, "f32")
    p.tokens = t
    blocks = lu.info("int8_dense", p).num_blocks
    assert lu.records("int8_dense", p) == (blocks, blocks)
    assert t > 0 or bool((y == 9.0).all())
    f = lu.randn(g, max(t, 1), k)
    p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=capi.F32, x_stride=k, q_stride=k, x=lu.ptr(f), q=lu.ptr(x), scale=lu.ptr(xs))
    blocks = lu.info("int8_quantize", p).num_blocks
    assert lu.records("int8_quantize", p) == (blocks, blocks)
