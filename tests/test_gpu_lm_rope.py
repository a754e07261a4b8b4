"""Head norms with rotation (pb_qk_rope) and the append to a paged cache (pb_kv_append) against the formulas in 64 bits.

Tolerance.  All arithmetic is in fp32 and the result is rounded once.  The sum of squares is of positive terms: a lane adds at
most 16 (wide) or 8 (single values, 4 chunks) of them, then five shuffles, so its relative error is below 23 x 2^-24, which the
root halves (12); rsqrtf is off by at most 2 ulp (4 half steps), the quotient, the sum with eps, the two products with weight and
the root's factor are one half step each (4), the rotation's two products and sum three.  Together below 32 x 2^-24 of the
products' magnitudes |a c| + |b s|, beside the output's own rounding."""
import ctypes as C

import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = pytest.mark.gpu
EPS = 1e-6


def table(positions, rot):
    at = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None]
    angle = at * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def ref_heads(x, weight, tab, positions, rot, interleaved):
    """(value, magnitude that the error counts of) in 64 bits"""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    out, mag = x.clone(), x.abs()
    if rot:
        row = tab.double()[positions.long()][:, None]
        c, s = row[..., :rot // 2], row[..., rot // 2:]
        i = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        a, b = x[..., i[0]], x[..., i[1]]
        out[..., i[0]], out[..., i[1]] = a * c - b * s, b * c + a * s
        mag[..., i[0]], mag[..., i[1]] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag


def check(got, ref, mag, ty):
    bound = lu.HALF_STEP[ty] * ref.abs() + 32 * 2.0 ** -24 * mag * (1 + lu.HALF_STEP[ty]) + lu.TINY[ty]
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def rope_params(ty, q, k, qo, ko, qw, kw, tab, pos, rot, interleaved):
    p = capi.QkRopeParams(dtype=lu.CODES[ty], tokens=q.shape[0], q_heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], rot_dim=rot,
                          interleaved=interleaved, max_position=tab.shape[0], eps=EPS, q=lu.ptr(q), k=lu.ptr(k), q_out=lu.ptr(qo), k_out=lu.ptr(ko),
                          q_weight=lu.ptr(qw), k_weight=lu.ptr(kw), cos_sin=lu.ptr(tab), positions=lu.ptr(pos))
    p.q_stride, p.q_head_stride, p.k_stride, p.k_head_stride = q.stride(0), q.stride(1), k.stride(0), k.stride(1)
    p.q_out_stride, p.q_out_head_stride, p.k_out_stride, p.k_out_head_stride = qo.stride(0), qo.stride(1), ko.stride(0), ko.stride(1)
    return p


def heads(g, t, h, d, ty, gap=0, shift=0):
    """[t][h][d] inside rows that are `gap` longer, `shift` elements into its buffer"""
    n = t * (h * d + gap)
    base = lu.randn(g, n + shift + 8).to(lu.TYPES[ty])
    return base[shift:shift + n].view(t, h * d + gap)[:, :h * d].view(t, h, d)


# head sizes on both sides of the vector widths; pairs in halves that vectors fit (8 | rot / 2) or not; whole, part, none rotated
@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, 0), (128, 64, 0), (128, 128, 1), (64, 64, 0), (96, 32, 1), (80, 80, 0), (256, 256, 0), (256, 0, 0),
                                               (72, 24, 0), (20, 10, 1), (7, 4, 0), (1, 0, 0), (129, 66, 0), (8, 8, 0), (256, 254, 1)])
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("norm", [True, False])
def test_rope_sizes(ty, d, rot, interleaved, norm):
    g = lu.gen(d * 7 + rot + norm)
    t, hq, hk = 5, 3, 2
    q, k = heads(g, t, hq, d, ty, gap=16), heads(g, t, hk, d, ty, gap=8)
    qo, ko = torch.full((t, hq, d), 9.0, device="cuda", dtype=q.dtype), torch.full((t + 1, hk, d), 9.0, device="cuda", dtype=q.dtype)
    qw, kw = (1 + 0.3 * lu.randn(g, d), 1 + 0.3 * lu.randn(g, d)) if norm else (None, None)
    tab = table(300, rot)
    pos = torch.randint(0, 300, (t,), generator=g, device="cuda", dtype=torch.int32)
    pos[0], pos[1] = 299, 0
    lu.launch("qk_rope", rope_params(ty, q, k, qo, ko, qw, kw, tab, pos, rot, interleaved))
    gu.sync()
    check(qo, *ref_heads(q, qw, tab, pos, rot, interleaved), ty)
    check(ko[:t], *ref_heads(k, kw, tab, pos, rot, interleaved), ty)
    assert bool((ko[t] == 9.0).all())
    assert gu.error_flag() == 0


# one token to so many that a group takes two and four heads; head counts that no group divides; one kind of head alone
@pytest.mark.parametrize("t,hq,hk", [(1, 1, 0), (1, 0, 1), (1, 33, 3), (700, 5, 2), (3001, 32, 8), (1201, 47, 0)])
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_rope_counts(ty, t, hq, hk):
    g, d = lu.gen(t + hq), 128
    x = heads(g, t, hq + hk, d, ty)
    q, k = x[:, :hq], x[:, hq:]
    o = torch.full((t + 2, hq + hk, d), 9.0, device="cuda", dtype=x.dtype)
    qw, kw, tab = 1 + 0.3 * lu.randn(g, d), 1 + 0.3 * lu.randn(g, d), table(4096, d)
    pos = torch.randint(0, 4096, (t,), generator=g, device="cuda", dtype=torch.int32)
    lu.launch("qk_rope", rope_params(ty, q, k, o[:t, :hq], o[:t, hq:], qw, kw, tab, pos, d, 0))
    gu.sync()
    for got, src, w in ((o[:t, :hq], q, qw), (o[:t, hq:], k, kw)):
        check(got, *ref_heads(src, w, tab, pos, d, 0), ty)
    assert bool((o[t:] == 9.0).all())


# so many tokens that a group takes four and eight heads; vectors in odd number, part rotated, kinds of head that change within a group
@pytest.mark.parametrize("t,hq,hk,d,rot", [(20000, 7, 2, 128, 128), (30011, 3, 5, 64, 32), (26003, 9, 1, 72, 48), (40000, 5, 2, 104, 32), (60000, 4, 4, 8, 0), (9001, 33, 4, 256, 256), (24000, 8, 3, 96, 96)])
@pytest.mark.parametrize("ty,interleaved,norm", [("f32", 0, True), ("f32", 1, False), ("bf16", 1, True), ("f16", 0, False), ("bf16", 0, True)])
def test_many_tokens(ty, interleaved, norm, t, hq, hk, d, rot):
    g = lu.gen(t + d)
    x = heads(g, t, hq + 2 * hk, d, ty)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    qw, kw = (1 + 0.3 * lu.randn(g, d), 1 + 0.3 * lu.randn(g, d)) if norm else (None, None)
    tab = table(777, rot)
    pos = torch.randint(0, 777, (t,), generator=g, device="cuda", dtype=torch.int32)
    qo, ko = torch.full((t, hq, d), 9.0, device="cuda", dtype=x.dtype), torch.full((t + 1, hk, d), 9.0, device="cuda", dtype=x.dtype)
    lu.launch("qk_rope", rope_params(ty, q, k, qo, ko, qw, kw, tab, pos, rot, interleaved))
    gu.sync()
    check(qo, *ref_heads(q, qw, tab, pos, rot, interleaved), ty)
    check(ko[:t], *ref_heads(k, kw, tab, pos, rot, interleaved), ty)
    assert bool((ko[t] == 9.0).all())
    page, pages = 32, t // 32 + 3
    kc, vc = (cache(pages, page, hk, d, ty, True) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
    slots[t // 3:t // 3 + 100] = -2
    qo.fill_(9.0)
    lu.launch("kv_append", append_params(ty, k, v, kc, vc, slots, page, tab, pos, rot, interleaved, kw, True, q=q, qo=qo, qw=qw))
    gu.sync()
    real = slots >= 0
    ref, mag = ref_heads(k, kw, tab, pos, rot, interleaved)
    check(rows(kc, slots[real], page, True), ref[real], mag[real], ty)
    assert torch.equal(rows(vc, slots[real], page, True), v[real])
    for c in (kc, vc):
        assert int((c != 9.0).any(-1).sum()) == int(real.sum()) * hk
    check(qo, *ref_heads(q, qw, tab, pos, rot, interleaved), ty)
    pos[5], slots[7] = 777, pages * page                         # and what is out of range is left out
    qo.fill_(9.0)
    lu.launch("kv_append", append_params(ty, k, v, kc, vc, slots, page, tab, pos, rot, interleaved, kw, True, q=q, qo=qo, qw=qw))
    gu.sync()
    assert gu.error_flag() != 0
    left = [5, 7] if rot else [7]
    assert bool((qo[left] == 9.0).all()) and bool((qo[[4, 6, 8]] != 9.0).any(-1).all())


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_rope_in_place_at_any_element(shift, interleaved):
    g, t, d = lu.gen(shift), 37, 64
    q, k = heads(g, t, 4, d, "bf16", shift=shift), heads(g, t, 2, d, "bf16", gap=shift, shift=shift)
    qw, kw, tab = 1 + 0.3 * lu.randn(g, d), None, table(64, d)
    pos = torch.randint(0, 64, (t,), generator=g, device="cuda", dtype=torch.int32)
    rq, rk = ref_heads(q, qw, tab, pos, d, interleaved), ref_heads(k, kw, tab, pos, d, interleaved)
    lu.launch("qk_rope", rope_params("bf16", q, k, q, k, qw, kw, tab, pos, d, interleaved))
    gu.sync()
    check(q, *rq, "bf16")
    check(k, *rk, "bf16")


@pytest.mark.parametrize("interleaved", [0, 1])
def test_rope_of_many_tokens_in_place(interleaved):
    """Queries and keys inside a fused projection's rows, turned where they lie; the values between them stay."""
    g, t, d = lu.gen(11), 21000, 64
    x = heads(g, t, 14, d, "bf16")
    q, k, v = x[:, :9], x[:, 9:11], x[:, 11:]
    qw, kw, tab, v0 = 1 + 0.3 * lu.randn(g, d), 1 + 0.3 * lu.randn(g, d), table(64, d), v.clone()
    pos = torch.randint(0, 64, (t,), generator=g, device="cuda", dtype=torch.int32)
    rq, rk = ref_heads(q, qw, tab, pos, d, interleaved), ref_heads(k, kw, tab, pos, d, interleaved)
    lu.launch("qk_rope", rope_params("bf16", q, k, q, k, qw, kw, tab, pos, d, interleaved))
    gu.sync()
    check(q, *rq, "bf16")
    check(k, *rk, "bf16")
    assert torch.equal(v, v0)


def test_rope_values_at_the_ends_of_the_range():
    """Zeros stay zeros, the type's largest values are normed without overflow of the mean, a NaN stays in its head."""
    d, t = 128, 4
    q = torch.zeros(t, 2, d, device="cuda", dtype=torch.bfloat16)
    q[1], q[2, 0, 5], q[3, 1, 7] = 1e18, float("nan"), float("inf")
    k = torch.ones(t, 1, d, device="cuda", dtype=torch.bfloat16)
    qo, ko, w, tab = torch.empty_like(q), torch.empty_like(k), torch.ones(d, device="cuda"), table(8, d)
    pos = torch.zeros(t, device="cuda", dtype=torch.int32)
    lu.launch("qk_rope", rope_params("bf16", q, k, qo, ko, w, w, tab, pos, d, 0))
    gu.sync()
    assert bool((qo[0] == 0).all()) and bool((qo[1] == 1).all())
    assert bool(qo[2, 0].isnan().all()) and bool((qo[2, 1] == 0).all())
    assert bool(qo[3, 1, 7].isnan()) and bool((qo[3, 0] == 0).all())
    assert bool((ko == 1).all())


def append_params(ty, k, v, kc, vc, slots, page, tab=None, pos=None, rot=0, interleaved=0, kw=None, heads_first=False, q=None, qo=None, qw=None):
    token, head = (kc.stride(2), kc.stride(1)) if heads_first else (kc.stride(1), kc.stride(2))
    p = capi.KvAppendParams(dtype=lu.CODES[ty], tokens=k.shape[0], q_heads=0, kv_heads=k.shape[1], head_dim=k.shape[2], rot_dim=rot, interleaved=interleaved,
                            max_position=0 if tab is None else tab.shape[0], eps=EPS, page_size=page, n_pages=kc.shape[0], k_stride=k.stride(0),
                            k_head_stride=k.stride(1), v_stride=v.stride(0), v_head_stride=v.stride(1), page_stride=kc.stride(0), token_stride=token,
                            head_stride=head, k=lu.ptr(k), v=lu.ptr(v), k_weight=lu.ptr(kw), cos_sin=lu.ptr(tab), positions=lu.ptr(pos),
                            slots=lu.ptr(slots), k_cache=lu.ptr(kc), v_cache=lu.ptr(vc))
    if q is not None:
        p.q_heads, p.q_stride, p.q_head_stride, p.q_out_stride, p.q_out_head_stride = q.shape[1], q.stride(0), q.stride(1), qo.stride(0), qo.stride(1)
        p.q, p.q_out, p.q_weight = lu.ptr(q), lu.ptr(qo), lu.ptr(qw)
    return p


def cache(pages, page, h, d, ty, heads_first):
    return torch.full((pages, h, page, d) if heads_first else (pages, page, h, d), 9.0, device="cuda", dtype=lu.TYPES[ty])


def rows(c, slots, page, heads_first):
    s = slots.long()
    return c[s // page, :, s % page] if heads_first else c[s // page, s % page]


@pytest.mark.parametrize("t,d,rot,page,interleaved,heads_first", [(1, 128, 128, 16, 0, False), (5, 64, 64, 1, 0, False), (100, 96, 48, 17, 1, True),
                                                                  (64, 128, 0, 64, 0, True), (33, 20, 20, 8, 0, False), (2500, 128, 128, 128, 0, False)])
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("with_q", [False, True])
def test_append(ty, t, d, rot, page, interleaved, heads_first, with_q):
    g, h, hq = lu.gen(t + d), 3, 6
    x = heads(g, t, hq + 2 * h, d, ty)
    q, k, v = x[:, :hq], x[:, hq:hq + h], x[:, hq + h:]
    pages = -(-t // page) + 3
    kc, vc = (cache(pages, page, h, d, ty, heads_first) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
    padded = slots.clone()
    padded[t // 2:t // 2 + t // 4] = -1
    tab, pos = (table(500, rot), torch.randint(0, 500, (t,), generator=g, device="cuda", dtype=torch.int32)) if rot else (None, None)
    kw, qw, qo = 1 + 0.3 * lu.randn(g, d), 1 + 0.3 * lu.randn(g, d), torch.empty(t, hq, d, device="cuda", dtype=x.dtype)
    more = dict(q=q, qo=qo, qw=qw) if with_q else {}
    lu.launch("kv_append", append_params(ty, k, v, kc, vc, padded, page, tab, pos, rot, interleaved, kw, heads_first, **more))
    gu.sync()
    real = padded >= 0
    ref, mag = ref_heads(k, kw, tab, pos, rot, interleaved)
    check(rows(kc, slots[real], page, heads_first), ref[real], mag[real], ty)
    assert torch.equal(rows(vc, slots[real], page, heads_first), v[real])
    for c in (kc, vc):                                           # nothing else was touched
        assert int((c != 9.0).any(-1).sum()) == int(real.sum()) * h
    if with_q:
        check(qo, *ref_heads(q, qw, tab, pos, rot, interleaved), ty)
    assert gu.error_flag() == 0


def test_append_copies_values_bit_for_bit():
    """Without norm and rotation keys, too, keep their bits: NaNs with payloads, signed zeros, infinities."""
    bits = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16)
    x = bits.view(64, 8, 128)
    kc, vc = torch.zeros(4, 16, 4, 128, device="cuda", dtype=torch.int16), torch.zeros(4, 16, 4, 128, device="cuda", dtype=torch.int16)
    lu.launch("kv_append", append_params("bf16", x[:, :4], x[:, 4:], kc, vc, torch.arange(64, device="cuda"), 16))
    gu.sync()
    assert torch.equal(kc.view(64, 4, 128), x[:, :4]) and torch.equal(vc.view(64, 4, 128), x[:, 4:])


def test_bad_slots_and_positions_are_left_out_and_flagged():
    g, t, d = lu.gen(3), 6, 64
    x, tab = heads(g, t, 3, d, "bf16"), table(10, d)
    q, k, v = x[:, :1], x[:, 1:2], x[:, 2:]
    for slots, pos, left, flag in (([0, 1, 32, 3, 4, 5], [0, 1, 2, 3, 4, 5], [2], True), ([0, 1, 2, 3, 4, 2 ** 40], [0] * 6, [5], True),
                                   ([0, 1, 2, 3, 4, 5], [0, 10, 2, -1, 4, 5], [1, 3], True), ([0, -7, 2, 3, 4, 5], [0, 99, 0, 0, 0, 0], [1], False)):
        kc, vc, qo = cache(4, 8, 1, d, "bf16", False), cache(4, 8, 1, d, "bf16", False), torch.full((t, 1, d), 9.0, device="cuda", dtype=x.dtype)
        sl, ps = torch.tensor(slots, device="cuda"), torch.tensor(pos, device="cuda", dtype=torch.int32)
        lu.launch("kv_append", append_params("bf16", k, v, kc, vc, sl, 8, tab, ps, d, q=q, qo=qo))
        gu.sync()
        assert (gu.error_flag() != 0) == flag and gu.error_flag() == 0
        keep = [i for i in range(t) if i not in left]
        assert torch.equal(vc.view(-1, 1, d)[sl[keep]], v[keep]) and int((vc != 9.0).any(-1).sum()) == len(keep)
        assert int((kc != 9.0).any(-1).sum()) == len(keep)
        assert bool((qo[left] == 9.0).all()) and bool((qo[keep] != 9.0).any(-1).all())
    qo, ko = torch.full((t, 1, d), 9.0, device="cuda", dtype=x.dtype), torch.full((t, 1, d), 9.0, device="cuda", dtype=x.dtype)
    pos = torch.tensor([0, 1, 2 ** 31 - 1, 3, 4, 5], device="cuda", dtype=torch.int32)
    lu.launch("qk_rope", rope_params("bf16", q, k, qo, ko, None, None, tab, pos, d, 0))
    gu.sync()
    assert gu.error_flag() != 0
    assert bool((qo[2] == 9.0).all()) and bool((ko[2] == 9.0).all()) and bool((ko[3] != 9.0).any())


def test_append_behind_four_billion_elements():
    d, page, pages = 128, 64, 66000                              # 66000 x 64 x 8 x 128 = 4.3e9 elements a cache
    kc, vc = (torch.empty(pages, page, 8, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kc[-1], vc[-1] = 9.0, 9.0
    x = heads(lu.gen(4), 2, 16, d, "bf16")
    slots = torch.tensor([pages * page - 1, 0], device="cuda")
    lu.launch("kv_append", append_params("bf16", x[:, :8], x[:, 8:], kc, vc, slots, page))
    gu.sync()
    assert torch.equal(kc[-1, -1], x[0, :8]) and torch.equal(vc[-1, -1], x[0, 8:]) and torch.equal(kc[0, 0], x[1, :8])
    assert bool((kc[-1, :-1] == 9.0).all())


def test_streams_graphs_and_empty_calls():
    """A captured launch reads what its buffers hold at the replay, behind a copy in the same graph; no token, no change."""
    g, t, d = lu.gen(5), 9, 128
    x, tab, src = heads(g, t, 3, d, "bf16"), table(100, d), torch.zeros(t, device="cuda", dtype=torch.int32)
    q, k, qo, ko, pos = x[:, :2], x[:, 2:], torch.empty(t, 2, d, device="cuda", dtype=x.dtype), torch.empty(t, 1, d, device="cuda", dtype=x.dtype), src.clone()
    p = rope_params("bf16", q, k, qo, ko, None, None, tab, pos, d, 0)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        pos.copy_(src)
        lu.launch("qk_rope", p)
        ko.mul_(2)
    for at in (3, 77):
        src.fill_(at)
        graph.replay()
        gu.sync()
        check(qo, *ref_heads(q, None, tab, src, d, 0), "bf16")
        ref, mag = ref_heads(k, None, tab, src, d, 0)
        check(ko / 2, ref, mag, "bf16")
    with torch.cuda.stream(st):
        st.wait_stream(torch.cuda.default_stream())
        src.fill_(12)
        pos.copy_(src)
        lu.launch("qk_rope", p)
    gu.sync()
    check(qo, *ref_heads(q, None, tab, src, d, 0), "bf16")
    before = qo.clone()
    p.tokens = 0
    lu.launch("qk_rope", p)
    gu.sync()
    assert torch.equal(qo, before)
    assert lu.records("qk_rope", p) == (1, 1)


@pytest.mark.parametrize("t", [1, 40, 3000])
def test_notifications_count_the_declared_blocks(t):
    g, d = lu.gen(6), 64
    x, tab = heads(g, t, 6, d, "bf16"), table(16, d)
    pos = torch.zeros(t, device="cuda", dtype=torch.int32)
    o = torch.empty_like(x)
    p = rope_params("bf16", x[:, :4], x[:, 4:], o[:, :4], o[:, 4:], None, None, tab, pos, d, 0)
    n = lu.info("qk_rope", p).num_blocks
    assert lu.records("qk_rope", p) == (n, n)
    kc = cache(t, 1, 2, d, "bf16", False)
    a = append_params("bf16", x[:, :2], x[:, 2:4], kc, kc.clone(), torch.arange(t, device="cuda"), 1)
    n = lu.info("kv_append", a).num_blocks
    assert lu.records("kv_append", a) == (n, n)
