"""Attention behind a shared prefix (pb_prefix_attn) against the formula in 64 bits.

Tolerance, relative to sum p |v| / sum p (`mag`): the softmax's values are rounded to the cache's type once (its half step); a
score's product sums head_dim terms in fp32, at most (head_dim + 8) x 2^-24 x scale x sum |q k| off, which changes its
exponential by as much, as do the score's scaling and the subtraction of the maximum (2^-23 x the largest |score|, in powers of
two), and ex2 is off by 2^-22; the sums of the p and of the p v add at most as many terms as there are tokens, each rounding
2^-24, and merging parts adds some 40 more.  Beside it the output's own rounding."""
import ctypes as C
import math

import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("prefix_kernel")]


@pytest.fixture(params=["rule", "0", "1"])
def prefix_kernel(request, monkeypatch):
    """Which kernel takes the prefix: by rule, the one of the sequences' own tokens, or that of the whole batch."""
    if request.param == "rule":
        monkeypatch.delenv("PB_ATTN_PREFIX", raising=False)
    else:
        monkeypatch.setenv("PB_ATTN_PREFIX", request.param)
    return request.param


class Problem:
    """`lens`: each sequence's own tokens.  Pages are dealt at random; what no token lies in holds NaNs and infinities."""

    def __init__(self, lens, hkv, group, d, prefix, page, ty="bf16", heads_first=False, most=None, q_gap=0, cache_gap=0, seed=0, q_size=1.5, extra_pages=2):
        g = lu.gen(seed + d + prefix + page)
        self.lens, self.hkv, self.group, self.d, self.prefix, self.page, self.ty, self.heads_first = list(lens), hkv, group, d, prefix, page, ty, heads_first
        b, t = len(self.lens), lu.TYPES[ty]
        self.most = max(self.lens + [0]) if most is None else most
        self.ahead, self.each = -(-prefix // page), -(-self.most // page)
        pages = self.ahead + b * self.each + extra_pages
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.prefix_pages = order[:self.ahead].contiguous()
        self.table = torch.full((b, self.each + 3), -5, dtype=torch.int32, device="cuda")          # entries behind max_blocks are not read
        self.table[:, :self.each] = order[self.ahead:self.ahead + b * self.each].view(b, self.each)
        inner = (hkv, page) if heads_first else (page, hkv)
        self.kc, self.vc = ((lu.randn(g, pages, *inner, d + cache_gap)).to(t)[..., :d] for _ in range(2))
        used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
        used[self.rows(self.prefix_pages, prefix)] = True
        for i, n in enumerate(self.lens):
            used[self.rows(self.table[i], n)] = True
        used = used.view(pages, page)
        for c, junk in ((self.kc, float("nan")), (self.vc, float("inf"))):
            (c.transpose(1, 2) if heads_first else c)[~used] = junk
        self.q = (q_size * lu.randn(g, b, hkv * group, d + q_gap)).to(t)[..., :d]
        self.own_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.out = torch.full((b + 1, hkv * group, d), 9.0, dtype=t, device="cuda")
        self.scale = d ** -0.5

    def rows(self, pages, n):
        at = torch.arange(n, device="cuda")
        return pages.long()[at // self.page] * self.page + at % self.page

    def params(self):
        kc, q = self.kc, self.q
        token, head = (kc.stride(2), kc.stride(1)) if self.heads_first else (kc.stride(1), kc.stride(2))
        p = capi.PrefixAttnParams(dtype=lu.CODES[self.ty], batch=len(self.lens), q_heads=q.shape[1], kv_heads=self.hkv, head_dim=self.d, page_size=self.page, max_blocks=self.each,
                                  prefix_len=self.prefix, max_own_len=self.most, scale=self.scale, n_pages=kc.shape[0], q_stride=q.stride(0), q_head_stride=q.stride(1),
                                  out_stride=self.out.stride(0), out_head_stride=self.out.stride(1), page_stride=kc.stride(0), token_stride=token, head_stride=head,
                                  table_stride=self.table.stride(0), q=lu.ptr(q), out=lu.ptr(self.out), k_cache=lu.ptr(kc), v_cache=lu.ptr(self.vc),
                                  prefix_pages=lu.ptr(self.prefix_pages), block_table=lu.ptr(self.table) if self.most else None, own_lens=lu.ptr(self.own_lens) if self.most else None)
        n = lu.info("prefix_attn", p).scratch_bytes
        self.scratch = torch.full((max(n, 16) + 16,), 255, dtype=torch.uint8, device="cuda")          # NaNs, and a guard behind the end
        p.scratch, p.scratch_bytes = lu.ptr(self.scratch), n
        return p

    def run(self):
        p = self.params()
        lu.launch("prefix_attn", p)
        gu.sync()
        assert bool((self.out[-1] == 9.0).all()) and bool((self.scratch[-16:] == 255).all())
        return self.out[:-1]

    def tokens(self, cache, i):
        c = (cache.transpose(1, 2) if self.heads_first else cache).reshape(-1, self.hkv, self.d)
        return c[torch.cat([self.rows(self.prefix_pages, self.prefix), self.rows(self.table[i], self.lens[i])])].double()

    def check(self, got, only=None):
        worst = 0.0
        for i, n in enumerate(self.lens):
            if only is not None and i not in only:
                continue
            if self.prefix + n == 0:
                assert bool((got[i] == 0).all())
                continue
            k, v = self.tokens(self.kc, i), self.tokens(self.vc, i)
            q = self.q[i].double().view(self.hkv, self.group, self.d)
            s = torch.einsum("hgd,nhd->hgn", q, k) * self.scale
            size = float(torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()).max() * abs(self.scale))
            w = torch.softmax(s, -1)
            ref, mag = torch.einsum("hgn,nhd->hgd", w, v), torch.einsum("hgn,nhd->hgd", w, v.abs())
            half, seen = lu.HALF_STEP[self.ty], self.prefix + n
            small = (self.d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + float(s.abs().max()) * 1.45) + (seen + 40) * 2.0 ** -23
            off = (got[i].double().view_as(ref) - ref).abs()
            bound = (half + small) * mag + half * ref.abs() + lu.TINY[self.ty] * 2
            worst = max(worst, float((off / bound).max()))
        assert worst <= 1.0, worst


# batches and groups that leave tiles of query rows partly filled; prefixes and own lengths around pages and key tiles, none of either, very uneven ones
@pytest.mark.parametrize("lens,hkv,group,d,prefix,page", [
    ([1], 1, 1, 64, 0, 16), ([0], 1, 1, 64, 1, 16), ([5], 2, 4, 128, 7, 16), ([0, 0, 0], 2, 3, 64, 130, 16), ([3, 0, 17, 64], 2, 4, 64, 300, 16),
    ([1, 2, 127, 128, 129, 255, 256, 257], 1, 8, 128, 128, 64), ([33] * 5, 8, 5, 80, 257, 32), ([0, 700], 1, 16, 96, 127, 8), ([40, 41], 4, 1, 128, 4096, 128),
    ([9] * 64, 2, 4, 64, 1000, 16), ([0, 64, 3] * 11, 1, 7, 112, 129, 24), ([20] * 17, 1, 8, 128, 640, 64), ([100] * 3, 2, 2, 8, 50, 8), ([7] * 40, 3, 8, 128, 2049, 256),
    ([1000, 0, 5, 2500], 2, 8, 128, 0, 64), ([600] * 2, 1, 32, 64, 333, 40), ([0] * 130, 1, 2, 128, 515, 32), ([3] * 300, 1, 1, 40, 77, 16), ([11] * 2, 1, 128, 128, 200, 16),
    ([5] * 3, 1, 71, 64, 5000, 64), ([2] * 100, 1, 6, 128, 9001, 128),
    ([0, 17, 40, 1] * 75, 2, 3, 64, 515, 16), ([33, 0] * 65, 8, 2, 128, 300, 24), ([1] * 64, 1, 128, 112, 200, 32)])
@pytest.mark.parametrize("ty,heads_first", [("bf16", False), ("f16", True)])
def test_attention(ty, heads_first, lens, hkv, group, d, prefix, page):
    p = Problem(lens, hkv, group, d, prefix, page, ty, heads_first)
    p.check(p.run())
    assert gu.error_flag() == 0


@pytest.mark.parametrize("lens,prefix", [([3, 0, 70, 12], 200), ([0, 0, 1], 0), ([4] * 40, 700)])
def test_strides_and_a_longer_bound(lens, prefix):
    """Rows of q inside longer ones, a cache whose rows have gaps, a bound on the lengths far above them."""
    p = Problem(lens, 2, 4, 64, prefix, 16, q_gap=24, cache_gap=8, most=1000)
    p.check(p.run())
    p = Problem(lens, 2, 4, 64, prefix, 16, heads_first=True, cache_gap=64, most=97)
    p.check(p.run())


@pytest.mark.parametrize("prefix,lens", [(900, [50, 0, 3]), (0, [300, 1, 0]), (129, [0, 0, 0])])
@pytest.mark.parametrize("q_size,scale", [(30.0, None), (0.0, None), (1.5, -0.3), (1.0, 0.0), (6.0, 1.0)])
def test_peaked_and_flat_softmax(prefix, lens, q_size, scale):
    """One key that takes all, all keys alike, a negative scale, growing maxima from tile to tile."""
    p = Problem(lens, 2, 4, 128, prefix, 32, q_size=q_size)
    if scale is not None:
        p.scale = scale
    p.check(p.run())
    if q_size == 6.0:                                            # keys that grow along the prefix: the maximum moves in every tile
        p = Problem(lens, 2, 4, 128, prefix, 32, q_size=q_size)
        rows = p.rows(p.prefix_pages, prefix)
        k = p.kc.reshape(-1, 2, 128)
        k[rows] = (k[rows].float() * torch.linspace(0.02, 1.0, max(prefix, 1), device="cuda")[:prefix, None, None]).to(k.dtype)
        p.kc = k.view_as(p.kc)
        p.check(p.run())


def test_infinite_and_nan_scores_stay_in_their_rows():
    p = Problem([4, 4, 4], 1, 2, 64, 150, 16)
    p.q[1, 0, 3] = float("nan")
    got = p.run()
    assert bool(got[1, 0].isnan().all()) and not bool(got[1, 1].isnan().any())
    p.q[1, 0, 3] = 0.0
    p.check(got, only=(0, 2))
    p = Problem([4, 4, 4], 1, 2, 64, 150, 16)
    p.kc.view(-1, 1, 64)[p.rows(p.table[2], 4)[1]] = float("nan")       # one own key of the last sequence
    got = p.run()
    assert bool(got[2].isnan().all()) and not bool(got[:2].isnan().any())
    p.check(got, only=(0, 1))


def test_bad_lengths_and_pages_are_flagged():
    for prefix in (0, 100):
        p = Problem([4, 30, 9], 2, 2, 64, prefix, 16)
        p.own_lens[0], p.own_lens[1] = -3, 31                    # count as 0 and as the most
        p.lens[0] = 0
        p.check(p.run())
        assert gu.error_flag() != 0 and gu.error_flag() == 0
    for bad in (-1, 10 ** 9, None):                              # None: the first number that is none
        p = Problem([4, 40, 9], 2, 2, 64, 100, 16)
        n = p.kc.shape[0]
        zero = torch.zeros(1, *p.kc.shape[1:], dtype=p.kc.dtype, device="cuda")
        kc, vc, pages, table = p.kc, p.vc, p.prefix_pages.clone(), p.table.clone()
        p.prefix_pages[2], p.table[1, 1] = n if bad is None else bad, n if bad is None else bad
        got = p.run()
        assert gu.error_flag() != 0 and gu.error_flag() == 0
        p.kc, p.vc = torch.cat([kc, zero]), torch.cat([vc, zero])
        p.prefix_pages, p.table = pages, table
        p.prefix_pages[2], p.table[1, 1] = n, n                  # a page of zeros
        p.check(got)


def test_cache_behind_four_billion_elements():
    p = Problem([20, 3], 8, 4, 128, 200, 64, extra_pages=0)
    pages, n = 66000, p.kc.shape[0]                              # 66000 x 64 x 8 x 128 = 4.3e9 elements
    big = [torch.empty(pages, 64, 8, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for b, c in zip(big, (p.kc, p.vc)):
        b[pages - n:] = c
    ref = p.run().clone()
    p.check(ref)
    p.kc, p.vc = big
    p.prefix_pages, p.table = p.prefix_pages + (pages - n), p.table + (pages - n)
    p.out.fill_(9.0)
    assert torch.equal(p.run(), ref)


@pytest.mark.parametrize("lens,prefix", [([5, 0, 300], 1000), ([5, 0, 300], 0), ([0, 0, 0], 1000), ([17] * 50, 3000), ([40, 3] * 150, 700)])
def test_captured_with_other_lengths_and_the_same_bits_again(lens, prefix):
    """A graph's launches read lengths, tables and queries at each replay; the same inputs give the same bits."""
    p = Problem(lens, 2, 4, 128, prefix, 32, most=max(lens))
    params, first = p.params(), None
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    q0, lens0 = p.q.clone(), p.own_lens.clone()
    qs, ls = q0.clone(), lens0.clone()
    with torch.cuda.graph(graph, stream=st):
        p.q.copy_(qs)
        p.own_lens.copy_(ls)
        lu.launch("prefix_attn", params)
        lu.launch("prefix_attn", params)                         # twice in a row over the same scratch memory
    for i in range(3):
        half = [n // 2 for n in lens] if i == 1 else lens
        ls.copy_(torch.tensor(half, dtype=torch.int32))
        qs.copy_(-q0 if i == 1 else q0)
        graph.replay()
        gu.sync()
        p.lens = half
        p.check(p.out[:-1])
        if i == 0:
            first = p.out.clone()
    assert torch.equal(first, p.out)
    assert gu.error_flag() == 0


@pytest.mark.parametrize("lens,prefix", [([5, 0, 300], 1000), ([5, 0, 300], 0), ([0, 0, 0], 1000), ([2] * 100, 50), ([], 100), ([9, 0] * 150, 400)])
def test_notifications_count_the_declared_blocks(lens, prefix):
    p = Problem(lens or [1], 2, 4, 128, prefix, 32)
    params = p.params()
    params.batch = len(lens)
    n = lu.info("prefix_attn", params).num_blocks
    assert lu.records("prefix_attn", params) == (n, n)
    if lens:
        p.check(p.out[:-1])
    else:
        assert bool((p.out == 9.0).all())


@pytest.mark.parametrize("most", [0, 64, 5000])
def test_no_tokens_at_all_and_no_sequences(most):
    p = Problem([0, 0, 0], 2, 4, 64, 0, 16, most=most)
    p.check(p.run())
    params = p.params()
    params.batch = 0
    p.out.fill_(9.0)
    n = lu.info("prefix_attn", params).num_blocks
    assert lu.records("prefix_attn", params) == (n, n)
    assert bool((p.out == 9.0).all()) and gu.error_flag() == 0


def test_sequences_that_share_pages():
    """The same page for several sequences, twice for one, and for the prefix too."""
    p = Problem([40, 64, 33], 2, 4, 64, 70, 16)
    p.table[1, :4], p.table[2, :3] = p.table[0, 0], p.prefix_pages[1]
    p.check(p.run())


def test_two_streams_at_once():
    """Calls with scratch memory of their own on two streams and the current one give what they give alone."""
    ps = [Problem([30, 0, 500], 2, 4, 128, 5000, 32), Problem([7] * 160, 4, 4, 64, 900, 16, ty="f16"), Problem([3, 90], 2, 8, 128, 300, 64)]
    alone = [p.run().clone() for p in ps]
    params, streams = [p.params() for p in ps], [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream()]
    for p in ps:
        p.out.fill_(9.0)
    torch.cuda.synchronize()
    for _ in range(30):
        for pa, st in zip(params, streams):
            lu.launch("prefix_attn", pa, st)
    torch.cuda.synchronize()
    for p, ref in zip(ps, alone):
        assert torch.equal(p.out[:-1], ref)
    assert gu.error_flag() == 0


@pytest.mark.parametrize("page", [16, 64, 128])
def test_long_prefix_of_one_row_tile(page):
    """Many tiles through the rings of a block whose groups take every other tile; the same bits each time."""
    p = Problem([1] * 16, 2, 8, 128, 70001, page)
    first = p.run().clone()
    p.check(first, only=(0, 15))
    params = p.params()
    for _ in range(40):
        lu.launch("prefix_attn", params)
    gu.sync()
    assert torch.equal(p.out[:-1], first) and gu.error_flag() == 0


def test_a_decode_step_of_the_operators_together():
    """Dense layer in 8-bit integers -> norms, rotation and append -> attention, two steps in a row: what a layer does to serve a token.  The second step
    reads what the first appended.  Compared with the operators' formulas on each operator's own inputs, so that each error counts once."""
    g, b, hkv, group, d, page, prefix, hidden = lu.gen(1), 6, 2, 4, 64, 16, 100, 512
    p = Problem([n for n in (3, 0, 31, 15, 16, 40)], hkv, group, d, prefix, page, most=64)
    width = (hkv * group + 2 * hkv) * d
    w = torch.randint(-127, 128, (width, hidden), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.full((width,), 1 / (73 * math.sqrt(hidden)), device="cuda")
    xq, xs = torch.empty(b, hidden, dtype=torch.int8, device="cuda"), torch.empty(b, device="cuda")
    qkv = torch.empty(b, width // d, d, dtype=torch.bfloat16, device="cuda")
    wt = torch.ones(d, device="cuda")
    at = torch.arange(400, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    tab = torch.cat([at.cos(), at.sin()], 1).float().contiguous()
    for step in range(2):
        x = lu.randn(g, b, hidden).bfloat16()
        q, k, v = qkv[:, :hkv * group], qkv[:, hkv * group:hkv * group + hkv], qkv[:, hkv * group + hkv:]
        lu.launch("int8_quantize", capi.Int8QuantizeParams(tokens=b, channels=hidden, x_dtype=capi.BF16, x_stride=hidden, q_stride=hidden, x=lu.ptr(x), q=lu.ptr(xq), scale=lu.ptr(xs)))
        lu.launch("int8_dense", capi.Int8DenseParams(tokens=b, in_channels=hidden, out_channels=width, y_dtype=capi.BF16, x_stride=hidden, w_stride=hidden, y_stride=width,
                                                     x=lu.ptr(xq), x_scale=lu.ptr(xs), w=lu.ptr(w), w_scale=lu.ptr(ws), y=lu.ptr(qkv)))
        lens = torch.tensor(p.lens, device="cuda")
        slots = p.table.gather(1, (lens // page)[:, None]).flatten().long() * page + lens % page
        pos = (prefix + lens).int()
        kc = p.kc
        lu.launch("kv_append", capi.KvAppendParams(dtype=capi.BF16, tokens=b, q_heads=hkv * group, kv_heads=hkv, head_dim=d, rot_dim=d, max_position=400, eps=1e-6, page_size=page,
                                                   n_pages=kc.shape[0], k_stride=width, k_head_stride=d, v_stride=width, v_head_stride=d, page_stride=kc.stride(0),
                                                   token_stride=kc.stride(1), head_stride=kc.stride(2), k=lu.ptr(k), v=lu.ptr(v), k_weight=lu.ptr(wt), cos_sin=lu.ptr(tab),
                                                   positions=lu.ptr(pos), slots=lu.ptr(slots), k_cache=lu.ptr(kc), v_cache=lu.ptr(p.vc), q_stride=width, q_head_stride=d,
                                                   q_out_stride=hkv * group * d, q_out_head_stride=d, q=lu.ptr(q), q_out=lu.ptr(p.q), q_weight=lu.ptr(wt)))
        p.own_lens += 1
        p.lens = [n + 1 for n in p.lens]
        got = p.run()
        # each operator against its formula on what it was given
        ref = (xq.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
        assert bool(((qkv.view(b, -1).double() - ref).abs() <= 2.0 ** -7 * ref.abs() + 1e-5).all())
        z = q.double() / (q.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        c, s = tab.double()[pos.long()][:, None, :d // 2], tab.double()[pos.long()][:, None, d // 2:]
        turned = torch.cat([z[..., :d // 2] * c - z[..., d // 2:] * s, z[..., d // 2:] * c + z[..., :d // 2] * s], -1)
        assert bool(((p.q.double() - turned).abs() <= 2.0 ** -7 * turned.abs() + 1e-4).all())
        assert torch.equal(p.vc.view(-1, hkv, d)[slots], v)
        p.check(got)
    assert gu.error_flag() == 0
