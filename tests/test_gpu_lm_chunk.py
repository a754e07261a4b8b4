"""Attention of chunks of new tokens over a paged cache (pb_chunk_attn) against the formula in 64 bits.

Tolerance, relative to sum p |v| / sum p (`mag`), as for pb_prefix_attn: the softmax's values are rounded to the cache's type once (its half step); a
score's product sums head_dim terms in fp32, at most (head_dim + 8) x 2^-24 x scale x sum |q k| off, which changes its
exponential by as much, as do the score's scaling and the subtraction of the maximum (2^-23 x the largest |score|, in powers of
two), and the exponentials are off by 2^-22; the sums of the p and of the p v add at most as many terms as there are tokens, each rounding
2^-24, and merging parts adds some 40 more.  Beside it the output's own rounding."""
import math

import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


class Problem:
    """`seqs`: (new tokens, tokens in the cache) of each sequence.  Pages are dealt at random; what no token lies in holds NaNs and infinities."""

    def __init__(self, seqs, hkv, group, d, page, ty="bf16", window=0, heads_first=False, most_new=None, most_len=None, q_gap=0, cache_gap=0, padded=0, seed=0, q_size=1.5, extra_pages=2):
        g = lu.gen(seed + d + page + len(seqs))
        self.seqs, self.hkv, self.group, self.d, self.page, self.ty, self.window, self.heads_first = list(seqs), hkv, group, d, page, ty, window, heads_first
        b, t = len(self.seqs), lu.TYPES[ty]
        self.most_new = max([n for n, _ in seqs] + [0]) if most_new is None else most_new
        self.most_len = max([l for _, l in seqs] + [0]) if most_len is None else most_len
        self.each = -(-self.most_len // page)
        need = [-(-l // page) for _, l in seqs]
        pages = sum(need) + extra_pages
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((b, self.each + 3), -5, dtype=torch.int32, device="cuda")          # entries behind a sequence's last page are not used
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        inner = (hkv, page) if heads_first else (page, hkv)
        self.kc, self.vc = ((lu.randn(g, pages, *inner, d + cache_gap)).to(t)[..., :d] for _ in range(2))
        used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
        for i, (_, l) in enumerate(self.seqs):
            used[self.rows(i, l)] = True
        used = used.view(pages, page)
        for c, junk in ((self.kc, NAN), (self.vc, INF)):
            (c.transpose(1, 2) if heads_first else c)[~used] = junk
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1] + padded
        self.starts, self.lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, [l for _, l in seqs]))
        self.first = starts
        self.q = (q_size * lu.randn(g, self.tokens, hkv * group, d + q_gap)).to(t)[..., :d]
        self.out = torch.full((self.tokens + 1, hkv * group, d), 9.0, dtype=t, device="cuda")
        self.scale = d ** -0.5

    def rows(self, i, n):
        at = torch.arange(n, device="cuda")
        return self.table[i].long()[at // self.page] * self.page + at % self.page

    def params(self):
        kc, q = self.kc, self.q
        token, head = (kc.stride(2), kc.stride(1)) if self.heads_first else (kc.stride(1), kc.stride(2))
        p = capi.ChunkAttnParams(dtype=lu.CODES[self.ty], batch=len(self.seqs), tokens=self.tokens, q_heads=self.hkv * self.group, kv_heads=self.hkv, head_dim=self.d, page_size=self.page,
                                 max_blocks=self.each, max_new=self.most_new, max_len=self.most_len, window=self.window, scale=self.scale, n_pages=kc.shape[0], q_stride=q.stride(0),
                                 q_head_stride=q.stride(1), out_stride=self.out.stride(0), out_head_stride=self.out.stride(1), page_stride=kc.stride(0), token_stride=token, head_stride=head,
                                 table_stride=self.table.stride(0), q=lu.ptr(q), out=lu.ptr(self.out), k_cache=lu.ptr(kc), v_cache=lu.ptr(self.vc), block_table=lu.ptr(self.table),
                                 starts=lu.ptr(self.starts), lens=lu.ptr(self.lens))
        n = lu.info("chunk_attn", p).scratch_bytes
        self.scratch = torch.full((max(n, 16) + 16,), 255, dtype=torch.uint8, device="cuda")          # NaNs, and a guard behind the end
        p.scratch, p.scratch_bytes = lu.ptr(self.scratch), n
        return p

    def run(self):
        p = self.params()
        lu.launch("chunk_attn", p)
        gu.sync()
        assert bool((self.out[self.first[-1]:] == 9.0).all()) and bool((self.scratch[-16:] == 255).all())
        return self.out[:-1]

    def cached(self, cache, i):
        c = (cache.transpose(1, 2) if self.heads_first else cache).reshape(-1, self.hkv, self.d)
        return c[self.rows(i, self.seqs[i][1])].double()

    def check(self, got, only=None, skip=None):
        worst = 0.0
        for i, (n, l) in enumerate(self.seqs):
            if n == 0 or (only is not None and i not in only):
                continue
            mine = got[self.first[i]:self.first[i] + n]
            none = max(0, n - l)                              # rows in front of the first token
            assert bool((mine[:none] == 0).all())
            if none == n:
                continue
            k, v = self.cached(self.kc, i).nan_to_num(0.0, 0.0, 0.0), self.cached(self.vc, i).nan_to_num(0.0, 0.0, 0.0)
            step = max(1, 40_000_000 // (self.hkv * self.group * l))
            for a in range(none, n, step):
                z = min(n, a + step)
                q = self.q[self.first[i] + a:self.first[i] + z].double().view(z - a, self.hkv, self.group, self.d)
                s = torch.einsum("nhgd,mhd->hgnm", q, k) * self.scale
                pos = torch.arange(l - n + a, l - n + z, device="cuda")[:, None]
                at = torch.arange(l, device="cuda")
                seen = at <= pos
                if self.window:
                    seen &= at > pos - self.window
                size = float(torch.einsum("nhgd,mhd->hgnm", q.abs(), k.abs()).max() * abs(self.scale))
                w = torch.softmax(s.masked_fill(~seen, -INF), -1)
                ref, mag = torch.einsum("hgnm,mhd->nhgd", w, v), torch.einsum("hgnm,mhd->nhgd", w, v.abs())
                half = lu.HALF_STEP[self.ty]
                small = (self.d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + float(s.abs().max()) * 1.45) + (min(l, self.window or l) + 40) * 2.0 ** -23
                off = (mine[a:z].double().view_as(ref) - ref).abs()
                bound = (half + small) * mag + half * ref.abs() + lu.TINY[self.ty] * 2
                off = (off / bound).nan_to_num(9e9)
                if skip is not None:
                    off = off.masked_fill(skip[self.first[i] + a:self.first[i] + z].view_as(off), 0.0)
                worst = max(worst, float(off.max()))
        assert worst <= 1.0, worst


SEQS = [[(1, 1)], [(1, 0)], [(1, 300)], [(5, 5)], [(5, 3)], [(7, 2), (0, 9), (3, 3)], [(1, 77), (1, 128), (1, 129), (1, 4000)], [(0, 0), (0, 50)], [(2, 2), (4, 900), (1, 17), (64, 64), (33, 190)],
        [(128, 128)], [(129, 129)], [(127, 383)], [(300, 300)], [(256, 1000), (1, 1000), (2, 1000)], [(700, 2500)], [(1, 500)] * 40 + [(90, 95)], [(16, 1030), (17, 1031)], [(1500, 1500)], [(40, 10), (40, 45)],
        [(3, 20)] * 70, [(1, 9000)], [(260, 9001)]]


# one token and many, in front of nothing and of long caches, rows that see nothing, groups and pages that end inside tiles
@pytest.mark.parametrize("seqs", SEQS, ids=range(len(SEQS)))
@pytest.mark.parametrize("hkv,group,d,page,ty,heads_first", [(2, 4, 128, 16, "bf16", False), (1, 1, 64, 64, "f16", True), (3, 5, 80, 24, "f16", False), (2, 8, 96, 32, "bf16", True), (1, 3, 8, 8, "bf16", False),
                                                             (1, 16, 128, 128, "bf16", False), (1, 71, 120, 40, "f16", True)])
def test_sequences(seqs, hkv, group, d, page, ty, heads_first):
    p = Problem(seqs, hkv, group, d, page, ty, heads_first=heads_first)
    p.check(p.run())
    assert gu.error_flag() == 0


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 1000, 100000])
@pytest.mark.parametrize("seqs", [SEQS[i] for i in (2, 5, 6, 8, 12, 13, 14, 15, 18, 20, 21)], ids=range(11))
@pytest.mark.parametrize("hkv,group,d,page,ty", [(2, 4, 128, 16, "bf16"), (1, 5, 64, 24, "f16")])
def test_windows(window, seqs, hkv, group, d, page, ty):
    p = Problem(seqs, hkv, group, d, page, ty, window=window)
    p.check(p.run())
    assert gu.error_flag() == 0


@pytest.mark.parametrize("seqs", [[(1, 700), (1, 20), (1, 0)], [(30, 700), (3, 20)], [(400, 700), (1, 200)]])
@pytest.mark.parametrize("kw", [dict(q_gap=8), dict(cache_gap=8), dict(q_gap=24, cache_gap=16, heads_first=True), dict(padded=37), dict(most_new=3000), dict(most_len=5000), dict(most_new=1000, most_len=3001, padded=2)])
def test_strides_bounds_and_padding(seqs, kw):
    p = Problem(seqs, 2, 4, 128, 16, **kw)
    p.check(p.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0, 1e-30])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("seqs", [[(1, 700), (1, 3)], [(200, 700), (1, 200)]])
def test_scales(scale, ty, seqs):
    p = Problem(seqs, 2, 4, 64, 16, ty, q_size=0.5)
    p.scale = scale
    p.check(p.run())


@pytest.mark.parametrize("seqs", [[(1, 900), (1, 130)], [(130, 900), (2, 130)], [(9, 900)]])
def test_scores_far_apart(seqs):
    """Maxima that grow from key to key, and keys that come to nothing beside one."""
    p = Problem(seqs, 1, 4, 128, 32)
    ramp = torch.linspace(-40, 40, 900, device="cuda")
    for i, (_, l) in enumerate(seqs):
        c = p.kc.view(-1, 1, 128)
        c[p.rows(i, l), 0, 0] = ramp[:l].to(c.dtype)
    p.q[:, :, 0] = 30.0
    p.check(p.run())
    p.q[:, :, 0] = -30.0
    p.check(p.run())


@pytest.mark.parametrize("where", ["last", "behind the first rows", "in front of the window", "first"])
@pytest.mark.parametrize("seqs,group,window", [([(200, 500)], 4, 0), ([(200, 500), (4, 300)], 1, 90), ([(6, 400)], 2, 0), ([(700, 700)], 8, 0), ([(3, 300)], 5, 100), ([(1, 200), (1, 300)], 4, 100)])
@pytest.mark.parametrize("kind", ["k nan", "k inf", "v nan", "v inf"])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(where, seqs, group, window, kind):
    p = Problem(seqs, 2, group, 64, 16, window=window)
    n, l = seqs[0]
    j = {"last": l - 1, "behind the first rows": l - n + n // 2, "in front of the window": max(0, l - n - (window or 0) + n // 2), "first": 0}[where]
    row = int(p.rows(0, l)[j])
    cache = p.kc if kind[0] == "k" else p.vc
    bad = NAN if kind.endswith("nan") else INF
    cache.view(-1, 2, 64)[row, 1, 5] = bad                         # of key head 1
    if kind == "k inf":
        p.q[:, :, 5] = p.q[:, :, 5].abs() + 0.1
    got = p.run()
    pos = torch.arange(l - n, l, device="cuda")
    sees = (j <= pos) & ((j > pos - window) if window else True)
    skip = torch.zeros(p.tokens, 2, group, 64, dtype=torch.bool, device="cuda")
    if kind[0] == "k":
        skip[:n, 1] = sees[:, None, None]
        assert bool(got.view(p.tokens, 2, group, 64)[skip[:p.tokens]].isnan().all())
    else:
        skip[:n, 1, :, 5] = sees[:, None]
        hit = got.view(p.tokens, 2, group, 64)[skip[:p.tokens]]
        assert bool((hit.isnan() if kind == "v nan" else hit == INF).all())
    p.check(got, skip=skip)


def test_bad_lengths_pages_and_starts():
    p = Problem([(1, 100), (1, 40)], 2, 4, 64, 16)
    p.lens[0] = 10 ** 6
    p.run()
    assert gu.error_flag() == 0x303
    for seqs in ([(1, 100), (1, 40), (1, 33)], [(20, 100), (1, 40), (30, 33)]):
        p = Problem(seqs, 2, 4, 64, 16)
        p.lens[0], p.lens[1] = 10 ** 6, -3                         # counts as max_len, which sequence 0 has; as 0
        got = p.run()
        p.check(got, only=[0, 2])
        assert bool((got[p.first[1]:p.first[2]] == 0).all())
        assert gu.error_flag() == 0x303
        for bad in (-1, p.kc.shape[0], 2 ** 31 - 1, -2 ** 31):
            p = Problem(seqs, 2, 4, 64, 16)
            rows, page = p.rows(0, 100)[32:48], int(p.table[0, 2])
            p.table[0, 2] = bad
            got = p.run()
            assert gu.error_flag() == 0x304
            p.table[0, 2] = page                                   # a page of zeros
            p.kc.view(-1, 2, 64)[rows] = 0.0
            p.vc.view(-1, 2, 64)[rows] = 0.0
            p.check(got)
    # more new tokens than max_new: the first of them, at the positions that they have
    p = Problem([(20, 100), (5, 40)], 2, 4, 64, 16, most_new=8)
    got = p.run()
    assert gu.error_flag() == 0x303 and bool((got[8:20] == 9.0).all())
    whole = Problem([(20, 100), (5, 40)], 2, 4, 64, 16)
    whole.check(torch.cat([got[:8], whole.run()[8:20], got[20:]]))
    # starts that fall, or lie outside
    for starts in ([-4, 20, 25], [0, 20, 10], [30, 20, 25], [0, 2 ** 31 - 1, 25], [5, 5, -9], [2 ** 31 - 1, -2 ** 31, 25]):
        p = Problem([(20, 100), (5, 40)], 2, 4, 64, 16)
        p.starts.copy_(torch.tensor(starts, dtype=torch.int64).to(torch.int32))
        lu.launch("chunk_attn", p.params())
        gu.sync()
        assert bool((p.out[-1] == 9.0).all()) and not bool(p.out.isnan().any()) and gu.error_flag() == 0x303


def test_the_same_bits_each_time_and_captured():
    for seqs in ([(1, 3000)] * 5, [(30, 700), (3, 20), (1, 5000)], [(900, 2000)]):
        p = Problem(seqs, 2, 4, 128, 32)
        params = p.params()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lu.launch("chunk_attn", params, stream=side)
        graph.replay()
        gu.sync()
        p.check(p.out[:-1])
        first = p.out.clone()
        for _ in range(20):
            graph.replay()
        gu.sync()
        assert torch.equal(p.out, first)
        # other lengths, read when the kernels run
        p.seqs = [(n, max(0, l - 7)) for n, l in p.seqs]
        p.lens -= 7
        p.lens.clamp_(min=0)
        graph.replay()
        gu.sync()
        p.check(p.out[:-1])


def test_notifications():
    for seqs in ([(1, 300)] * 9, [(30, 700), (3, 20)], [(900, 2000)], []):
        p = Problem(seqs, 2, 4, 128, 32)
        params = p.params()
        li = lu.info("chunk_attn", params)
        assert lu.records("chunk_attn", params) == (li.num_blocks, li.num_blocks)


def test_several_streams_with_a_scratch_each():
    a, b = Problem([(300, 1500), (1, 900)], 2, 4, 128, 32), Problem([(20, 5000), (700, 900)], 2, 4, 128, 32, seed=3)
    pa, pb, sa, sb = a.params(), b.params(), torch.cuda.Stream(), torch.cuda.Stream()
    gu.sync()
    for _ in range(30):
        lu.launch("chunk_attn", pa, stream=sa)
        lu.launch("chunk_attn", pb, stream=sb)
    gu.sync()
    a.check(a.out[:-1])
    b.check(b.out[:-1])


def test_a_cache_whose_offsets_pass_32_bits():
    """Pages that lie 2^31 elements apart and more."""
    hkv, group, d, page, n_pages, stride = 1, 4, 64, 16, 5, 2 ** 30 + 2 ** 29
    store = torch.zeros((n_pages - 1) * stride + page * d, dtype=torch.bfloat16, device="cuda")
    for seqs in ([(1, 70)], [(40, 70)]):
        p = Problem(seqs, hkv, group, d, page, extra_pages=0)
        assert p.kc.shape[0] == n_pages
        view = torch.as_strided(store, (n_pages, page, hkv, d), (stride, d, d, 1))
        view.copy_(p.kc)
        params = p.params()
        params.k_cache, params.page_stride = lu.ptr(store), stride
        vs = torch.zeros_like(store)
        torch.as_strided(vs, (n_pages, page, hkv, d), (stride, d, d, 1)).copy_(p.vc)
        params.v_cache = lu.ptr(vs)
        lu.launch("chunk_attn", params)
        gu.sync()
        del vs
        p.check(p.out[:-1])
