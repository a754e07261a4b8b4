"""Starts of sequences that fall (pb_chunk_attn): each counts as the highest in front of it, so that no row belongs to two sequences.  The results are those, bit for bit, of a call that is given the
starts as they count, and those are compared with 64 bits."""
import pytest
import torch

from paella_b200 import capi
from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_chunk import Problem

pytestmark = pytest.mark.gpu


def counted(starts, tokens):
    out, high = [], 0
    for s in starts:
        high = max(high, min(max(s, 0), tokens))
        out.append(high)
    return out


def run(starts, lens, most_new, tokens, hkv=2, group=4, d=64, page=16, ty="bf16", window=0, bad=()):
    """Out of a call with these starts (in a problem whose sequences are those of the starts as they count), and its problem."""
    as_they_count = counted(starts, tokens)
    seqs = [(b - a, l) for a, b, l in zip(as_they_count, as_they_count[1:], lens)]
    p = Problem(seqs, hkv, group, d, page, ty, window=window, most_new=most_new)
    assert p.first[-1] + as_they_count[0] == as_they_count[-1]
    p.q = 1.5 * lu.randn(lu.gen(3), tokens, hkv * group, d)
    p.q = p.q.to(lu.TYPES[ty])
    p.tokens, p.first = tokens, as_they_count
    outs = []
    for given in (starts, as_they_count):
        p.out = torch.full((tokens + 1, hkv * group, d), 9.0, dtype=lu.TYPES[ty], device="cuda")
        p.starts = torch.tensor(given, dtype=torch.int64).to(torch.int32).to("cuda")
        params = p.params()
        for _ in range(4):
            lu.launch("chunk_attn", params)
        gu.sync()
        assert bool((p.scratch[-16:] == 255).all())
        want = 0x303 if list(given) != as_they_count or any(n > most_new for n, _ in seqs) else 0
        assert gu.error_flag(reset=True) == want
        outs.append(p.out)
    assert torch.equal(outs[0], outs[1])
    mine = torch.zeros(tokens + 1, dtype=torch.bool, device="cuda")
    for (n, _), a in zip(seqs, as_they_count):
        mine[a:a + min(n, most_new)] = True
    assert bool((outs[0][~mine] == 9.0).all())
    if max(n for n, _ in seqs) <= most_new:
        p.check(outs[0][:-1])


STARTS = [[0, 20, 10, 25], [0, 20, 10, 15, 30], [0, 5, 2, 4, 3, 9, 1, 12], [30, 20, 10, 0, 40], [0, 300, 20, 320], [0, 300, 20, 900], [0, 600, 0, 600, 0, 600, 700], [3, 1, 2, 3, 4, 5, 6, 7, 8],
          [0, 2 ** 31 - 1, 5, 9], [-4, 10, -9, 12, -2 ** 31, 20], [0, 40, 30, 31, 32, 33, 34, 35, 36, 37, 38, 39, 41, 42], [0, 1000, 999, 1001, 1000, 1003]]


@pytest.mark.parametrize("starts", STARTS, ids=range(len(STARTS)))
@pytest.mark.parametrize("most_new", [1, 4, 100, 2000])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("group,d,ty", [(4, 64, "bf16"), (5, 96, "f16")])
def test_starts_that_fall(starts, most_new, window, group, d, ty):
    tokens = max(s for s in starts if s < 10 ** 6) + 30
    run(starts, [30 + 700 * (i % 3) for i in range(len(starts) - 1)], most_new, tokens, group=group, d=d, ty=ty, window=window)


# more sequences than a warp looks through, than a block has threads, and as many as both take
@pytest.mark.parametrize("batch", [31, 32, 33, 255, 256, 257, 300, 1023, 1024, 1025, 2600])
@pytest.mark.parametrize("most_new", [1, 40])
@pytest.mark.parametrize("falls", [False, True])
def test_many_sequences(batch, most_new, falls):
    g = torch.Generator().manual_seed(batch)
    starts = torch.arange(batch + 1) * 2
    if falls:
        starts = starts + torch.where(torch.rand(batch + 1, generator=g) < 0.1, torch.randint(-60, 60, (batch + 1,), generator=g), torch.zeros((), dtype=torch.int64))
        starts[batch // 2] = 7
    run(starts.tolist(), [5 + (37 * i) % 90 for i in range(batch)], most_new, 2 * batch + 30, hkv=1)


def test_a_high_start_far_in_front():
    for batch, at in ((200, 0), (256, 3), (300, 40), (1500, 900), (2100, 1023)):
        starts = list(range(batch + 1))
        starts[at] = batch - 5
        run(starts, [3 + i % 50 for i in range(batch)], 1, batch + 1, hkv=1)


def test_captured_and_replayed_with_other_starts():
    """The starts are read when the kernels run."""
    for batch in (20, 300):
        p = Problem([(2, 60)] * batch, 1, 4, 64, 16)
        params = p.params()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lu.launch("chunk_attn", params, stream=side)
        graph.replay()
        gu.sync()
        p.check(p.out[:-1])
        plain = p.out.clone()
        p.starts[batch // 2] = 0
        p.out.fill_(9.0)
        graph.replay()
        gu.sync()
        assert gu.error_flag(reset=True) == 0x303
        # the sequence in front of the fallen start has no row; the next one has its rows and its own, more than max_new
        a = batch - 2
        assert torch.equal(p.out[:a], plain[:a]) and torch.equal(p.out[a + 4:], plain[a + 4:])
        assert bool((p.out[a + 2:a + 4] == 9.0).all()) and not bool((p.out[a:a + 2] == 9.0).any(2).any())
        p.starts[batch // 2] = batch
        graph.replay()
        gu.sync()
        assert gu.error_flag(reset=True) == 0 and torch.equal(p.out, plain)


def test_scratch_of_many_sequences_is_needed():
    p = Problem([(1, 20)] * 300, 1, 2, 64, 16)
    params = p.params()
    assert params.scratch_bytes >= 4 * 301
    params.scratch_bytes -= 1
    with pytest.raises(Exception, match="scratch"):
        lu.launch("chunk_attn", params)
    params = Problem([(1, 20)] * 256, 1, 2, 64, 16).params()
    assert params.scratch_bytes == 0 and isinstance(params, capi.ChunkAttnParams)
