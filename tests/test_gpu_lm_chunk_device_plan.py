"""The plan that pb_chunk_attn's first kernel leaves in the scratch memory, read back: units, ranges and cuts are those that `test_lm_chunk_plan.py` restates, every tile of keys of every pair of row
tiles is taken once, and the parts of cut pairs are those that are joined."""
import pytest
import torch

from tests import gpu_util as gu
from tests import lm_util as lu
from tests.test_gpu_lm_chunk import Problem
from tests.test_lm_chunk_plan import BLOCKS, FEW, ONE, PAIR, ROUNDS, TWO, joined, plan, units_of, walk

pytestmark = pytest.mark.gpu


def up(n, to=128):
    return -(-n // to) * to


def device_plan(p):
    """(sequences of so many rows are own_kernel's, units, cuts, the most ranges) of a problem's launch."""
    b, group, d = len(p.seqs), p.group, 64 if p.d <= 64 else 128
    rows = min(p.most_new, p.tokens) * group
    ranges = BLOCKS * min(max((b * p.most_len * p.hkv * p.d * 4) >> 26, 1), ROUNDS)
    units = min(p.tokens * group // 256 + b, b * -(-rows // 256))
    at, where = 0, {}
    for name, size in (("counted", 4 * (b + 1)), ("counts", 12), ("cuts", 48 * (ranges + 2)), ("units", 32 * units), ("before", 8 * (units + 1)), ("part_ml", 2 * ranges * 256 * 8), ("part_o", 2 * ranges * 256 * d * 4)):
        where[name] = at
        at += up(size)
    params = p.params()
    assert params.scratch_bytes == at                                # the layout is as above
    lu.launch("chunk_attn", params)
    gu.sync()
    words = lambda name, n: p.scratch[where[name]:where[name] + 4 * n].cpu().view(torch.int32)
    assert words("counted", b + 1).tolist() == p.first
    n_units, n_ranges, few = words("counts", 3).tolist()
    assert n_units <= units and n_ranges <= ranges
    return few, words("units", 8 * n_units).view(-1, 8).tolist(), words("cuts", 12 * (n_ranges + 1)).view(-1, 12).tolist(), ranges


def some(g, batch, most, ctx):
    n = torch.randint(0, most + 1, (batch,), generator=g)
    return [(int(a), max(0, int(a) + int(c))) for a, c in zip(n, torch.randint(-2, ctx + 1, (batch,), generator=g))]


CASES = {"one prompt": ([(3000, 3000)], 8, 4, 0), "a whole pair a block": ([(512, 512)], 8, 4, 0), "behind a long cache": ([(700, 20000)], 2, 5, 0), "one token far behind": ([(1, 300000)], 8, 4, 0), "a window": ([(2500, 9000)], 4, 2, 700),
         "few and many rows": ([(1, 900), (30, 700), (3, 20), (0, 9), (400, 1700), (5, 3)] * 3, 2, 4, 0), "under a window": ([(1, 900), (30, 700), (300, 290), (900, 2700)] * 8, 3, 5, 256),
         "nothing": ([(0, 40), (0, 0)], 2, 4, 0), "rows that see nothing": ([(40, 3), (600, 5)], 2, 8, 0), "more sequences than threads": (some(torch.Generator().manual_seed(1), 1500, 40, 300), 1, 4, 0),
         "more units than fit shared memory": (some(torch.Generator().manual_seed(2), 2500, 130, 200), 1, 5, 0), "costs beyond 32-bit quotients": ([(16384, 147456)], 8, 4, 0)}


@pytest.mark.parametrize("case", CASES)
def test_plan(case):
    seqs, heads, group, window = CASES[case]
    p = Problem(seqs, heads, group, 64, 64, window=window, most_new=None if any(n for n, _ in seqs) else 50)
    if case == "nothing":
        p.tokens = 50                                                # rows that belong to no sequence
        p.q, p.out = (torch.zeros(51, heads * group, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    few, units, cuts, most = device_plan(p)
    assert few in (0, FEW // 2 if group <= FEW // 2 else FEW)
    if case == "one token far behind":
        assert few == 0
    want = units_of(seqs, group, window, few)
    where = [(i, r) for i, (n, _) in enumerate(seqs) if n * group > few for r in range(0, n * group, 256)]
    assert len(units) == len(want)
    for u, w, (i, row0) in zip(units, want, where):
        n, length = seqs[i]
        last = length - n + (min(row0 + 256, n * group) - 1) // group
        assert u == [i, p.first[i], n * group, length - n, row0, w["tile0"], w["tiles"], max(last + 1, 0)]
    found = [(c[1], c[0], c[2]) for c in cuts]
    if not want:
        assert found == [(heads, 0, 0)]
        return
    assert found == plan(want, heads, most)
    assert all(c[4:] == units[c[0]] for c in cuts[:-1])               # a copy of the unit that a range begins in
    spans, parts, slots = {}, {}, set()
    for _, head, unit, step, end, slot in walk(found, want, BLOCKS):
        spans.setdefault((head, unit), []).append((step, end))
        if slot >= 0:
            assert slot not in slots
            slots.add(slot)
            parts.setdefault((head, unit), []).append(slot)
    assert len(spans) == heads * len(want)
    for (_, unit), s in spans.items():
        s.sort()
        assert s[0][0] == 0 and s[-1][1] == want[unit]["tiles"] and all(a[1] == b[0] for a, b in zip(s, s[1:]))
    assert {k: sorted(v) for k, v in parts.items()} == {k: sorted(v) for k, v in joined(found).items()}
    total = heads * sum(PAIR + u["tiles"] * (TWO if u["row0"] + 128 < u["rows"] else ONE) for u in want)
    assert (total >= 2 ** 32 // (BLOCKS * ROUNDS)) == (case == "costs beyond 32-bit quotients")
    assert (len(units) > 2048) == (case == "more units than fit shared memory")


@pytest.mark.parametrize("seqs", [[(1, 300)], [(1, 1)], [(1, 0)], [(2, 700)], [(1, 500), (1, 40)], [(3, 90), (1, 2000)], [(40, 700)], [(1, 300)] * 9], ids=range(8))
@pytest.mark.parametrize("most_len", [70000, 131072, 1 << 20])
@pytest.mark.parametrize("window", [0, 128])
def test_bounds_far_above_the_lengths(seqs, most_len, window):
    """A step that was captured for the longest context, run behind short ones."""
    p = Problem(seqs, 8, 4, 128, 64, window=window, most_new=max(n for n, _ in seqs), most_len=most_len)
    p.check(p.run())
    assert gu.error_flag() == 0
