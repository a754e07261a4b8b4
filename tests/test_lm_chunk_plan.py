"""How pb_chunk_attn deals its work out, restated step by step: a plan's ranges, walked as its blocks walk them, take every tile of keys of every pair of row tiles exactly once, and the parts that
cut pairs leave are those that the kernel which joins them looks for."""
import pathlib
import random
import re

import pytest

SOURCE = (pathlib.Path(__file__).parents[1] / "paella_b200" / "csrc" / "lm_chunk.cuh").read_text()


def constant(name):
    return int(re.search(rf"\b{name} = (\d+)", SOURCE).group(1))


FEW, BLOCKS, ROUNDS, TWO, ONE, PAIR = (constant(n) for n in ("kFewRows", "kChunkBlocks", "kMaxRounds", "kCostTwo", "kCostOne", "kCostPair"))


def units_of(seqs, group, window, few):
    out = []
    for n, length in seqs:
        rows, first = n * group, length - n
        if rows <= few:
            continue
        for row0 in range(0, rows, 256):
            pos0, pos1 = first + row0 // group, first + (min(row0 + 256, rows) - 1) // group
            end = max(pos1 + 1, 0)
            tile0 = max(pos0 - window + 1, 0) // 128 if window else 0
            out.append(dict(row0=row0, rows=rows, tile0=tile0, tiles=max(-(-end // 128) - tile0, 0)))
    return out


def each_of(u):
    return TWO if u["row0"] + 128 < u["rows"] else ONE


def plan(units, heads, max_ranges):
    before = [0]
    for u in units:
        before.append(before[-1] + PAIR + u["tiles"] * each_of(u))
    total = before[-1] * heads
    rounds = min(max(total // (BLOCKS * 400), 1), max_ranges // BLOCKS)
    n = min(BLOCKS * rounds, max(total // (PAIR + 3 * TWO), 1))
    if len(units) * heads <= BLOCKS and max(b - a for a, b in zip(before, before[1:])) <= PAIR + 8 * TWO:
        return [(r // len(units), r % len(units), 0) for r in range(len(units) * heads)] + [(heads, 0, 0)]
    cuts = []
    for r in range(n):
        w = total * r // n
        head = w // before[-1]
        rest = w - head * before[-1]
        at = max(i for i in range(len(units)) if before[i] <= rest)
        each, tiles = each_of(units[at]), units[at]["tiles"]
        near, step = min(total // n // (8 * each), 2), max(rest - before[at] - PAIR, 0) // each
        if near < step < tiles - near:
            cuts.append((head, at, step))
        elif step > near or 2 * step > tiles:
            cuts.append((head, at + 1, 0) if at + 1 < len(units) else (head + 1, 0, 0))
        else:
            cuts.append((head, at, 0))
    return cuts + [(heads, 0, 0)]


def walk(cuts, units, blocks):
    for block in range(blocks):
        for r in range(block, len(cuts) - 1, blocks):
            (head, unit, step), to = cuts[r], cuts[r + 1]
            while (head, unit) < to[:2] or ((head, unit) == to[:2] and step < to[2]):
                tiles = units[unit]["tiles"]
                end = to[2] if (head, unit) == to[:2] else tiles
                yield r, head, unit, step, end, 2 * r if step > 0 else 2 * r + 1 if end < tiles else -1
                step, unit = 0, unit + 1
                if unit == len(units):
                    unit, head = 0, head + 1


def joined(cuts):
    """(head, unit) -> the parts that are put together"""
    out, n = {}, len(cuts) - 1
    for r in range(1, n):
        same = lambda c: c[:2] == cuts[r][:2]
        if cuts[r][2] > 0 and not (same(cuts[r - 1]) and cuts[r - 1][2] > 0):
            last = r
            while last + 1 < n and same(cuts[last + 1]) and cuts[last + 1][2] > 0:
                last += 1
            assert cuts[r][:2] not in out
            out[cuts[r][:2]] = [2 * (r - 1) + 1 if i == 0 else 2 * (r + i - 1) for i in range(last - r + 2)]
    return out


def some_seqs(rng):
    b = rng.choice([1, 1, 2, 5, 40])
    most, ctx = rng.choice([(3, 10), (30, 500), (700, 700), (3000, 40), (600, 20000), (50, 100000)])
    return [(n, max(0, n + rng.randint(-3, ctx))) for n in (rng.randint(0, most) for _ in range(b))]


@pytest.mark.parametrize("seed", range(60))
def test_every_tile_once_and_every_part_joined(seed):
    rng = random.Random(seed)
    for _ in range(6):
        seqs, group, heads, window = some_seqs(rng), rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 8]), rng.choice([0, 0, 1, 100, 1000])
        units = units_of(seqs, group, window, rng.choice([0, FEW]))
        if not units:
            continue
        cuts = plan(units, heads, BLOCKS * rng.randint(1, ROUNDS))
        assert cuts == sorted(cuts) and cuts[0] == (0, 0, 0)
        seen, parts, whole, slots = {}, {}, set(), set()
        for r, head, unit, step, end, slot in walk(cuts, units, BLOCKS):
            tiles = units[unit]["tiles"]
            assert 0 <= step <= end <= tiles and (step < end or tiles == 0)
            for s in range(step, end):
                assert (head, unit, s) not in seen
                seen[head, unit, s] = True
            if slot < 0:
                whole.add((head, unit))
            else:
                assert slot not in slots and slot < 2 * (len(cuts) - 1)
                slots.add(slot)
                parts.setdefault((head, unit), []).append(slot)
        assert len(seen) == heads * sum(u["tiles"] for u in units)
        assert len(whole) + len(parts) == heads * len(units) and not whole & set(parts)
        assert {k: sorted(v) for k, v in parts.items()} == {k: sorted(v) for k, v in joined(cuts).items()}
