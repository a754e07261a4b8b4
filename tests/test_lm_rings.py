"""The order in which pb_prefix_attn's warps fill and use their rings, as a model: copies land in any order, and a wait for a barrier's phase sees, as the hardware
does, only the parity of the phase.  No copy may overwrite an entry that is still needed, and nobody may use an entry before its copy has landed."""
import random

import pytest


def shared(n, stages):
    """Two row tiles: tile t's keys and values at 2 t and 2 t + 1 of one ring, a copying warp each, both groups use all."""
    at = {(kind, t): ((2 * t + i) % stages, (2 * t + i) // stages) for t in range(n) for i, kind in enumerate("kv")}
    group = [("k", 0)] + [e for t in range(n) for e in ([("v", t)] + ([("k", t + 1)] if t + 1 < n else []))]
    return at, [[(kind, t) for t in range(n)] for kind in "kv"], [group, group], 2


def apart(n, stages):
    """A lone row tile: halves of every other tile, a ring, a copying warp and a group each."""
    at, orders = {}, []
    for g in range(2):
        tiles = list(range(g, n, 2))
        order = [("k", t, h) for t in tiles[:1] for h in range(2)]
        for i, t in enumerate(tiles):
            for h in range(2):
                order += [("v", t, h)] + [("k", u, h) for u in tiles[i + 1:i + 2]]
        at.update({e: (g * stages + i % stages, i // stages) for i, e in enumerate(order)})
        orders.append(order)
    return at, orders, orders, 1


def one_ring_for_both(n, stages):
    """What must not be: groups that use every other tile of one ring.  A wait may see a phase two behind."""
    order = [("k", 0)] + [e for t in range(n) for e in ([("k", t + 1)] if t + 1 < n else []) + [("v", t)]]
    at = {e: (i % stages, i // stages) for i, e in enumerate(order)}
    return at, [order], [[e for e in order if e[1] % 2 == g] for g in range(2)], 1


def play(at, copies, groups, users, rng):
    """One interleaving; what went wrong, or None."""
    places = 1 + max(place for place, _ in at.values())
    full, empty, left = [0] * places, [0] * places, [users] * places         # phases that have ended; uses until the next ends
    held, flying, done, uses = [None] * places, [], [0] * len(copies), [0, 0]
    used = dict.fromkeys(at, 0)
    ended = lambda phases, parity: phases & 1 != parity                      # what a wait for the phase of this parity sees
    while True:
        moves = [("land", e) for e in flying]
        moves += [("copy", i) for i, order in enumerate(copies) if done[i] < len(order) and ended(empty[at[order[done[i]]][0]], 1 ^ at[order[done[i]]][1] & 1)]
        moves += [("use", g) for g, order in enumerate(groups) if uses[g] < len(order) and ended(full[at[order[uses[g]]][0]], at[order[uses[g]]][1] & 1)]
        if not moves:
            return None if all(d == len(o) for d, o in zip(done + uses, copies + groups)) else "stuck"
        move, which = rng.choices(moves, [rng.random() ** 4 for _ in moves])[0]
        if move == "land":
            flying.remove(which)
            full[at[which][0]] += 1
        elif move == "copy":
            e = copies[which][done[which]]
            done[which] += 1
            place = at[e][0]
            if held[place] is not None and used[held[place]] < users:
                return "overwritten"
            held[place] = e
            flying.append(e)
        else:
            e = groups[which][uses[which]]
            uses[which] += 1
            place = at[e][0]
            if held[place] != e or e in flying:
                return "used too early"
            used[e] += 1
            left[place] -= 1
            if left[place] == 0:
                left[place], empty[place] = users, empty[place] + 1


@pytest.mark.parametrize("scheme,stages", [(shared, 5), (shared, 10), (apart, 6), (apart, 11)])
def test_rings_hold_in_any_order(scheme, stages):
    rng = random.Random(stages)
    for n in [*range(1, 16), 41]:
        for _ in range(60):
            assert play(*scheme(n, stages), rng) is None


def test_one_ring_for_groups_that_take_turns_does_not():
    rng = random.Random(0)
    assert any(play(*one_ring_for_both(41, 6), rng) == "used too early" for _ in range(300))
