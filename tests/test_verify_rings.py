"""The rings of operand tiles that the Q8_0 decode of rf_tree_tc.cu fills: no slot is written while a product may
still read it, whatever the timing.

Every order in which the parties can take their steps is gone through, for each shape of the kernel.  The parties are
those of the kernel: two sets of decoding warps that take the tiles in turn, the raw tiles they wait for, and the two
groups of products, which give a tile back at once or when their products on it are over.  An mbarrier is what the
hardware has: a count of completed phases, of which a waiting thread is told the parity.  The kernel's rule for the
wait on the other set is read from its source.
"""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ramforge_b200", "csrc",
                      "rf_tree_tc.cu")
TILES, NRAW, SETS, LEAD = 7, 4, 2, 2


def slots(D, split):
    """NSLOT of one row tile over a Q8_0 cache."""
    tile = 128 * D * 2
    return min(6, (224 * 1024 - tile * (2 if split else 1) - NRAW * 128 * D) // tile)


def waits_for_other_set(nslot):
    m = re.search(r"if constexpr \(([^)]*)\) ok = __all_sync\(~0u, ok && wait\(&B\.full\[ring\.s\], ring\.phase \^ 1\)\);",
                  open(SOURCE).read())
    if not m:
        return False
    return bool(eval(m.group(1).replace("S::", "").replace("&&", "and"), {"SETS": SETS, "NSLOT": nslot}))


def program(g, nt):
    """What product group g does with its tiles, in order: (wait for tile e and keep it), (give tile e back at once),
    (give it back when the products issued so far are over)."""
    ops, at = [], 0

    def take(mine):
        nonlocal at
        ops.append(("take", at))
        if not mine:
            ops.append(("give", at))
        at += 1
        return at - 1

    for i in range(min(LEAD, nt)):
        e = take(i % 2 == g)
        if i % 2 == g:
            ops.append(("commit", e))
    for i in range(nt):
        more, mine = i + 2 < nt, i % 2 == g
        v = take(mine)
        k = take(mine) if more else None
        if mine:
            ops.append(("commit", v))
            if more:
                ops.append(("commit", k))
    return ops


def explore(nslot, extra):
    """All reachable states from the start; returns the first breach (tile written over, or nobody can go on)."""
    n = 2 * TILES
    progs = [program(g, TILES) for g in range(2)]
    # state: tiles that each set has finished, whether it is writing, each group's place, its commits under way
    start = ((0, 0), (False, False), (0, 0), ((), ()), (0,) * n)
    seen, todo = {start}, [start]

    def passed(phases, parity):
        return phases % 2 != parity

    while todo:
        done, busy, pc, pend, freed = state = todo.pop()
        finished = {e for s in range(SETS) for e in range(s, s + 2 * done[s], 2)}
        full = [sum(e % nslot == s for e in finished) for s in range(nslot)]
        free = [sum(f for e, f in enumerate(freed) if e % nslot == s) // 2 for s in range(nslot)]
        nxt = []
        for s in range(SETS):
            e = s + 2 * done[s]
            if e >= n:
                continue
            if busy[s]:
                nxt.append((tuple(d + (i == s) for i, d in enumerate(done)),
                            tuple(b and i != s for i, b in enumerate(busy)), pc, pend, freed))
                continue
            if any(x not in finished for x in range(e - NRAW + 1)):  # raw tiles come in order, a slot after its last use
                continue
            use = e // nslot
            before = (use & 1) ^ 1
            if extra and not passed(full[e % nslot], before):
                continue
            if not passed(free[e % nslot], before):
                continue
            if use and freed[e - nslot] < 2:
                return "tile %d is written over tile %d" % (e, e - nslot)
            nxt.append((done, tuple(b or i == s for i, b in enumerate(busy)), pc, pend, freed))
        for g in range(2):
            if pend[g]:
                e = pend[g][0]
                nxt.append((done, busy, pc, tuple(p[1:] if i == g else p for i, p in enumerate(pend)),
                            tuple(f + (i == e) for i, f in enumerate(freed))))
            if pc[g] == len(progs[g]):
                continue
            op, e = progs[g][pc[g]]
            step = tuple(p + (i == g) for i, p in enumerate(pc))
            if op == "take":
                if passed(full[e % nslot], (e // nslot) & 1):
                    nxt.append((done, busy, step, pend, freed))
            elif op == "give":
                nxt.append((done, busy, step, pend, tuple(f + (i == e) for i, f in enumerate(freed))))
            else:
                nxt.append((done, busy, step, tuple(p + (e,) if i == g else p for i, p in enumerate(pend)), freed))
        if not nxt and sum(freed) < 2 * n:
            return "nobody can go on: %r" % (state,)
        for x in nxt:
            if x not in seen:
                seen.add(x)
                todo.append(x)
    return None


def test_slot_counts():
    assert [slots(128, True), slots(128, False), slots(64, True), slots(64, False)] == [3, 4, 6, 6]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("split", [False, True])
def test_no_tile_is_written_over(D, split):
    nslot = slots(D, split)
    assert explore(nslot, waits_for_other_set(nslot)) is None


def test_three_slots_need_the_wait():
    assert explore(3, False) is not None and explore(4, False) is None
