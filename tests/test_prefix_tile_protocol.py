"""Model of the mbarrier protocol of prefix_tile_sm100.cu (the shared-prefix
decode's tensor-core kernel), run under random schedules: no deadlock and no
ambiguous parity wait.  A piece is (steps, two): two says that both warpgroups
take every step, otherwise they take turns.  One warp brings K, one V, each
half (K or V of a step) into a ring of its own; a half that its lanes
copy is reported before the warp's next wait or copy, one that comes as TMA
boxes arrives by itself.  The softmax warpgroups bring Q.  A step's key masks
stay until the softmax has read them."""
import random

import pytest

from test_barrier_protocols import _run


def _roles(pieces, ring, lose=None, boxes=lambda g: False, grows=lambda: False):
    def mine(n, two, w):
        return [j for j in range(n) if two or j % 2 == w]

    def make(bar, W, A):
        bar("QF", 2)
        bar("QE")
        for s in range(ring[0]):
            bar(("FULL", 0, s))
            bar(("FREE", 0, s))
        for s in range(ring[1]):
            bar(("FULL", 1, s))
            bar(("FREE", 1, s))
        masks = [None] * 8                # the step whose key masks are kept
        for w in range(2):
            bar(("OF", w))
            for u in range(2):
                for n in ("SF", "PF", "OD"):
                    bar((n, w, u))

        def copies(kv):
            due, g = None, 0
            for n, two in pieces:
                for j in range(n):
                    slot, whole = g % ring[kv], boxes(2 * g + kv)
                    full = ("FULL", kv, slot)
                    if g >= ring[kv] and lose != "FREE":
                        if due:
                            yield A(due)
                            due = None
                        yield W(("FREE", kv, slot), g // ring[kv])
                    if kv == 0:
                        masks[g % 8] = g
                    if whole:
                        yield A(full)
                    else:
                        if due:
                            yield A(due)
                        due = full
                    g += 1
            if due:
                yield A(due)

        def s_issuer():
            g, t = 0, [0, 0]
            for k, (n, two) in enumerate(pieces):
                yield W("QF", k + 1)
                for j in range(n):
                    yield W(("FULL", 0, g % ring[0]), g // ring[0] + 1)
                    for u, w in ((0, 0), (0, 1), (1, 0), (1, 1)):
                        if j not in mine(n, two, w):
                            continue
                        if t[w] and lose != "S":
                            yield W(("OD", w, u), t[w])
                        yield A(("SF", w, u))
                        t[w] += u
                    yield A(("FREE", 0, g % ring[0]))
                    if j == n - 1:
                        yield A("QE")
                    g += 1

        def pv():
            g, t, done = 0, [0, 0], [0, 0]
            for n, two in pieces:
                for j in range(n):
                    yield W(("FULL", 1, g % ring[1]), g // ring[1] + 1)
                    for u, w in ((0, 0), (0, 1), (1, 0), (1, 1)):
                        if j not in mine(n, two, w):
                            continue
                        if u == 0 and j < (1 if two else 2) and done[w]:
                            yield W(("OF", w), done[w])
                        yield W(("PF", w, u), t[w] + 1)
                        yield A(("OD", w, u))
                        t[w] += u
                    yield A(("FREE", 1, g % ring[1]))
                    g += 1
                done[0] += 1
                done[1] += two or n > 1

        def softmax(w):
            g, t = 0, 0
            for k, (n, two) in enumerate(pieces):
                yield A("QF")
                steps = mine(n, two, w)
                for j in steps:
                    for u in range(2):
                        yield W(("SF", w, u), t + 1)
                        assert masks[(g + j) % 8] == g + j
                        if grows() and (t or u):          # a rescaling waits for the half before
                            yield W(("OD", w, 1 - u), t + u)
                        yield A(("PF", w, u))
                    t += 1
                yield W("QE", k + 1)      # O is turned over where Q was
                if steps:
                    yield W(("OD", w, 0), t)
                    yield W(("OD", w, 1), t)
                    yield A(("OF", w))
                g += n

        return [("K", copies(0)), ("V", copies(1)), ("S", s_issuer()), ("PV", pv()), ("softmax0", softmax(0)), ("softmax1", softmax(1))]
    return make


PIECES = [[(1, False)], [(1, True)], [(7, True), (1, False), (2, False), (5, True)], [(1, False)] * 6, [(2, False), (9, False), (1, True)],
          [(12, True), (3, False)]]


@pytest.mark.parametrize("ring", [(2, 3), (4, 4)])
@pytest.mark.parametrize("pieces", PIECES)
def test_protocol(pieces, ring):
    for trial in range(60):
        stuck, hazards = _run(_roles(pieces, ring), 1000 + trial)
        assert stuck is None, stuck
        assert not hazards, hazards[:3]


def test_random_pieces():
    rnd = random.Random(3)
    for trial in range(150):
        pieces = [(rnd.randint(1, 9), rnd.random() < 0.5) for _ in range(rnd.randint(1, 6))]
        for ring in ((2, 3), (4, 4)):
            lanes = {g for g in range(120) if rnd.random() < trial % 4 / 3}      # steps copied by lanes
            stuck, hazards = _run(_roles(pieces, ring, boxes=lambda g: g not in lanes,
                                          grows=lambda: rnd.random() < 0.3), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


@pytest.mark.parametrize("lose", ["S", "FREE"])
def test_the_model_sees_a_lost_wait(lose):
    """S before the product that reads its last P, a slot copied over before its use: phases run ahead."""
    def caught(trial):
        try:
            return _run(_roles(PIECES[2], (2, 3), lose=lose), trial)[1]
        except AssertionError:            # a step's masks were overwritten
            return True
    assert any(caught(trial) for trial in range(40))
