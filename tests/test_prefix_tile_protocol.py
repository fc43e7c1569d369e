"""Model of the mbarrier protocol of prefix_tile_sm100.cu (the shared-prefix
decode's tensor-core kernel), run under random schedules: no deadlock and no
ambiguous parity wait.  A piece is (steps, two): two says that both warpgroups
take every step, otherwise they take turns.  The copying warps report a half
(K or V of a step) when LAG more are on their way, and everything that is due
before they wait for the query buffer; a step that comes as TMA boxes arrives
by itself, and what is due is reported before its waits for a slot and after
its issue.  A step's key masks stay until the softmax has read them."""
import random

import pytest

from test_barrier_protocols import _run


def _roles(pieces, slots, lag=2, lose=None, boxes=lambda g: False, grows=lambda: False):
    def mine(n, two, w):
        return [j for j in range(n) if two or j % 2 == w]

    def make(bar, W, A):
        bar("QF")
        bar("QE")
        for s in range(slots):
            bar(("FULL", s))
            bar(("FREE", s))
        masks = [None] * 8                # the step whose key masks are kept
        for w in range(2):
            bar(("OF", w))
            for u in range(2):
                for n in ("SF", "PF", "OD"):
                    bar((n, w, u))

        def copies():
            due, g = [], 0
            for k, (n, two) in enumerate(pieces):
                if lose != "flush":
                    while due:
                        yield A(due.pop(0))
                if k:
                    yield W("QE", k)
                due.append("QF")
                for j in range(n):
                    whole = boxes(g)
                    for half in (2 * g, 2 * g + 1):
                        if half >= slots:
                            while whole and due and lose != "flush":
                                yield A(due.pop(0))
                            yield W(("FREE", half % slots), half // slots)
                        if half % 2 == 0:
                            masks[g % 8] = g
                        full = ("FULL", half % slots)
                        if whole:
                            yield A(full)
                            while half % 2 and due:
                                yield A(due.pop(0))
                            continue
                        if len(due) == lag:
                            yield A(due.pop(0))
                        due.append(full)
                    g += 1
            while due:
                yield A(due.pop(0))

        def s_issuer():
            g, t = 0, [0, 0]
            for k, (n, two) in enumerate(pieces):
                yield W("QF", k + 1)
                for j in range(n):
                    yield W(("FULL", 2 * g % slots), 2 * g // slots + 1)
                    for u, w in ((0, 0), (0, 1), (1, 0), (1, 1)):
                        if j not in mine(n, two, w):
                            continue
                        if t[w] and lose != "S":
                            yield W(("OD", w, u), t[w])
                        yield A(("SF", w, u))
                        t[w] += u
                    yield A(("FREE", 2 * g % slots))
                    if j == n - 1:
                        yield A("QE")
                    g += 1

        def pv():
            g, t, done = 0, [0, 0], [0, 0]
            for n, two in pieces:
                for j in range(n):
                    half = 2 * g + 1
                    yield W(("FULL", half % slots), half // slots + 1)
                    for u, w in ((0, 0), (0, 1), (1, 0), (1, 1)):
                        if j not in mine(n, two, w):
                            continue
                        if u == 0 and j < (1 if two else 2) and done[w]:
                            yield W(("OF", w), done[w])
                        yield W(("PF", w, u), t[w] + 1)
                        yield A(("OD", w, u))
                        t[w] += u
                    yield A(("FREE", half % slots))
                    g += 1
                done[0] += 1
                done[1] += two or n > 1

        def softmax(w):
            g, t = 0, 0
            for n, two in pieces:
                steps = mine(n, two, w)
                for j in steps:
                    for u in range(2):
                        yield W(("SF", w, u), t + 1)
                        assert masks[(g + j) % 8] == g + j
                        if grows() and (t or u):          # a rescaling waits for the half before
                            yield W(("OD", w, 1 - u), t + u)
                        yield A(("PF", w, u))
                    t += 1
                if steps:
                    yield W(("OD", w, 0), t)
                    yield W(("OD", w, 1), t)
                    yield A(("OF", w))
                g += n

        return [("copies", copies()), ("S", s_issuer()), ("PV", pv()), ("softmax0", softmax(0)), ("softmax1", softmax(1))]
    return make


PIECES = [[(1, False)], [(1, True)], [(7, True), (1, False), (2, False), (5, True)], [(1, False)] * 6, [(2, False), (9, False), (1, True)],
          [(12, True), (3, False)]]


@pytest.mark.parametrize("slots", [5, 8])
@pytest.mark.parametrize("pieces", PIECES)
def test_protocol(pieces, slots):
    for trial in range(60):
        stuck, hazards = _run(_roles(pieces, slots), 1000 + trial)
        assert stuck is None, stuck
        assert not hazards, hazards[:3]


def test_random_pieces():
    rnd = random.Random(3)
    for trial in range(150):
        pieces = [(rnd.randint(1, 9), rnd.random() < 0.5) for _ in range(rnd.randint(1, 6))]
        for slots in (5, 8):
            lanes = {g for g in range(60) if rnd.random() < trial % 4 / 3}      # steps copied by lanes
            stuck, hazards = _run(_roles(pieces, slots, boxes=lambda g: g not in lanes,
                                          grows=lambda: rnd.random() < 0.3), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


def test_the_model_sees_a_lost_wait_and_a_lost_report():
    """Without its wait, S runs phases ahead; without the reports before the query buffer's wait, the copies stop."""
    assert any(_run(_roles(PIECES[2], 5, lose="S"), t)[1] for t in range(40))
    assert any(_run(_roles(PIECES[2], 5, lose="flush"), t)[0] for t in range(40))
