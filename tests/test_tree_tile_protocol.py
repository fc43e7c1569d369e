"""Model of the mbarrier protocol of prefix_tile_sm100.cu with its two query tiles' places, run under random schedules: no
deadlock, no ambiguous parity wait, and nothing written to a place that is still read.  A piece is (steps, two), as in
test_prefix_tile_protocol.py; of two pieces of one tile that follow one another, the second one's queries come while the
first one's O goes out through the other place.  A step of V that comes as some boxes is reported when what its keys
without a row leave has been cleared, before the copying warp's next wait or such step.  The K warp tells the others the
pieces through a queue, whose places it uses again without asking: none may be read after that."""
import random

import pytest

from test_barrier_protocols import _run


def _roles(pieces, ring, lose=None, edge=lambda g: False, queue_places=16):
    def mine(n, two, w):
        return [j for j in range(n) if two or j % 2 == w]

    def make(bar, W, A):
        bar("QF", 2)
        bar("QE")
        bar("VE")
        bar("TD", 2)
        bar("step", 1 << 30)              # a point where another role may run
        queue = [None] * queue_places
        for i in range(queue_places):
            bar(("PQ", i))

        def tell(k):
            queue[k % queue_places] = k
            return A(("PQ", k % queue_places))

        def told(k):
            return W(("PQ", k % queue_places), k // queue_places + 1)

        def read(k):
            assert queue[k % queue_places] == k, (k, queue)
        for kv in range(2):
            for s in range(ring[kv]):
                bar(("FULL", kv, s))
                bar(("FREE", kv, s))
        for w in range(2):
            bar(("OF", w))
            for u in range(2):
                for n in ("SF", "PF", "OD"):
                    bar((n, w, u))
        masks = [None] * 8
        place = [[None, None], [None, None]]      # what the halves of the two places hold: ("Q", piece) or ("O", piece, warpgroup)

        def places():
            """Of each piece: the place of its tile (None: both)."""
            at, single, out = 0, False, []
            for _, two in pieces:
                at = 1 - at if not two and single else 0
                single = not two
                out.append(None if two else at)
            return out

        def k_copies():
            g = 0
            for k, (n, _) in enumerate(pieces):
                yield tell(k)
                for _ in range(n):
                    slot = g % ring[0]
                    if g >= ring[0]:
                        yield W(("FREE", 0, slot), g // ring[0])
                    masks[g % 8] = g
                    yield A(("FULL", 0, slot))
                    g += 1
            yield tell(len(pieces))

        def v_copies():
            g, due, edges = 0, None, 0
            for n, _ in pieces:
                for _ in range(n):
                    slot = g % ring[1]
                    is_edge = edge(g)
                    if due is not None and (g >= ring[1] or is_edge):
                        edges += 1
                        yield W("VE", edges)
                        yield A(due)
                        due = None
                    if g >= ring[1]:
                        yield W(("FREE", 1, slot), g // ring[1])
                    if is_edge:
                        yield A("VE")     # (the boxes have landed)
                        due = ("FULL", 1, slot)
                    else:
                        yield A(("FULL", 1, slot))
                    g += 1
            if due is not None:
                yield W("VE", edges + 1)
                yield A(due)

        def s_issuer():
            g, t = 0, [0, 0]
            for k, ((n, two), at) in enumerate(zip(pieces, places())):
                yield told(k)
                read(k)
                yield W("QF", k + 1)
                for j in range(n):
                    yield W(("FULL", 0, g % ring[0]), g // ring[0] + 1)
                    for u, w in ((0, 0), (0, 1), (1, 0), (1, 1)):
                        if j not in mine(n, two, w):
                            continue
                        if t[w]:
                            yield W(("OD", w, u), t[w])
                        assert place[w if two else at] == [("Q", k)] * 2, (k, place)
                        yield A(("SF", w, u))
                        t[w] += u
                    yield A(("FREE", 0, g % ring[0]))
                    if j == n - 1:
                        yield A("QE")
                    g += 1
            yield told(len(pieces))
            read(len(pieces))

        def pv():
            g, t, done = 0, [0, 0], [0, 0]
            for k, (n, two) in enumerate(pieces):
                yield told(k)
                read(k)
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

        out_of = [[False, False], [False, False]]         # an O is on its way out through this half of a place

        def bring(k, at):
            assert not any(out_of[at]), (k, at)
            place[at] = [("Q", k)] * 2

        def softmax(w):
            g, t, at, ahead = 0, 0, 0, False
            yield told(0)
            read(0)
            for k, (n, two) in enumerate(pieces):
                if not ahead:
                    if two or w == 0:
                        bring(k, w if two else at)
                    yield A("QF")
                steps = mine(n, two, w)
                for j in steps:
                    for u in range(2):
                        yield W(("SF", w, u), t + 1)
                        assert masks[(g + j) % 8] == g + j
                        yield A(("PF", w, u))
                    t += 1
                more = k + 1 < len(pieces)
                yield told(k + 1)
                read(k + 1)
                ahead = more and not two and not pieces[k + 1][1]
                if ahead and w == 0:
                    if k and lose != "TD":
                        yield W("TD", k)
                    bring(k + 1, 1 - at)
                if ahead and w == 1 and lose == "QE":
                    yield A("QF")
                yield W("QE", k + 1)
                if ahead and w == 1 and lose != "QE":
                    yield A("QF")
                if steps:
                    yield W(("OD", w, 0), t)
                    yield W(("OD", w, 1), t)
                if ahead and w == 0:
                    yield A("QF")
                if steps:
                    p, halves = (w, (0, 1)) if two else (at, (w,))
                    for h in halves:
                        place[p][h] = ("O", k, w)
                        out_of[p][h] = True
                    yield A("step")
                    for h in halves:
                        assert place[p][h] == ("O", k, w), (k, w, place)
                        out_of[p][h] = False
                    yield A(("OF", w))
                yield A("TD")
                if more and not two and pieces[k + 1][1] and lose != "both":
                    yield W("TD", k + 1)
                at = 1 - at if ahead else 0
                g += n

        return [("K", k_copies()), ("V", v_copies()), ("S", s_issuer()), ("PV", pv()), ("softmax0", softmax(0)), ("softmax1", softmax(1))]
    return make


PIECES = [[(1, False)], [(1, True)], [(7, True), (1, False), (2, False), (5, True)], [(1, False)] * 7, [(2, False), (9, False), (1, True)],
          [(12, True), (3, False)], [(1, False), (1, False), (1, True)] * 3, [(2, False), (1, False), (8, False)] * 2, [(1, True), (2, True), (1, False)] * 2]


@pytest.mark.parametrize("ring", [(2, 3), (4, 4)])
@pytest.mark.parametrize("pieces", PIECES)
def test_protocol(pieces, ring):
    for trial in range(80):
        stuck, hazards = _run(_roles(pieces, ring, edge=lambda g: g % 3 == trial % 5), 1000 + trial)
        assert stuck is None, stuck
        assert not hazards, hazards[:3]


def test_long_runs_of_short_pieces():
    """The queue's places come around several times."""
    rnd = random.Random(9)
    for trial in range(60):
        pieces = [(rnd.randint(1, 2), rnd.random() < trial % 3 / 4) for _ in range(50)]
        for ring in ((2, 3), (4, 4)):
            stuck, hazards = _run(_roles(pieces, ring), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


def test_random_pieces():
    rnd = random.Random(5)
    for trial in range(300):
        pieces = [(rnd.randint(1, 6), rnd.random() < 0.3) for _ in range(rnd.randint(1, 8))]
        for ring in ((2, 3), (4, 4)):
            edges = {g for g in range(80) if rnd.random() < trial % 4 / 3}
            stuck, hazards = _run(_roles(pieces, ring, edge=lambda g: g in edges), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


@pytest.mark.parametrize("lose", ["TD", "QE", "both", "places"])
def test_the_model_sees_a_lost_wait(lose):
    """Queries over the other warpgroup's O; a report of queries ahead of the piece before; both places before they are free; too
    short a queue."""
    def caught(pieces, trial):
        try:
            stuck, hazards = _run(_roles(pieces, (2, 3), lose=lose, queue_places=3 if lose == "places" else 16), trial)
            return stuck or hazards
        except AssertionError:
            return True
    assert any(caught(pieces, trial) for pieces in PIECES for trial in range(200))
