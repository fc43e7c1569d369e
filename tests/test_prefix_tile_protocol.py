"""Model of the mbarrier protocol of prefix_tile_sm100.cu (the shared-prefix
decode's tensor-core kernel), run under random schedules: no deadlock and no
ambiguous parity wait.  A piece is (steps, two): two says that both warpgroups
take every step, otherwise they take turns.  The copying warps report a half
(K or V of a step) when LAG more are on their way, and everything that is due
before they wait for the query buffer."""
import random

import pytest

from test_barrier_protocols import _run


def _roles(pieces, stages, over, lag=2, lose=None):
    def mine(n, two, w):
        return [j for j in range(n) if two or j % 2 == w]

    def make(bar, W, A):
        bar("QF")
        bar("QE")
        for s in range(stages):
            bar(("KF", s))
            bar(("VF", s))
            bar(("KVE", s), 2)
        for w in range(2):
            for n in ("SF", "SE", "PF", "OD", "OF"):
                bar((n, w))

        def copies():
            due, g = [], 0
            for k, (n, two) in enumerate(pieces):
                if lose != "flush":
                    while due:
                        yield A(due.pop(0))
                if k:
                    yield W("QE", k)
                halves = ["QF"]
                for j in range(n):
                    halves += [("wait", g + j), ("KF", (g + j) % stages), ("VF", (g + j) % stages)]
                for h in halves:
                    if h[0] == "wait":
                        if h[1] >= stages:
                            yield W(("KVE", h[1] % stages), h[1] // stages)
                        continue
                    if len(due) == lag:
                        yield A(due.pop(0))
                    due.append(h)
                g += n
            while due:
                yield A(due.pop(0))

        def s_issuer():
            g, t = 0, [0, 0]
            for k, (n, two) in enumerate(pieces):
                yield W("QF", k + 1)
                for j in range(n):
                    yield W(("KF", g % stages), g // stages + 1)
                    for w in range(2):
                        if j not in mine(n, two, w):
                            continue
                        if t[w] and lose != "S":
                            yield W(("OD" if over else "SE", w), t[w])
                        yield A(("SF", w))
                        t[w] += 1
                    yield A(("KVE", g % stages))
                    if j == n - 1:
                        yield A("QE")
                    g += 1

        def pv():
            g, t, done = 0, [0, 0], [0, 0]
            for n, two in pieces:
                for j in range(n):
                    yield W(("VF", g % stages), g // stages + 1)
                    for w in range(2):
                        if j not in mine(n, two, w):
                            continue
                        if j < (1 if two else 2) and done[w]:
                            yield W(("OF", w), done[w])
                        yield W(("PF", w), t[w] + 1)
                        yield A(("OD", w))
                        t[w] += 1
                    yield A(("KVE", g % stages))
                    g += 1
                done[0] += 1
                done[1] += two or n > 1

        def softmax(w):
            g, t = 0, 0
            for n, two in pieces:
                steps = mine(n, two, w)
                for j in steps:
                    yield W(("SF", w), t + 1)
                    yield W(("KF", (g + j) % stages), (g + j) // stages + 1)
                    if not over:
                        yield A(("SE", w))
                    if t:
                        yield W(("OD", w), t)
                    yield A(("PF", w))
                    t += 1
                if steps:
                    yield W(("OD", w), t)
                    yield A(("OF", w))
                g += n

        return [("copies", copies()), ("S", s_issuer()), ("PV", pv()), ("softmax0", softmax(0)), ("softmax1", softmax(1))]
    return make


PIECES = [[(1, False)], [(1, True)], [(7, True), (1, False), (2, False), (5, True)], [(1, False)] * 6, [(2, False), (9, False), (1, True)],
          [(12, True), (3, False)]]


@pytest.mark.parametrize("stages,over", [(2, True), (4, False)])
@pytest.mark.parametrize("pieces", PIECES)
def test_protocol(pieces, stages, over):
    for trial in range(60):
        stuck, hazards = _run(_roles(pieces, stages, over), 1000 + trial)
        assert stuck is None, stuck
        assert not hazards, hazards[:3]


def test_random_pieces():
    rnd = random.Random(3)
    for trial in range(150):
        pieces = [(rnd.randint(1, 9), rnd.random() < 0.5) for _ in range(rnd.randint(1, 6))]
        for stages, over in ((2, True), (4, False)):
            stuck, hazards = _run(_roles(pieces, stages, over), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


def test_the_model_sees_a_lost_wait_and_a_lost_report():
    """Without its wait, S runs phases ahead; without the reports before the query buffer's wait, the copies stop."""
    assert any(_run(_roles(PIECES[2], 2, True, lose="S"), t)[1] for t in range(40))
    assert any(_run(_roles(PIECES[2], 2, True, lose="flush"), t)[0] for t in range(40))
