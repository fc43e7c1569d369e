"""The mbarrier protocol of prefix_tile_sm100.cu (test_tree_tile_protocol.py) where no boxes are used (pages of fewer than 8
rows): the lanes copy each half (K or V of a step) and report it before their next wait for a slot or their next copy, and
at the end.  And, with boxes and without, softmax warpgroups that rescale O now and then, for which they wait for the
product of the half before.  The roles are that file's, with those reports and waits put in."""
import random

import pytest

from test_barrier_protocols import _run
from test_tree_tile_protocol import PIECES, _roles


def _with(pieces, ring, lanes=False, grows=lambda: False, edge=lambda g: False, lose=None):
    def make(bar, W, A):
        def copies(gen):
            due = None
            for op in gen:
                name = op[1].name[0]
                if due and (name == "FREE" or name == "FULL"):
                    yield due
                    due = None
                if name == "FULL":
                    due = op
                elif name != "FREE" or lose != "FREE":
                    yield op
            if due and lose != "last":
                yield due

        def rescaling(gen, w):
            n = 0                         # halves so far
            for op in gen:
                if op[0] == "arr" and op[1].name[0] == "PF":
                    if n and grows():
                        yield W(("OD", w, (n - 1) % 2), (n + 1) // 2)
                    n += 1
                yield op

        def without(gen, name):
            return (op for op in gen if not (op[0] == "wait" and op[1].name[0] == name))

        roles = []
        for name, gen in _roles(pieces, ring, edge=edge)(bar, W, A):
            if lanes and name in ("K", "V"):
                gen = copies(gen)
            if name.startswith("softmax"):
                gen = rescaling(gen, int(name[-1]))
            if name == "S" and lose == "S":
                gen = without(gen, "OD")
            roles.append((name, gen))
        return roles
    return make


@pytest.mark.parametrize("ring", [(2, 3), (4, 4)])
@pytest.mark.parametrize("pieces", PIECES)
def test_copies_by_lanes(pieces, ring):
    rnd = random.Random(2)
    for trial in range(80):
        stuck, hazards = _run(_with(pieces, ring, lanes=True, grows=lambda: rnd.random() < trial % 3 / 2), 3000 + trial)
        assert stuck is None, stuck
        assert not hazards, hazards[:3]


@pytest.mark.parametrize("lanes", [False, True])
def test_random_pieces(lanes):
    rnd = random.Random(7)
    for trial in range(200):
        pieces = [(rnd.randint(1, 6), rnd.random() < 0.3) for _ in range(rnd.randint(1, 8))]
        for ring in ((2, 3), (4, 4)):
            edges = set() if lanes else {g for g in range(80) if rnd.random() < trial % 4 / 3}
            stuck, hazards = _run(_with(pieces, ring, lanes, lambda: rnd.random() < 0.4, lambda g: g in edges), trial)
            assert stuck is None and not hazards, (pieces, stuck, hazards[:3])


@pytest.mark.parametrize("lose", ["FREE", "last", "S"])
def test_the_model_sees_what_is_lost(lose):
    """A slot copied over before its use; the last half never reported; S before the product that reads its last P."""
    def caught(pieces, trial):
        try:
            stuck, hazards = _run(_with(pieces, (2, 3), lanes=True, lose=lose), trial)
            return stuck or hazards
        except AssertionError:            # masks or queries were overwritten
            return True
    assert any(caught(pieces, trial) for pieces in PIECES for trial in range(100))
