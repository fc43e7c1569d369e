"""Plain forms of the drafted trees' plan and commit, loop by loop, and random trees, for the tests."""
import numpy as np


def random_tree(r, n, back=8):
    """Parents of n drafts: draft 0 has none, each other one descends from one of the `back` before it, or from none."""
    return [-1] + [int(r.randint(max(-1, i - back), i)) for i in range(1, n)]


def path(parents, at):
    """Ancestors of a draft and itself, from the first."""
    p = []
    while at >= 0:
        p.append(at)
        at = parents[at]
    return p[::-1]


def masks_of(trees, words):
    """(rows, words) uint32 of the trees' drafts, one request after another."""
    m = np.zeros((sum(map(len, trees)), words), np.uint32)
    row = 0
    for t in trees:
        for i in range(len(t)):
            for j in path(t, i):
                m[row + i, j // 32] |= np.uint32(1) << np.uint32(j % 32)
        row += len(t)
    return m


def plan(cu, parents, positions, positions_out, masks):
    """attn_tree_plan_ex on numpy arrays; returns (positions_out, masks) and whether anything was reported."""
    rows, words = masks.shape
    positions_out, masks, code = positions_out.copy(), masks.copy(), 0
    for s in range(len(cu) - 1):
        first = min(max(int(cu[s]), 0), rows)
        n = min(max(int(cu[s + 1]), first), rows) - first
        up = []
        for i in range(n):
            p = int(parents[first + i])
            if i < 32 * words and not -1 <= p < i:
                code, p = code or 0x704, -1
            up.append(p if i < 32 * words else -1)
        if n > 32 * words:
            code = 0x705
        for i in range(n):
            line = path(up, i) if i < 32 * words else []
            positions_out[first + i] = positions[first] + max(len(line) - 1, 0)
            masks[first + i] = 0
            for j in line:
                masks[first + i, j // 32] |= np.uint32(1) << np.uint32(j % 32)
    return positions_out, masks, code


def commit(cu, ctx, lens, leaf, masks, table, page, free, free_count, caches):
    """attn_tree_commit_ex: returns (lens_out, free, counts); moves the rows of `caches`, arrays whose rows follow the
    table."""
    free, out, kept_in_all, none, back = free.copy(), [], 0, 0, []
    for s in range(len(ctx)):
        n = max(int(lens[s]) - int(ctx[s]), 0)
        accepted = []
        if 0 <= leaf[s] < min(n, int(cu[s + 1]) - int(cu[s])):
            accepted = [j for j in range(int(leaf[s]) + 1) if masks is None or masks[cu[s] + leaf[s], j // 32] >> np.uint32(j % 32) & 1]
        row = lambda t: int(table[s, t // page]) * page + t % page  # noqa: E731
        for c in caches:
            for i, j in enumerate(accepted):
                c[row(int(ctx[s]) + i)] = c[row(int(ctx[s]) + j)]
        after = min(int(ctx[s]), int(lens[s])) + len(accepted)
        out.append(after)
        kept_in_all += len(accepted)
        none += not accepted
        back += [table[s, j] for j in range(-(-after // page), -(-int(lens[s]) // page))]
    for i, id in enumerate(back):
        if free_count + i < len(free):
            free[free_count + i] = id
    return out, free, [min(free_count + len(back), len(free)), kept_in_all, none, len(back)]
