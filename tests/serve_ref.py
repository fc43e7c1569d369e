"""Plain 64-bit forms of the serving operators, loop by loop in numpy, for the tests."""
import numpy as np


def page_plan(lens, new, base, free, free_count, table, page, max_tokens):
    """Returns (lens_out, cu_new, slots, positions, token_seq, counts, table, free) of attn_page_plan_ex."""
    n, max_pages = table.shape
    table, free = table.copy(), free.copy()
    cap = max_pages * page
    lens = [min(max(int(x), 0), cap) for x in lens]
    pages = list(free[:free_count]) + [table[s, j] for s in range(n) if new[s] < 0 for j in range(-(-lens[s] // page))]
    listed = len(pages)
    out_lens, cu, refused, out_of_pages = [], [0], 0, False
    slots, pos, seq = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int32), np.full(max_tokens, -1, np.int32)
    for s in range(n):
        k = max(int(new[s]), 0)
        first = cu[-1]
        cu.append(first + k)
        have = -(-lens[s] // page)
        need = -(-(lens[s] + k) // page) - have
        ok = new[s] >= 0 and (k == 0 or (lens[s] + k <= cap and cu[-1] <= max_tokens))
        if ok and need:
            out_of_pages = out_of_pages or need > len(pages)
            ok = not out_of_pages
        if ok:
            for j in range(need):
                table[s, have + j] = pages.pop()
        elif new[s] >= 0:
            refused += 1
        out_lens.append(0 if new[s] < 0 else lens[s] + k if ok else lens[s])
        for i in range(k):
            if first + i < max_tokens:
                p = lens[s] + i
                seq[first + i], pos[first + i] = s, base[s] + p
                if ok:
                    slots[first + i] = int(table[s, p // page]) * page + p % page
    free[free_count:len(pages)] = pages[free_count:]
    counts = [len(pages), cu[-1], refused, listed - len(pages)]
    return out_lens, cu, slots, pos, seq, counts, table, free


def rope(x, heads, table, positions, rot, interleaved, transpose=False):
    """x (tokens, heads * d) float64; table (max_pos, rot / 2, 2)."""
    n = x.shape[0]
    y = x.reshape(n, heads, -1).astype(np.float64).copy()
    src = y.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = (table[positions, i, k].astype(np.float64)[:, None] for k in (0, 1))
        if transpose:
            s = -s
        y[:, :, a] = src[:, :, a] * c - src[:, :, b] * s
        y[:, :, b] = src[:, :, b] * c + src[:, :, a] * s
    return y.reshape(n, -1)


def rope_table(rot, max_pos, base=10000.0, scaling="plain", factor=1.0, trained=0, fast=0.0, slow=0.0, magnitude=1.0):
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling == "ramp":
        low, high = (rot * np.log(trained / (t * 2 * np.pi)) / (2 * np.log(base)) for t in (fast, slow))
        w = np.clip((np.arange(rot // 2) - low) / (high - low), 0, 1)
        f = f * (1 - w) + f / factor * w
    angle = np.arange(max_pos)[:, None] * f[None, :]
    return np.stack([np.cos(angle), np.sin(angle)], -1) * magnitude


def prefix_decode(q, k_rows, v_rows, heads, kv_heads, scale):
    """q (heads * d) against rows k, v (n, kv_heads * d), all float64.  Returns (out, lse, weight, reach): weight is
    sum_j p_j |v_j| and reach the largest scale * sum_i |q_i k_ji| of each head, for error bounds."""
    d = q.size // heads
    out, lse = np.zeros(heads * d), np.full(heads, -np.inf)
    weight, reach = np.zeros(heads * d), np.zeros(heads)
    for h in range(heads):
        j = h // (heads // kv_heads)
        k, v = k_rows[:, j * d:(j + 1) * d], v_rows[:, j * d:(j + 1) * d]
        if not len(k):
            continue
        qh = q[h * d:(h + 1) * d]
        x = k @ qh * scale
        e = np.exp(x - x.max())
        at = slice(h * d, (h + 1) * d)
        out[at], weight[at] = e @ v / e.sum(), e @ np.abs(v) / e.sum()
        lse[h] = x.max() + np.log(e.sum())
        reach[h] = (np.abs(k) @ np.abs(qh)).max() * scale
    return out, lse, weight, reach
