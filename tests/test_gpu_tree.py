"""Drafted token trees over a paged cache on the GPU: plan, attention and commit, against the plain forms of tree_ref.py
and 64-bit attention (serve_ref.py).

Tolerances: whole numbers and moved rows are equal.  Attention: as in test_gpu_serve.py, whose kernels take the prefixes
and contexts; the drafted rows add fp32 sums and exponentials of the same kind: a score is off by at most
delta = 2^-21 (1 + scale sum|q k|), the output by 4 delta sum p|v| and for bf16 2^-8 sum p|v| more, a probability under
2^-126 may count as 0; lse by delta + 2^-22 |lse|."""
import ctypes

import numpy as np
import pytest

import serve_ref as R
import synth
import tree_ref as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A(cuda):
    import attn_b200
    return attn_b200


def dev(x, dtype=None):
    import torch
    x = np.ascontiguousarray(x)
    t = torch.from_numpy(x.view(np.int32) if x.dtype == np.uint32 else x).cuda()
    return t if dtype is None else t.to(dtype)


def device_error(A):
    code = ctypes.c_int()
    A.check(A.lib.attn_device_error(0, ctypes.byref(code)))
    return code.value


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def run_plan(A, cu, parents, positions, words, in_place=False):
    rows = len(parents)
    pos = dev(positions)
    out = pos if in_place else dev(np.full(rows, -7, np.int32))
    masks = dev(np.full((rows, words), -9, np.int32))
    A.tree_plan_t(dev(cu), dev(parents), pos, out, masks)
    return out.cpu().numpy(), masks.cpu().numpy().view(np.uint32)


def check_plan(A, cu, parents, positions, words, code=0):
    rows = len(parents)
    device_error(A)
    for in_place in (False, True):
        before = positions if in_place else np.full(rows, -7, np.int32)
        want_p, want_m, want_code = T.plan(cu, parents, positions, before, np.full((rows, words), -9, np.int32).view(np.uint32))
        got_p, got_m = run_plan(A, cu, parents, positions, words, in_place)
        np.testing.assert_array_equal(got_p, want_p)
        np.testing.assert_array_equal(got_m, want_m)
        assert device_error(A) == want_code == code


@pytest.mark.parametrize("words", [1, 2, 32])
@pytest.mark.parametrize("sizes", [[1], [32, 0, 5, 31], [0, 0], [33, 64, 1, 0, 7], [1024, 100, 3], [2] * 300])
def test_plan(A, sizes, words):
    """Requests of no drafts, words' edges, chains and random trees, rows behind the last draft, rows before the first."""
    if max(sizes) > 32 * words:
        sizes = [min(s, 32 * words) for s in sizes]
    r = np.random.RandomState(len(sizes) + words)
    for lead in (0, 3):
        trees = [T.random_tree(r, n) if i % 2 else list(range(-1, n - 1)) for i, n in enumerate(sizes) if n]
        parents = np.array([9] * lead + [p for t in trees for p in t] + [77] * 5, np.int32)
        cu = np.concatenate([[lead], lead + np.cumsum(sizes)]).astype(np.int32)
        check_plan(A, cu, parents, r.randint(0, 5000, len(parents)).astype(np.int32), words)


def test_plan_bad_parents_and_too_many_drafts(A):
    pos = np.arange(10, 50, dtype=np.int32)
    parents = np.array([-1, 0, 2, 1, -2, 9, 3, 5] + [-1] * 32, np.int32)
    check_plan(A, np.array([0, 4, 8], np.int32), parents, pos, 1, code=0x704)
    check_plan(A, np.array([0, 40], np.int32), np.arange(-1, 39, dtype=np.int32), pos, 1, code=0x705)
    check_plan(A, np.array([0, 6, 2 ** 31 - 1, 2 ** 31 - 1], np.int32), np.tile(np.array([-1, 0], np.int32), 10), pos[:20], 1)   # past the rows there are


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class TreeCase:
    """Random trees over a cache whose unused rows are NaN and inf (INT8: NaN scales) and whose unused table entries lie
    outside the cache.  refused: requests whose drafts have no rows.  masks: "tree"; "chain" (none given); "any" (random
    bits, rows without any among them)."""

    def __init__(self, A, seed, kind, d, heads, kv_heads, page, drafts, ctx, group_sizes=(), prefix_lens=(), refused=(), masks="tree",
                 spare=3, q_std=1.0, extra_stride=0, words=None):
        import torch
        r = np.random.RandomState(seed)
        self.A, self.kind, self.d, self.heads, self.kv_heads, self.page = A, kind, d, heads, kv_heads, page
        self.n, self.ctx = len(drafts), np.array(ctx, np.int32)
        assert len(ctx) == self.n and sum(group_sizes) <= self.n
        self.cu = np.concatenate([[0], np.cumsum(drafts)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + spare
        self.lens = np.array([c + (0 if s in refused else k) for s, (c, k) in enumerate(zip(ctx, drafts))], np.int32)
        nodes = max(list(drafts) + [0])
        words = words or max(1, (nodes + 31) // 32)
        self.trees = [T.random_tree(r, k) for k in drafts]
        self.bits = np.zeros((self.rows, nodes), bool)
        for s in range(self.n):
            for i in range(drafts[s]):
                row = self.bits[self.cu[s] + i]
                if masks == "tree":
                    row[T.path(self.trees[s], i)] = True
                elif masks == "chain":
                    row[:i + 1] = True
                else:
                    row[:] = r.rand(nodes) < r.choice([0, 0.1, 0.6, 1.0])
        if masks == "any":
            self.bits[self.cu[:-1][np.array(drafts) > 0]] = False
        packed = np.zeros((self.rows, 32 * words), bool)
        packed[:, :nodes] = self.bits
        self.masks = None if masks == "chain" else (packed.reshape(self.rows, words, 32) * (np.uint64(1) << np.arange(32, dtype=np.uint64))).sum(-1).astype(np.uint32)
        self.begin = np.concatenate([[0], np.cumsum(group_sizes)]).astype(np.int32)
        self.plens = np.array(prefix_lens, np.int32)
        held = list(prefix_lens) + [int(x) for x in self.lens]
        mp, mo = (max([1] + [-(-int(x) // page) for x in v]) for v in (prefix_lens, self.lens))
        n_pages = sum(-(-int(x) // page) for x in held) + 4
        ids = r.permutation(n_pages)
        self.ptable, self.table = np.full((max(1, len(group_sizes)), mp), 2 ** 30, np.int32), np.full((self.n, mo), -5, np.int32)
        at, used = 0, np.zeros(n_pages * page, bool)
        for table, ls in ((self.ptable, prefix_lens), (self.table, self.lens)):
            for i, x in enumerate(ls):
                for j in range(-(-int(x) // page)):
                    table[i, j] = ids[at]
                    used[ids[at] * page:ids[at] * page + min(page, int(x) - j * page)] = True
                    at += 1
        rows, w = n_pages * page, kv_heads * d
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.float32}[kind]
        self.q = dev(synth.normal(seed + 1, (self.rows, heads * d), 0, q_std), dt)
        self.ks = self.vs = None
        if kind == "int8":
            self.kc, self.vc = (torch.zeros((rows, w + extra_stride), dtype=torch.int8, device="cuda")[:, :w] for _ in range(2))
            codes = [r.randint(-127, 128, (rows, w)).astype(np.int8) for _ in range(2)]
            scales = [(0.005 + 0.02 * r.rand(rows, kv_heads)).astype(np.float32) for _ in range(2)]
            self.k64, self.v64 = (c.astype(np.float64) * np.repeat(s.astype(np.float64), d, 1) for c, s in zip(codes, scales))
            for s in scales:
                s[~used] = np.nan
            self.kc.copy_(dev(codes[0]))
            self.vc.copy_(dev(codes[1]))
            self.ks, self.vs = dev(scales[0]), dev(scales[1])
        else:
            self.kc, self.vc = (torch.full((rows, w + extra_stride), float("nan"), dtype=dt, device="cuda")[:, :w] for _ in range(2))
            for i, c in enumerate((self.kc, self.vc)):
                x = dev(synth.normal(seed + 5 + i, (rows, w)), dt)
                x[~dev(used)] = float("nan") if i else float("inf")
                c.copy_(x)
            self.k64, self.v64 = (c.float().cpu().numpy().astype(np.float64) for c in (self.kc, self.vc))
        self.cache = A.PageCache.of(self.kc, self.vc, self.ks, self.vs)
        self.shape = A.TreeShape(self.n, self.rows, len(group_sizes), heads, kv_heads, d, A.BF16 if kind == "bf16" else A.F32, page, mp, mo,
                                 max([0] + list(prefix_lens)), int(max([0] + list(self.lens))), nodes, 0 if masks == "chain" else words, 0, 0, 0.0)

    def arrays(self):
        groups = dict(group_begin=dev(self.begin), prefix_table=dev(self.ptable), prefix_lens=dev(self.plens)) if self.shape.n_groups else {}
        return (dev(self.cu), dev(self.ctx), dev(self.lens), None if self.masks is None else dev(self.masks), dev(self.table)), groups

    def workspace(self):
        import torch
        return torch.full((self.A.tree_decode_workspace_bytes(self.shape, self.cache),), 0xff, dtype=torch.uint8, device="cuda")

    def run(self, q=None, out=None, workspace="own", lse=True):
        import torch
        out = torch.full_like(self.q, 7.0) if out is None else out
        ls = torch.full((self.rows, self.heads), 7.0, device="cuda") if lse else None
        args, groups = self.arrays()
        self.A.tree_decode_t(self.shape, self.cache, self.q if q is None else q, *args, out, lse=ls, **groups,
                             workspace=self.workspace() if workspace == "own" else workspace)
        return out, ls

    def slot(self, s, t):
        return int(self.table[s, t // self.page]) * self.page + t % self.page

    def rows_of(self, s, i):
        """Cache rows that draft i of request s attends to."""
        rows = []
        for g in range(len(self.plens)):
            if self.begin[g] <= s < self.begin[g + 1]:
                rows += [int(self.ptable[g, t // self.page]) * self.page + t % self.page for t in range(self.plens[g])]
        seen = [t for t in range(self.ctx[s], self.lens[s]) if self.bits[self.cu[s] + i, t - self.ctx[s]]]
        return rows + [self.slot(s, t) for t in list(range(self.ctx[s])) + seen]

    def check(self, out, lse, only=None, absent=()):
        scale = 1.0 / np.sqrt(self.d)
        q64 = self.q.float().cpu().numpy().astype(np.float64)
        out, lse = out.float().cpu().numpy().astype(np.float64), None if lse is None else lse.cpu().numpy().astype(np.float64)
        absent = set(absent)
        for s in range(self.n):
            for i in range(self.cu[s + 1] - self.cu[s]):
                x = self.cu[s] + i
                if only is not None and x not in only:
                    continue
                rows = [y for y in self.rows_of(s, i) if y not in absent]
                want, wl, weight, reach = R.prefix_decode(q64[x], self.k64[rows], self.v64[rows], self.heads, self.kv_heads, scale)
                delta = 2.0 ** -21 * (1 + reach)
                tol = 4 * np.repeat(delta, self.d) * weight + (2.0 ** -8 * weight if self.kind == "bf16" else 0)
                tol = tol + len(rows) * 2.0 ** -126 * (np.abs(self.v64[rows]).max() if rows else 0)
                assert (np.abs(out[x] - want) <= tol).all(), (s, i, np.nanmax(np.abs(out[x] - want) / np.maximum(tol, 1e-300)))
                if lse is not None:
                    finite = np.isfinite(wl)
                    assert np.array_equal(lse[x][~finite], wl[~finite])
                    assert (np.abs(lse[x][finite] - wl[finite]) <= (delta + 2.0 ** -22 * np.abs(wl))[finite]).all(), (s, i)
        if only is None:
            assert (out[self.cu[-1]:] == 7).all() and (lse is None or (lse[self.cu[-1]:] == 7).all())


KINDS = ["f32", "bf16", "int8"]


@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,heads,kv_heads,page", [(32, 4, 4, 16), (64, 6, 2, 8), (96, 3, 3, 32), (128, 8, 1, 64), (64, 2, 2, 1), (128, 4, 4, 1024)])
def test_tree_small(A, kind, d, heads, kv_heads, page, masks):
    """Contexts of 0 and 1 rows, tiles' edges, requests without drafts, refused ones, empty prefixes, none, rows to spare."""
    c = TreeCase(A, d + heads, kind, d, heads, kv_heads, page, [1, 5, 0, 33, 2, 7, 1, 64, 3], [0, 1, 9, 77, 0, 128, 129, 33, 64], [3, 2, 2], [129, 0, 1],
                 refused=[4, 5], masks=masks)
    device_error(A)
    out, lse = c.run()
    c.check(out, lse)
    assert device_error(A) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("drafts,ratio", [(1, 1), (4, 1), (9, 1), (16, 2), (30, 4), (70, 8)])
def test_tree_query_rows(A, kind, drafts, ratio):
    """Each way through the query rows of a line, and lines of several blocks, with and without a prefix."""
    for groups in ((), (2, 1)):
        c = TreeCase(A, drafts + ratio, kind, 64, 2 * ratio, 2, 16, [drafts] * 4, [300, 5, 0, 129], groups, (200, 65)[:len(groups)], spare=0)
        c.check(*c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("kv_heads", [1, 5, 13])
def test_tree_blocks(A, kind, d, kv_heads):
    """Blocks of each size at each head size, full and in part, with key heads that divide a CTA's warps and that do not."""
    for drafts, groups in (([3, 4, 2, 4], ()), ([7, 5, 8, 8], ()), ([7, 5, 8, 8], (2, 1)), ([16, 9, 13, 16], ()), ([16, 30, 32, 25], (1, 2)),
                           ([64, 50, 33, 60], ())):
        c = TreeCase(A, d + len(groups), kind, d, kv_heads, kv_heads, 16, drafts, [300, 5, 31, 129], groups, (200, 65)[:len(groups)], spare=0)
        c.check(*c.run())


@pytest.mark.parametrize("d,heads,kv_heads,page,drafts,ctx,groups,prefix", [
    (128, 8, 2, 64, [40, 33, 1, 64], [700, 256, 128, 1], (), ()),
    (64, 16, 4, 16, [32] * 6, [129, 127, 400, 0, 3, 1000], (4, 2), (1000, 300)),
    (128, 4, 4, 4, [128, 60], [300, 257], (2,), (500,)),
    (64, 8, 1, 128, [100, 20, 16], [2000, 5, 50], (3,), (4097,)),
    (64, 2, 2, 16, [5] * 40, [30] * 20 + [1] * 20, (40,), (300,)),
])
def test_tree_tiles(A, d, heads, kv_heads, page, drafts, ctx, groups, prefix):
    """bf16 lines of many query rows: up to 128 of a block, more, pages below a box, prefixes beside contexts."""
    c = TreeCase(A, 5, "bf16", d, heads, kv_heads, page, drafts, ctx, groups, prefix)
    c.check(*c.run())


@pytest.mark.parametrize("d,heads,kv_heads,drafts,groups", [
    (32, 4, 4, 6, ()), (32, 8, 2, 16, (2, 1)), (32, 8, 1, 30, ()), (64, 4, 4, 7, ()), (64, 4, 2, 8, (3,)), (64, 8, 2, 8, ()), (64, 8, 2, 32, ()),
    (64, 16, 2, 40, (2, 1)), (96, 3, 3, 8, ()), (96, 6, 2, 16, (1, 2)), (128, 4, 4, 8, ()), (128, 4, 2, 8, ()), (128, 16, 2, 25, ()), (128, 8, 2, 40, (4,))])
def test_tree_bf16_error_is_the_outputs_rounding(A, d, heads, kv_heads, drafts, groups):
    """The same precision on every path: rounding the output (2^-8 of it), a probability's second part (what the first drops,
    2^-8 of it, rounded in its turn: 2^-16 of sum p|v|), and the fp32 errors as above."""
    c = TreeCase(A, d + drafts, "bf16", d, heads, kv_heads, 16, [drafts] * 4, [900, 33, 0, 400], groups, (700, 65)[:len(groups)])
    out, _ = c.run()
    out, q64 = out.float().cpu().numpy().astype(np.float64), c.q.float().cpu().numpy().astype(np.float64)
    for s in range(c.n):
        for i in range(0, drafts, 5):
            x, rows = c.cu[s] + i, c.rows_of(s, i)
            want, _, weight, reach = R.prefix_decode(q64[x], c.k64[rows], c.v64[rows], heads, kv_heads, 1.0 / np.sqrt(d))
            own = (2.0 ** -16 + 4 * 2.0 ** -21 * (1 + np.repeat(reach, d))) * weight
            tol = 2.0 ** -8 * (np.abs(want) + own) + own
            assert (np.abs(out[x] - want) <= tol).all(), (s, i, (np.abs(out[x] - want) / tol).max())


@pytest.mark.parametrize("kind", KINDS)
def test_tree_long(A, kind):
    """A long context beside short ones, drafts up to the limit of 1024 in a chain, and a tree of 1000."""
    c = TreeCase(A, 8, kind, 64, 2, 2, 64, [3, 1, 2], [20011, 3, 700])
    c.check(*c.run())
    for masks, n in (("chain", 1024), ("tree", 1000)):
        c = TreeCase(A, 9, kind, 32, 2, 1, 64, [n, 2], [40, 0], masks=masks)
        c.check(*c.run(), only=list(range(0, n + 2, 97)) + [n - 1, n, n + 1])


@pytest.mark.parametrize("kind", KINDS)
def test_tree_none(A, kind):
    """No rows anywhere: zeros and -inf; no requests, no token rows: nothing is written."""
    c = TreeCase(A, 1, kind, 64, 4, 2, 16, [2, 3], [0, 0], refused=[0, 1])
    out, lse = c.run()
    assert (out[:5] == 0).all() and (lse[:5] == float("-inf")).all() and (out[5:] == 7).all()
    for change in (dict(n_seq=0), dict(n_rows=0)):
        c = TreeCase(A, 1, kind, 64, 4, 2, 16, [2, 3], [4, 0])
        for k, v in change.items():
            setattr(c.shape, k, v)
        out, lse = c.run(workspace=None)
        assert (out == 7).all() and (lse == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,ratio,ctx", [(6, 1, 0), (6, 1, 40), (40, 4, 200)])
def test_tree_hidden_rows_may_hold_anything(A, kind, n, ratio, ctx, bad):
    """A draft whose key and value are no numbers reaches itself and its descendants, and no other row."""
    import torch
    if kind == "int8" and bad != bad:
        pass
    elif kind == "int8":
        pytest.skip("an INT8 cache's scales: NaN alone")
    c = TreeCase(A, 21, kind, 64, 2 * ratio, 2, 16, [n, 3], [ctx, 7])
    want, wl = c.run()
    at = c.slot(0, ctx + 2)
    for x in ((c.ks, c.vs) if kind == "int8" else (c.kc, c.vc)):
        x[at] = bad
    sees = c.bits[:c.rows, 2].copy()
    sees[n:] = False
    assert sees.any() and not sees[:n].all()
    out, lse = c.run()
    rows = dev(np.flatnonzero(~sees))
    assert torch.equal(out[rows], want[rows]) and torch.equal(lse[rows], wl[rows])
    if bad != bad:
        assert out[dev(np.flatnonzero(sees))].isnan().all()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_bad_pages_and_lengths(A, kind):
    """Pages outside the cache: their rows count as absent; lengths out of bounds are clamped; both are reported."""
    c = TreeCase(A, 3, kind, 64, 4, 2, 8, [6, 40, 5], [30, 100, 9], [2], [50])
    absent = [c.slot(1, t) for t in range(16, 24)] + [c.slot(2, t) for t in range(8, 14)] + \
        [int(c.ptable[0, 1]) * 8 + t for t in range(8)]
    keep = [c.rows_of(s, i) for s in range(3) for i in range(c.cu[s + 1] - c.cu[s])]
    good = [c.table.copy(), c.ptable.copy()]
    c.table[1, 2], c.table[2, 1], c.ptable[0, 1] = 2 ** 30, -1, len(c.k64)
    device_error(A)
    out, lse = c.run()
    assert device_error(A) == 0x702
    c.table, c.ptable = good
    assert keep
    c.check(out, lse, absent=absent)
    c.shape.max_len -= 1                          # the second request's last draft is past the bound
    c.lens[2] = -4
    out, lse = c.run()
    assert device_error(A) == 0x703
    c.lens[1] -= 1
    c.lens[2] = c.ctx[2]                          # no drafted rows
    c.check(out, lse)
    c.shape.max_len += 1
    c.shape.max_nodes = 39                        # more drafted rows than the bound
    c.lens[1] += 1
    out, lse = c.run()
    assert device_error(A) == 0x703
    c.lens[1] -= 1
    c.check(out, lse)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_strides_and_repeats(A, kind):
    """q and out inside wider tensors, cache rows apart, no lse; the same bits on every run."""
    import torch
    c = TreeCase(A, 31, kind, 64, 8, 4, 16, [12, 20, 3], [90, 500, 0], [1, 2], [70, 300], extra_stride=64)
    out, lse = c.run()
    c.check(out, lse)
    width = c.heads * c.d
    wide = torch.full((c.rows, 3 * width), 7.0, dtype=c.q.dtype, device="cuda")
    q = torch.cat([c.q, c.q, c.q], 1)[:, width:2 * width]
    c.shape.q_row_stride = c.shape.out_row_stride = 3 * width
    again, _ = c.run(q=q, out=wide[:, width:2 * width], lse=False)
    assert torch.equal(again, out) and (wide[:, :width] == 7).all() and (wide[:, 2 * width:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_many_requests(A, kind):
    """More lines than running sums are kept for, most of them short, with prefixes of single requests among them."""
    r = np.random.RandomState(2)
    n = 1300
    drafts, ctx = r.randint(0, 4, n), r.randint(0, 30, n)
    c = TreeCase(A, 12, kind, 32, 2, 1, 8, list(drafts), list(ctx), [1] * 5 + [40] + [0, 3], [5, 9, 0, 33, 2, 100, 7, 8])
    c.check(*c.run())


def test_tree_cache_past_32_bits(A):
    """Rows whose elements lie past 2^31 (and bytes past 2^32)."""
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough free memory")
    d, kv, page = 128, 8, 64
    rows = (2 ** 31 // (kv * d) // page + 40) * page
    small = TreeCase(A, 77, "bf16", d, 32, kv, page, [20, 3], [300, 70], [1], [130])
    want, wl = small.run()
    far = rows // page - small.kc.shape[0] // page
    big = [torch.zeros((rows, kv * d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b, s in zip(big, (small.kc, small.vc)):
        b[far * page:] = s
    small.table[small.table >= 0] += far
    small.ptable[small.ptable < 2 ** 30] += far
    small.cache = A.PageCache.of(*big)
    out, lse = small.run()
    assert torch.equal(out, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_captured_and_on_two_streams(A, kind):
    """A captured call replayed while another runs beside it, each with its workspace: the bits of plain calls."""
    import torch
    a, b = (TreeCase(A, s, kind, 64, 8, 2, 16, [10, 33, 4], [200, 1000, 0], [2], [90]) for s in (51, 52))
    want = [x.run() for x in (a, b)]
    args, groups = a.arrays()
    out, lse, work = torch.full_like(a.q, 7.0), torch.full((a.rows, a.heads), 7.0, device="cuda"), a.workspace()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.tree_decode_t(a.shape, a.cache, a.q, *args, out, lse=lse, **groups, workspace=work)
    b_args, b_groups = b.arrays()
    b_out, b_lse, b_work = torch.full_like(b.q, 7.0), torch.full((b.rows, b.heads), 7.0, device="cuda"), b.workspace()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        g.replay()
        with torch.cuda.stream(side):
            A.tree_decode_t(b.shape, b.cache, b.q, *b_args, b_out, lse=b_lse, **b_groups, workspace=b_work)
    torch.cuda.synchronize()
    for got, w in (((out, lse), want[0]), ((b_out, b_lse), want[1])):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_tree_of_one_draft_is_the_prefix_decode(A):
    """One draft per request, which sees itself: the decode of one token over the same rows."""
    import torch
    for kind in KINDS:
        c = TreeCase(A, 61, kind, 64, 4, 2, 16, [1] * 7, [0, 1, 15, 16, 100, 333, 64], [4, 2], [77, 130], spare=0)
        out, lse = c.run()
        shape = A.PrefixShape(c.n, 2, 4, 2, 64, c.shape.dtype, 16, c.shape.max_prefix_pages, c.shape.max_pages, c.shape.max_prefix_len,
                              c.shape.max_len, 0, 0, 0.0)
        ref, rl = torch.empty_like(out), torch.empty_like(lse)
        A.prefix_decode_t(shape, c.cache, c.q, dev(c.begin), dev(c.ptable), dev(c.plens), dev(c.table), dev(c.lens), ref, lse=rl)
        c.check(ref, rl)
        c.check(out, lse)


# ---------------------------------------------------------------------------
# commit
# ---------------------------------------------------------------------------
class CommitCase:
    def __init__(self, A, seed, kind, layers, kv_heads, d, page, drafts, ctx, refused=(), chain=False, slack=4, leaves=None, extra_stride=0, words=None):
        import torch
        r = np.random.RandomState(seed)
        self.A, self.page, self.kv_heads, self.d = A, page, kv_heads, d
        n = self.n = len(drafts)
        self.cu = np.concatenate([[0], np.cumsum(drafts)]).astype(np.int32)
        self.ctx = np.array(ctx, np.int32)
        self.lens = np.array([c + (0 if s in refused else k) for s, (c, k) in enumerate(zip(ctx, drafts))], np.int32)
        trees = [T.random_tree(r, k) if k else [] for k in drafts]
        self.words = words or max(1, (max(list(drafts) + [1]) + 31) // 32)
        self.masks = None if chain else T.masks_of(trees, self.words)
        self.leaf = np.array([r.randint(-1, max(k, 1)) for k in drafts] if leaves is None else leaves, np.int32)
        mo = max([1] + [-(-int(x) // page) for x in self.lens]) + 1
        ids = r.permutation(n * mo + slack).astype(np.int32)
        self.table = ids[:n * mo].reshape(n, mo).copy()
        self.free = np.full(n * mo + slack, -1, np.int32)
        self.free[:slack] = ids[n * mo:]
        self.count = slack
        rows = (n * mo + slack) * page
        self.caches, self.kv = [], []
        for i in range(layers):
            ts = []
            for j in range(2):
                x = synth.normal(seed + 10 * i + j, (rows, kv_heads * d))
                t = torch.zeros((rows, kv_heads * d + extra_stride), dtype={"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}[kind], device="cuda")
                t = t[:, :kv_heads * d]
                t.copy_(dev(np.clip(x * 40, -127, 127).astype(np.int8) if kind == "int8" else x))
                ts.append(t)
            if kind == "int8":
                ts += [dev(r.rand(rows, kv_heads).astype(np.float32)) for _ in range(2)]
            self.caches.append(ts)
            self.kv.append(A.PageCache.of(*ts))

    def run(self, free_entries=None):
        import torch
        A = self.A
        n_pages = len(self.free) if free_entries is None else free_entries
        shape = A.PageShape(self.n, self.page, self.table.shape[1], int(self.cu[-1]), n_pages, 0)
        free = dev(self.free)
        lens_out, counts = torch.full((self.n,), -9, dtype=torch.int32, device="cuda"), torch.full((4,), -9, dtype=torch.int32, device="cuda")
        A.tree_commit_t(shape, A.cache_array(self.kv), self.kv_heads, self.d, dev(self.cu), dev(self.ctx), dev(self.lens), dev(self.leaf),
                        None if self.masks is None else dev(self.masks), dev(self.table), free, dev(np.array([self.count], np.int32)), lens_out, counts)
        return lens_out.cpu().numpy(), free.cpu().numpy(), counts.cpu().numpy()

    def check(self, free_entries=None, skip=()):
        before = [t.float().cpu().numpy() for c in self.caches for t in c]
        want = T.commit(self.cu, self.ctx, self.lens, self.leaf, self.masks, self.table, self.page, self.free[:free_entries], self.count, before)
        got = self.run(free_entries)
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1][:free_entries], want[1])
        if free_entries is not None:
            np.testing.assert_array_equal(got[1][free_entries:], self.free[free_entries:])
        np.testing.assert_array_equal(got[2], want[2])
        for t, w in zip((t for c in self.caches for t in c), before):
            np.testing.assert_array_equal(t.float().cpu().numpy(), w)


@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("kind,layers,kv_heads,d,page", [("f32", 1, 1, 32, 16), ("bf16", 3, 8, 128, 64), ("int8", 2, 3, 96, 8), ("f32", 2, 16, 128, 4),
                                                        ("int8", 1, 1, 32, 1), ("bf16", 1, 5, 64, 1024)])
def test_commit(A, kind, layers, kv_heads, d, page, chain):
    c = CommitCase(A, d + page, kind, layers, kv_heads, d, page, [1, 5, 0, 33, 2, 7, 1, 40, 3], [0, 1, 9, 77, 0, 128, 129, 33, 64], refused=[4, 5], chain=chain,
                   extra_stride=16)
    c.check()


def test_commit_many_requests_and_a_long_path(A):
    r = np.random.RandomState(4)
    c = CommitCase(A, 6, "bf16", 1, 1, 32, 2, [int(x) for x in r.randint(0, 6, 700)], [int(x) for x in r.randint(0, 9, 700)])
    c.check()
    c = CommitCase(A, 7, "f32", 2, 1, 32, 16, [1024, 1000, 3], [5, 0, 40], leaves=[1023, 998, 2], words=32)
    c.check()


def test_commit_with_a_short_free_list_and_without_caches(A):
    c = CommitCase(A, 9, "f32", 0, 1, 32, 2, [9, 12, 30], [3, 3, 3], leaves=[-1, 2, 4])
    c.check()
    c = CommitCase(A, 9, "f32", 1, 1, 32, 2, [9, 12, 30], [3, 3, 3], leaves=[-1, 2, 4])
    c.check(free_entries=c.count + 6)


def test_commit_leaves_and_pages_that_are_none(A):
    c = CommitCase(A, 13, "f32", 1, 2, 32, 4, [6, 6, 6, 6], [5, 6, 7, 8], leaves=[6, -2, 5, 3], refused=[1])
    device_error(A)
    before = c.leaf.copy()
    want_leaf = np.array([-1, -1, 5, 3], np.int32)
    kept = [t.float().cpu().numpy() for t in c.caches[0]]
    c.leaf = want_leaf
    want = T.commit(c.cu, c.ctx, c.lens, c.leaf, c.masks, c.table, c.page, c.free, c.count, kept)
    c.leaf = before
    got = c.run()
    assert device_error(A) == 0x706
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    for t, w in zip(c.caches[0], kept):
        np.testing.assert_array_equal(t.float().cpu().numpy(), w)
    c.leaf = np.array([5, 1, -1, -1], np.int32)   # the second request was refused: nothing to keep, and no error
    c.masks = None
    c.check()
    assert device_error(A) == 0
    c.masks, c.leaf = T.masks_of([[-1, -1, 0, 1, 3, -1]] * 4, 1), np.array([4, -1, -1, -1], np.int32)
    c.table[0, 2] = 2 ** 20                       # drafts 3 and 4 lie there, and go to places 1 and 2
    kept = [t.float().cpu().numpy() for t in c.caches[0]]
    s0 = int(c.table[0, 1]) * 4
    for k in kept:
        k[s0 + 1] = k[s0 + 2]                     # draft 1 (row 6) to row 5; the others stay
    c.run()
    assert device_error(A) == 0x702
    for t, w in zip(c.caches[0], kept):
        np.testing.assert_array_equal(t.float().cpu().numpy(), w)


def commit_of_rows(A, c, rows):
    """The case's commit with `rows` rows of masks."""
    import torch
    shape = A.PageShape(c.n, c.page, c.table.shape[1], rows, len(c.free), 0)
    free = dev(c.free)
    lens_out, counts = (torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (c.n, 4))
    A.tree_commit_t(shape, A.cache_array(c.kv), c.kv_heads, c.d, dev(c.cu), dev(c.ctx), dev(c.lens), dev(c.leaf),
                    None if c.masks is None else dev(c.masks[:rows]), dev(c.table), free, dev(np.array([c.count], np.int32)), lens_out, counts)
    return lens_out.cpu().numpy(), free.cpu().numpy(), counts.cpu().numpy()


@pytest.mark.parametrize("kind", ["f32", "int8"])
def test_commit_with_fewer_mask_rows_than_drafts(A, kind):
    """cu_rows past the rows of masks: the drafts that have a row are drafts, as the plan and the decode have them, and the
    others are none."""
    for cut, leaves, want_leaf in ((2, [3, 4, 2], [3, 4, 2]), (2, [3, 4, 4], [3, 4, -1]), (5, [3, 5, 0], [3, 5, -1]), (8, [5, 2, 1], [5, 2, -1])):
        c = CommitCase(A, 17 + cut, kind, 2, 2, 32, 4, [6, 6, 5], [5, 6, 7], leaves=leaves)
        rows = int(c.cu[-1]) - cut
        before = [t.float().cpu().numpy() for x in c.caches for t in x]
        want = T.commit(c.cu, c.ctx, c.lens, np.array(want_leaf), c.masks, c.table, c.page, c.free, c.count, before)
        device_error(A)
        got = commit_of_rows(A, c, rows)
        assert device_error(A) == (0x706 if want_leaf != leaves else 0)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)
        for t, w in zip((t for x in c.caches for t in x), before):
            np.testing.assert_array_equal(t.float().cpu().numpy(), w)


def test_commit_of_chains_needs_no_rows_of_masks(A):
    c = CommitCase(A, 19, "f32", 1, 2, 32, 4, [6, 3, 40], [5, 6, 7], leaves=[4, -1, 39], chain=True)
    device_error(A)
    before = [t.float().cpu().numpy() for t in c.caches[0]]
    want = T.commit(c.cu, c.ctx, c.lens, c.leaf, None, c.table, c.page, c.free, c.count, before)
    got = commit_of_rows(A, c, 0)
    assert device_error(A) == 0
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    for t, w in zip(c.caches[0], before):
        np.testing.assert_array_equal(t.float().cpu().numpy(), w)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_drafts_example(A, cache):
    """The example's loop: page plan, tree plan, projection, normed append, tree decode and commit, several steps; fp32
    arithmetic, the repository's 1e-5."""
    import os
    import runpy
    from conftest import ROOT
    m = runpy.run_path(os.path.join(ROOT, "examples", "serve_drafts.py"))
    assert m["main"](requests=5, prompt=130, steps=6, nodes=40 if cache == "f32" else 9, cache=cache) < 1e-5


def test_a_captured_step(A):
    """A whole step, from the page plan to the commit, captured and replayed on other lengths, drafts and leaves: what plain
    calls give."""
    import torch
    r = np.random.RandomState(3)
    n, nodes, page, heads, d, most = 7, 8, 4, 4, 64, 60
    rows, cols = n * nodes, -(-(most + nodes) // page)
    ids = r.permutation(n * cols).astype(np.int32)
    free = np.full(n * cols, -1, np.int32)
    q, k, v = (dev(synth.normal(50 + i, (rows, heads * d))) for i in range(3))
    caches = [[dev(synth.normal(60 + 2 * i + j, (n * cols * page, heads * d))) for j in range(2)] for i in range(2)]
    kv = [A.PageCache.of(*c) for c in caches]
    weight = dev((1 + 0.1 * synth.normal(70, (d,))).astype(np.float32))
    norm = A.HeadNorm.of(weight, weight, 1e-6)
    table = dev(R.rope_table(d, most + 2 * nodes).astype(np.float32))
    pages = A.PageShape(n, page, cols, rows, n * cols, 0)
    out = A.page_outputs(pages)
    z = dict(dtype=torch.int32, device="cuda")
    state = dict(lens=torch.zeros(n, **z), new=torch.zeros(n, **z), free=dev(free), count=torch.zeros(1, **z), table=torch.zeros((n, cols), **z),
                 parents=torch.zeros(rows, **z), leaf=torch.zeros(n, **z), masks=torch.zeros((rows, 1), **z), lens_out=torch.zeros(n, **z),
                 counts=torch.zeros(4, **z), att=torch.zeros((rows, heads * d), device="cuda"), turned=torch.zeros((rows, heads * d), device="cuda"))
    shape = A.RopeShape(rows, 0, heads, heads, d, d, 0, most + 2 * nodes, 0, 0, 0, 0, 0)
    tree = A.TreeShape(n, rows, 0, heads, heads, d, A.F32, page, 0, cols, 0, cols * page, nodes, 1, 0, 0, 0.0)
    work = torch.empty(A.tree_decode_workspace_bytes(tree, kv[0]), dtype=torch.uint8, device="cuda")
    array = A.cache_array(kv)

    def step():
        s = state
        A.page_plan_t(pages, s["lens"], s["new"], s["free"], s["count"], s["table"], out)
        A.tree_plan_t(out["cu_new"], s["parents"], out["positions"], out["positions"], s["masks"])
        for c in kv:
            A.norm_rope_append_t(shape, norm, c, table, out["positions"], out["slot_map"], q, k, v, s["turned"])
            A.tree_decode_t(tree, c, s["turned"], out["cu_new"], s["lens"], out["lens"], s["masks"], s["table"], s["att"], workspace=work)
        A.tree_commit_t(pages, array, heads, d, out["cu_new"], s["lens"], out["lens"], s["leaf"], s["masks"], s["table"], s["free"], out["counts"][:1],
                        s["lens_out"], s["counts"])

    def load(seed):
        x = np.random.RandomState(seed)
        lens = x.randint(0, most - nodes, n).astype(np.int32)
        new = x.randint(0, nodes + 1, n).astype(np.int32)
        new[x.randint(0, n)] = -1
        held = -(-lens // page)
        tab, at = np.full((n, cols), -1, np.int32), 0
        for s in range(n):
            tab[s, :held[s]] = ids[at:at + held[s]]
            at += held[s]
        left = np.full(n * cols, -1, np.int32)
        left[:n * cols - at] = ids[at:]
        parents = np.zeros(rows, np.int32)
        first = 0
        for m in np.maximum(new, 0):
            if m:
                parents[first:first + m] = T.random_tree(x, int(m))
            first += m
        leaf = np.array([x.randint(-1, max(int(m), 1)) for m in new], np.int32)
        for name, value in (("lens", lens), ("new", new), ("free", left), ("count", np.array([n * cols - at], np.int32)), ("table", tab), ("parents", parents),
                            ("leaf", leaf)):
            state[name].copy_(dev(value))
        for i, c in enumerate(caches):
            for j in range(2):
                c[j].copy_(dev(synth.normal(60 + 2 * i + j, (n * cols * page, heads * d))))
        for name in ("masks", "lens_out", "counts", "att"):
            state[name].zero_()

    def results():
        torch.cuda.synchronize()
        return [t.clone() for t in list(state.values()) + list(out.values()) + [c for pair in caches for c in pair]]

    load(1)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    device_error(A)
    for seed in (2, 3, 4):
        load(seed)
        step()
        want = results()
        load(seed)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(results(), want))
        assert int(state["counts"][1]) > 0
    assert device_error(A) == 0
