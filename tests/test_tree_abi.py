"""Refusals of the drafted trees' calls and of their torch forms, the plain forms of their tests, and where the pieces of
the tree decode lie (prefix.cuh, compiled for the host)."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import attn_b200 as A
import tree_ref as T
from conftest import PKG, ROOT
from test_serve_abi import Given, calls, each_refused, ints, kv, refused  # noqa: F401

P, Q = 1 << 20, 1 << 21


def test_plan_refusals():
    def call(n_seq=4, n_rows=32, words=2, cu=P, parents=P, positions=P, out=Q, masks=Q):
        return A.lib.attn_tree_plan_ex(n_seq, n_rows, words, cu, parents, positions, out, masks, None)

    for bad, status in ((dict(n_seq=-1), A.ERR_INVALID), (dict(n_seq=65536), A.ERR_INVALID), (dict(n_rows=-1), A.ERR_INVALID),
                        (dict(words=0), A.ERR_UNSUPPORTED), (dict(words=33), A.ERR_UNSUPPORTED), (dict(cu=None), A.ERR_INVALID),
                        (dict(parents=None), A.ERR_INVALID), (dict(positions=None), A.ERR_INVALID), (dict(out=None), A.ERR_INVALID),
                        (dict(masks=None), A.ERR_INVALID), (dict(cu=P + 2), A.ERR_INVALID), (dict(masks=Q + 1), A.ERR_INVALID),
                        (dict(out=P + 4), A.ERR_INVALID)):
        assert call(**bad) == status, bad
    assert "overlap" in A.last_error()
    assert call(n_seq=0) == A.OK


def test_decode_refusals():
    ok = dict(n_seq=4, n_rows=12, n_groups=1, heads=4, kv_heads=2, head_dim=64, dtype=A.F32, page_size=16, max_prefix_pages=4, max_pages=4,
              max_prefix_len=64, max_len=64, max_nodes=40, mask_words=2, q_row_stride=0, out_row_stride=0, scale=0.0)

    def call(shape, cache, q=P, cu=P, ctx=P, lens=P, masks=P, begin=P, ptable=P, plens=P, table=P, out=Q, lse=None, ws=P, ws_bytes=1 << 40):
        return A.lib.attn_tree_decode_ex(shape, cache, q, cu, ctx, lens, masks, begin, ptable, plens, table, out, lse, ws, ws_bytes, None)

    assert call(None, kv()) == A.ERR_INVALID
    for bad, status in ((dict(n_seq=-1), A.ERR_INVALID), (dict(n_seq=65536), A.ERR_INVALID), (dict(n_rows=-1), A.ERR_INVALID),
                        (dict(n_rows=1 << 23), A.ERR_INVALID), (dict(heads=3), A.ERR_INVALID), (dict(head_dim=80), A.ERR_UNSUPPORTED),
                        (dict(dtype=A.BF16), A.ERR_UNSUPPORTED), (dict(page_size=20), A.ERR_UNSUPPORTED), (dict(max_len=65), A.ERR_INVALID),
                        (dict(max_prefix_len=65), A.ERR_INVALID), (dict(max_nodes=-1), A.ERR_UNSUPPORTED), (dict(max_nodes=1025), A.ERR_UNSUPPORTED),
                        (dict(max_nodes=65), A.ERR_INVALID), (dict(mask_words=33), A.ERR_INVALID), (dict(mask_words=-1), A.ERR_INVALID),
                        (dict(q_row_stride=255), A.ERR_INVALID), (dict(out_row_stride=258), A.ERR_INVALID), (dict(scale=-1.0), A.ERR_INVALID),
                        (dict(scale=float("nan")), A.ERR_INVALID), (dict(n_groups=-1), A.ERR_INVALID)):
        shape = A.TreeShape(**{**ok, **bad})
        assert call(shape, kv()) == status, bad
        assert A.tree_decode_workspace_bytes(shape, kv()) == 0
    shape = A.TreeShape(**ok)
    need = A.tree_decode_workspace_bytes(shape, kv())
    assert need > 0 and need % 256 == 0
    assert call(shape, None) == A.ERR_INVALID and call(shape, kv(kv_dtype=A.I8)) == A.ERR_INVALID
    assert call(shape, kv(rows=15)) == A.ERR_INVALID and call(shape, kv(rows=2 ** 31)) == A.ERR_UNSUPPORTED
    for bad in (dict(q=None), dict(out=None), dict(cu=None), dict(ctx=None), dict(lens=None), dict(table=None), dict(begin=None), dict(ptable=None),
                dict(plens=None), dict(q=P + 8), dict(out=Q + 4), dict(lens=P + 2), dict(masks=P + 2), dict(lse=P + 1)):
        assert call(shape, kv(), **bad) == A.ERR_INVALID, bad
    for bad in (dict(ws=None), dict(ws=P + 16), dict(ws_bytes=need - 1)):
        assert call(shape, kv(), **bad) == A.ERR_WORKSPACE, bad
    assert call(A.TreeShape(**{**ok, "mask_words": 0}), kv()) == A.ERR_INVALID and "0 words" in A.last_error()
    for empty in ("n_seq", "n_rows"):
        assert call(A.TreeShape(**{**ok, empty: 0}), kv(), ws=None) == A.OK


def test_commit_refusals():
    ok = dict(n_seq=4, page_size=16, max_pages=8, max_tokens=32, n_pages=64, table_stride=0)

    def call(shape, caches=None, layers=None, heads=2, d=64, words=1, cu=P, ctx=P, lens=P, leaf=P, masks=P, table=P, free=P, count=P, out=Q, counts=Q):
        caches = (A.PagedKV * 2)(*(caches or (kv(), kv())))
        return A.lib.attn_tree_commit_ex(shape, len(caches) if layers is None else layers, caches, heads, d, cu, ctx, lens, leaf, masks, words, table,
                                         free, count, out, counts, None)

    assert call(None) == A.ERR_INVALID
    for bad, status in ((dict(n_seq=-1), A.ERR_INVALID), (dict(n_seq=16385), A.ERR_UNSUPPORTED), (dict(page_size=24), A.ERR_UNSUPPORTED),
                        (dict(max_pages=2 ** 27), A.ERR_INVALID), (dict(table_stride=7), A.ERR_INVALID), (dict(max_tokens=-1), A.ERR_INVALID),
                        (dict(n_pages=-1), A.ERR_INVALID)):
        assert call(A.PageShape(**{**ok, **bad})) == status, bad
    shape = A.PageShape(**ok)
    for bad, status in ((dict(words=0), A.ERR_UNSUPPORTED), (dict(words=33), A.ERR_UNSUPPORTED), (dict(layers=65), A.ERR_INVALID),
                        (dict(layers=-1), A.ERR_INVALID), (dict(heads=0), A.ERR_INVALID), (dict(d=48), A.ERR_UNSUPPORTED),
                        (dict(caches=(kv(), kv(k=None))), A.ERR_INVALID), (dict(caches=(kv(), kv(kv_dtype=A.BF16))), A.ERR_UNSUPPORTED),
                        (dict(caches=(kv(), kv(rows=2 ** 31))), A.ERR_UNSUPPORTED), (dict(caches=(kv(), kv(row_stride=100))), A.ERR_INVALID)):
        assert call(shape, **bad) == status, bad
    for bad in (dict(cu=None), dict(ctx=None), dict(lens=None), dict(leaf=None), dict(table=None), dict(free=None), dict(count=None), dict(out=None),
                dict(counts=None), dict(lens=P + 2), dict(masks=P + 1), dict(out=P + 4), dict(counts=P)):
        assert call(shape, **bad) == A.ERR_INVALID, bad
    assert "overlap" in A.last_error()
    # a cache twice would have its rows moved twice at the same time
    for caches in ((kv(), kv()), (kv(), kv(k=P + (1 << 20))), (kv(), kv(v=P + (1 << 20))), (kv(v=P), kv(k=P + (1 << 20), v=P + (2 << 20)))):
        assert call(shape, caches=caches) == A.ERR_INVALID and "twice" in A.last_error()


def test_commit_refuses_an_array_in_another_part():
    """K of one layer that is V of another, and scales that two layers, or K and V, share: rows and scales would be moved twice
    at the same time."""
    shape = A.PageShape(n_seq=4, page_size=16, max_pages=8, max_tokens=32, n_pages=64, table_stride=0)

    def call(*caches):
        caches = (A.PagedKV * len(caches))(*caches)
        return A.lib.attn_tree_commit_ex(shape, len(caches), caches, 2, 64, P, P, P, P, P, 1, P, P, P, Q, Q + 64, None)

    def layer(i, **kw):
        at = {name: P + (4 * i + j + 1 << 20) for j, name in enumerate(("k", "v", "kscale", "vscale"))}
        return kv(**{**at, **kw})
    one, i8 = layer(0), dict(kv_dtype=A.I8)
    for caches in ((one, layer(1, k=one.v)), (one, layer(1, v=one.k)), (one, layer(1), layer(2, v=one.k)),
                   (layer(0, **i8), layer(1, kscale=one.kscale, **i8)), (layer(0, **i8), layer(1, vscale=one.vscale, **i8)),
                   (layer(0, **i8), layer(1, vscale=one.kscale, **i8)), (layer(0, vscale=one.kscale, **i8),)):
        assert call(*caches) == A.ERR_INVALID and "twice" in A.last_error(), A.last_error()


def test_commit_refuses_outputs_over_inputs():
    """Each of lens_out and counts over each of lens, ctx_lens, leaf, free_count and the other output, from either end."""
    shape = A.PageShape(n_seq=8, page_size=16, max_pages=8, max_tokens=32, n_pages=64, table_stride=0)
    at = dict(ctx=P + 256, lens=P + 512, leaf=P + 768, count=P + 1024, out=Q, counts=Q + 256)

    def call(**kw):
        x = {**at, **kw}
        return A.lib.attn_tree_commit_ex(shape, 1, (A.PagedKV * 1)(kv(v=P + (1 << 20))), 2, 64, P, x["ctx"], x["lens"], x["leaf"], P, 1, P, P, x["count"],
                                         x["out"], x["counts"], None)
    for output in ("out", "counts"):
        for other in ("ctx", "lens", "leaf", "count", "counts"):
            if other == output:
                continue
            for by in (0, 4 if other != "count" else 0, -12):
                assert call(**{output: at[other] + by}) == A.ERR_INVALID and "overlap" in A.last_error(), (output, other, by)


def test_torch_forms(calls):  # noqa: F811
    import torch
    f, b = dict(dtype=torch.float32), dict(dtype=torch.bfloat16)
    given = dict(cu_rows=ints(5), parents=ints(30), positions=ints(30), positions_out=ints(30), masks=ints(30, 2))

    def plan(**kw):
        A.tree_plan_t(kw["cu_rows"], kw["parents"], kw["positions"], kw["positions_out"], kw["masks"])
    for name in given:
        for device in (-1, 1):
            refused(plan, given, {name: Given(given[name].t, device)}, ValueError)
        refused(plan, given, {name: Given(given[name].t.to(torch.int64))}, TypeError)
        if name not in ("cu_rows", "parents"):
            refused(plan, given, {name: Given(given[name].t[:-1])}, ValueError)
    refused(plan, given, {"masks": ints(60)}, ValueError)
    with pytest.raises(Exception, match="^$"):
        plan(**given)

    shape = A.TreeShape(4, 9, 2, 4, 2, 32, A.BF16, 16, 3, 5, 48, 80, 60, 2, 0, 0, 0.0)
    given = dict(q=ints(9, 128, **b), cu_rows=ints(5), ctx_lens=ints(4), lens=ints(4), masks=ints(9, 2), block_table=ints(4, 5), out=ints(9, 128, **b),
                 lse=ints(9, 4, **f), group_begin=ints(3), prefix_table=ints(2, 3), prefix_lens=ints(2), workspace=ints(64, dtype=torch.uint8))
    cache = A.PageCache.of(ints(32, 64, **b), ints(32, 64, **b))

    def decode(cache=cache, **kw):
        A.tree_decode_t(shape, cache, kw["q"], kw["cu_rows"], kw["ctx_lens"], kw["lens"], kw["masks"], kw["block_table"], kw["out"], lse=kw["lse"],
                        group_begin=kw["group_begin"], prefix_table=kw["prefix_table"], prefix_lens=kw["prefix_lens"], workspace=kw["workspace"])
    each_refused(decode, given, optional=("lse", "masks"))
    refused(decode, given, {"q": ints(9, 128, **f)}, TypeError)
    for masks in (ints(18), ints(9, 3), ints(9, 1)):
        refused(decode, given, {"masks": masks}, ValueError)
    with pytest.raises(ValueError, match="device 1"):
        decode(cache=A.PageCache.of(*(Given(torch.zeros((32, 64), **b), 1) for _ in range(2))), **given)

    pages = A.PageShape(4, 16, 8, 30, 64, 0)
    given = dict(cu_rows=ints(5), ctx_lens=ints(4), lens=ints(4), leaf=ints(4), masks=ints(30, 2), block_table=ints(4, 8), free_pages=ints(64),
                 free_count=ints(1), lens_out=ints(4), counts=ints(4))

    def commit(caches=A.cache_array([cache, cache]), **kw):
        A.tree_commit_t(pages, caches, 2, 32, kw["cu_rows"], kw["ctx_lens"], kw["lens"], kw["leaf"], kw["masks"], kw["block_table"], kw["free_pages"],
                        kw["free_count"], kw["lens_out"], kw["counts"])
    each_refused(commit, given, optional=("masks",))
    with pytest.raises(ValueError, match="rows of 32"):
        commit(caches=A.cache_array([cache, A.PageCache.of(ints(32, 32, **b), ints(32, 32, **b))]), **given)


def test_plain_forms():
    """The forms that the GPU tests compare with, on a tree written out: 0 - 1 - 3, 0 - 2 - 4 - 5."""
    tree = [-1, 0, 0, 1, 2, 4]
    pos, masks, code = T.plan(np.array([0, 6]), np.array(tree), np.full(6, 40), np.zeros(6, int), np.zeros((6, 1), np.uint32))
    assert code == 0 and pos.tolist() == [40, 41, 41, 42, 42, 43]
    assert [int(x) for x in masks[:, 0]] == [0b1, 0b11, 0b101, 0b1011, 0b10101, 0b110101]
    assert (T.masks_of([tree], 1) == masks).all()
    cache = np.arange(16.0)[:, None]
    lens, free, counts = T.commit([0, 6], [3], [9], [5], masks, np.array([[2, 0, 1, 3]]), 4, np.full(8, -1), 2, [cache])
    # rows 3, 5, 7, 8 of the request to rows 3, 4, 5, 6; page 1 behind them handed back
    assert lens == [7] and counts == [3, 4, 0, 1] and free.tolist() == [-1, -1, 1, -1, -1, -1, -1, -1]
    assert cache[[8 + 3, 0, 1, 2], 0].tolist() == [11, 1, 3, 4]


PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "prefix.cuh"
using namespace attn::prefix;
// Every piece that any division of the work can leave, of lines of all sizes: within the workspace, and none in another's rows.
int main() {
    for (int tile = 0; tile < 2; tile++)
        for (int variant = 0; variant < 6; variant++) {
            Params p = {};
            p.ratio = variant % 3 + 1;
            p.kv_heads = 3;
            const int tokens[] = {0, 1, 40, 128, 200, 3, 0, 65, 129 % (variant + 100)};
            const int groups[][2] = {{0, 3}, {3, 6}, {6, 9}};
            const int n = 9, g = variant < 3 ? 3 : 0;
            std::vector<int> cu(1, 0);
            for (int t : tokens) cu.push_back(cu.back() + t);
            p.n_seq = cu.back(); p.n_req = n; p.n_groups = g;
            Part w = {};
            w.half = tile ? 128 : 0;
            w.log_rows = tile ? 8 : variant % 4 + 1;
            w.head_block = tile ? 1 : 2;
            w.n_blocks = tile ? 3 : 2;
            const long long rows = (long long)p.n_seq * p.ratio, heads = (long long)w.n_blocks * w.head_block;
            w.rows = 1 << w.log_rows;
            w.after = g ? (rows + (long long)w.half * g) * heads : 0;
            const int teams = 5;
            std::vector<int> owner((size_t)(w.after + rows * (w.half ? 2 : 1) * heads + (long long)teams * w.head_block * w.rows), 0);
            int segment = 0, of_team = 7, team = 0, left = of_team;      // a team ends within every few segments
            for (int i = 0; i < g + n; i++) {
                Line l = {};
                l.prefix = i < g;
                const int a = cu[l.prefix ? groups[i][0] : i - g], b = cu[l.prefix ? groups[i][1] : i - g + 1];
                l.first_req = a;
                l.rows = (b - a) * p.ratio;
                l.blocks = (l.rows + w.rows - 1) / w.rows;
                l.base = (a * p.ratio >> w.log_rows) + (l.prefix ? i : i - g);
                for (int rb = 0; rb < l.blocks; rb++)
                    for (int hb = 0; hb < w.n_blocks; hb++, segment++) {
                        const Place x = place_of<TREES>(p, w, l, rb, hb);
                        const int r = l.rows - (rb << w.log_rows) < w.rows ? l.rows - (rb << w.log_rows) : w.rows;
                        for (int steps = 1 + segment % 3; steps > 0;) {
                            const int now = steps < left ? steps : left;
                            const int parts = tile ? 2 : w.head_block;
                            for (int k = 0; k < parts; k++) {
                                const int own = tile ? (r <= 128 ? r : k ? r - 128 : 128) : r;
                                for (int y = 0; y < own; y++) {
                                    const long long at = x.first + team * x.step + (long long)k * x.apart + y;
                                    if (at < 0 || at >= (long long)owner.size()) return printf("outside %lld of %zu\n", at, owner.size()), 1;
                                    if (owner[at]++) return printf("twice %lld (tile %d, line %d)\n", at, tile, i), 1;
                                }
                            }
                            steps -= now;
                            left -= now;
                            if (!left) left = ++team < teams - 1 ? of_team : 1 << 30;
                        }
                    }
            }
        }
    puts("ok");
}
"""


def test_pieces_have_places_of_their_own(tmp_path):
    if shutil.which("nvcc") is None:
        pytest.skip("nvcc not present")
    (tmp_path / "t.cu").write_text(PROGRAM)
    build = subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                            "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(PKG, "csrc"), "-o", "t", "t.cu", "-lcudart"],
                           cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr
    run = subprocess.run(["./t"], cwd=tmp_path, capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout
