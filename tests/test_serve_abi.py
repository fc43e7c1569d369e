"""Refusals of the serving entry points: argument checks run before any CUDA call."""
import ctypes

import attn_b200 as A

P = 1 << 20                                      # an aligned stand-in address
Q = 1 << 21


def plan(shape, **change):
    args = dict(lens=P, new=P, base=None, free=P, count=P, table=P, lens_out=Q, cu=Q, slots=Q, positions=Q, seq=None,
                counts=Q)
    args.update(change)
    return A.lib.attn_page_plan_ex(shape, *args.values(), None)


def test_page_plan_refusals():
    ok = dict(n_seq=4, page_size=16, max_pages=8, max_tokens=32, n_pages=64, table_stride=0)
    assert plan(None) == A.ERR_INVALID
    for bad, status in ((dict(n_seq=-1), A.ERR_INVALID), (dict(n_seq=16385), A.ERR_UNSUPPORTED), (dict(page_size=24), A.ERR_UNSUPPORTED),
                        (dict(page_size=0), A.ERR_UNSUPPORTED), (dict(page_size=2048), A.ERR_UNSUPPORTED),
                        (dict(max_pages=2 ** 27), A.ERR_INVALID), (dict(table_stride=7), A.ERR_INVALID),
                        (dict(max_tokens=-1), A.ERR_INVALID), (dict(n_pages=-1), A.ERR_INVALID)):
        assert plan(A.PageShape(**{**ok, **bad})) == status, bad
    shape = A.PageShape(**ok)
    for bad in (dict(lens=None), dict(count=None), dict(table=None), dict(slots=None), dict(counts=None), dict(free=None),
                dict(lens=P + 2), dict(slots=Q + 4), dict(lens_out=P + 4), dict(counts=P)):
        assert plan(shape, **bad) == A.ERR_INVALID, bad
    assert "overlap" in A.last_error()


def test_rope_refusals():
    ok = dict(tokens=4, seq_len=0, heads=4, kv_heads=2, head_dim=64, rot_dim=64, interleaved=0, max_pos=16, q_row_stride=0,
              k_row_stride=0, v_row_stride=0, q_out_row_stride=0, k_out_row_stride=0)

    def rope(shape, dtype=A.F32, table=P, pos=P, q=P, k=P, q_out=Q, k_out=Q):
        return A.lib.attn_rope_ex(shape, dtype, table, pos, q, k, q_out, k_out, 0, None)

    assert rope(None) == A.ERR_INVALID
    for bad, status in ((dict(tokens=-1), A.ERR_INVALID), (dict(head_dim=48), A.ERR_UNSUPPORTED), (dict(rot_dim=3), A.ERR_INVALID),
                        (dict(rot_dim=66), A.ERR_INVALID), (dict(max_pos=0), A.ERR_INVALID), (dict(q_row_stride=255), A.ERR_INVALID),
                        (dict(k_out_row_stride=127), A.ERR_INVALID), (dict(kv_heads=0), A.ERR_INVALID)):
        assert rope(A.RopeShape(**{**ok, **bad})) == status, bad
    shape = A.RopeShape(**ok)
    assert rope(shape, dtype=A.I8) == A.ERR_UNSUPPORTED
    for bad in (dict(table=None), dict(table=P + 4), dict(pos=None), dict(pos=P + 2), dict(q=None), dict(q_out=None), dict(k=None),
                dict(k_out=None), dict(q=P + 2)):
        assert rope(shape, **bad) == A.ERR_INVALID, bad
    inplace = A.RopeShape(**{**ok, "q_row_stride": 512})
    assert rope(inplace, q=P, q_out=P) == A.ERR_INVALID and "in place" in A.last_error()
    assert rope(A.RopeShape(**{**ok, "tokens": 0})) == A.OK


def test_rope_table_refusals():
    ok = dict(rot_dim=64, max_pos=16, scaling=A.ROPE_PLAIN, trained_len=0, base=10000.0, factor=0.0, fast=0.0, slow=0.0, magnitude=0.0)

    def table(**change):
        return A.lib.attn_rope_table_ex(A.RopeConfig(**{**ok, **change}), P, None)

    for bad, status in ((dict(rot_dim=0), A.ERR_INVALID), (dict(rot_dim=7), A.ERR_INVALID), (dict(rot_dim=130), A.ERR_INVALID),
                        (dict(base=1.0), A.ERR_INVALID), (dict(scaling=4), A.ERR_UNSUPPORTED), (dict(scaling=A.ROPE_LINEAR), A.ERR_INVALID),
                        (dict(scaling=A.ROPE_BASE, factor=2.0, rot_dim=2), A.ERR_INVALID),
                        (dict(scaling=A.ROPE_RAMP, factor=2.0, trained_len=4096, fast=1.0, slow=1.0), A.ERR_INVALID)):
        assert table(**bad) == status, bad
    assert A.lib.attn_rope_table_ex(A.RopeConfig(**ok), None, None) == A.ERR_INVALID
    assert A.lib.attn_rope_table_ex(None, P, None) == A.ERR_INVALID
    assert table(max_pos=0) == A.OK


def kv(**change):
    ok = dict(kv_dtype=A.F32, rows=64, row_stride=0, k=P, v=P, kscale=None, vscale=None)
    return A.PagedKV(**{**ok, **change})


def test_rope_append_refusals():
    shape = A.RopeShape(4, 0, 4, 2, 64, 64, 0, 16, 0, 0, 0, 0, 0)

    def append(cache, dtype=A.F32, slots=P, q=P, k=P, v=P, q_out=Q):
        return A.lib.attn_rope_append_ex(shape, cache, dtype, P, P, slots, q, k, v, q_out, None)

    assert append(None) == A.ERR_INVALID
    assert append(kv(kv_dtype=9)) == A.ERR_UNSUPPORTED
    assert append(kv(kv_dtype=A.BF16)) == A.ERR_UNSUPPORTED and append(kv(), dtype=A.BF16) == A.ERR_UNSUPPORTED
    for bad in (dict(k=None), dict(v=P + 8), dict(row_stride=127), dict(row_stride=130), dict(kv_dtype=A.I8), dict(rows=-1)):
        assert append(kv(**bad)) == A.ERR_INVALID, bad
    for bad in (dict(slots=None), dict(slots=P + 4), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(v=P + 2)):
        assert append(kv(), **bad) == A.ERR_INVALID, bad


def test_prefix_decode_refusals():
    ok = dict(n_seq=4, n_groups=1, heads=4, kv_heads=2, head_dim=64, dtype=A.F32, page_size=16, max_prefix_pages=4, max_pages=4,
              max_prefix_len=64, max_len=64, q_row_stride=0, out_row_stride=0, scale=0.0)

    def decode(shape, cache, q=P, begin=P, ptable=P, plens=P, table=P, lens=P, out=Q, lse=None, ws=None, ws_bytes=0):
        return A.lib.attn_prefix_decode_ex(shape, cache, q, begin, ptable, plens, table, lens, out, lse, ws, ws_bytes, None)

    assert decode(None, kv()) == A.ERR_INVALID
    for bad, status in ((dict(n_seq=-1), A.ERR_INVALID), (dict(n_seq=65536), A.ERR_INVALID), (dict(heads=3), A.ERR_INVALID),
                        (dict(head_dim=80), A.ERR_UNSUPPORTED), (dict(dtype=A.BF16), A.ERR_UNSUPPORTED), (dict(page_size=20), A.ERR_UNSUPPORTED),
                        (dict(max_len=65), A.ERR_INVALID), (dict(max_prefix_len=65), A.ERR_INVALID), (dict(q_row_stride=255), A.ERR_INVALID),
                        (dict(out_row_stride=258), A.ERR_INVALID), (dict(scale=-1.0), A.ERR_INVALID), (dict(scale=float("nan")), A.ERR_INVALID),
                        (dict(n_groups=-1), A.ERR_INVALID)):
        shape = A.PrefixShape(**{**ok, **bad})
        assert decode(shape, kv()) == status, bad
        assert A.prefix_decode_workspace_bytes(shape, kv()) == 0
    shape = A.PrefixShape(**ok)
    assert A.prefix_decode_workspace_bytes(shape, kv()) > 0
    assert decode(shape, None) == A.ERR_INVALID and decode(shape, kv(kv_dtype=A.I8)) == A.ERR_INVALID
    assert decode(shape, kv(kv_dtype=A.BF16)) == A.ERR_UNSUPPORTED
    assert decode(shape, kv(rows=15)) == A.ERR_INVALID and decode(shape, kv(rows=2 ** 31)) == A.ERR_UNSUPPORTED
    for bad in (dict(q=None), dict(out=None), dict(lens=None), dict(table=None), dict(begin=None), dict(ptable=None), dict(plens=None),
                dict(q=P + 8), dict(out=Q + 4), dict(lens=P + 2), dict(lse=P + 1)):
        assert decode(shape, kv(), **bad) == A.ERR_INVALID, bad
    assert decode(shape, kv(), ws=P, ws_bytes=1) == A.ERR_WORKSPACE
    assert decode(shape, kv(), ws=P + 16, ws_bytes=1 << 30) == A.ERR_WORKSPACE
    assert decode(A.PrefixShape(**{**ok, "n_seq": 0}), kv()) == A.OK
