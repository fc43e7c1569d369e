"""Refusals of the serving entry points: argument checks run before any CUDA call."""
import ctypes

import pytest

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


# ---------------------------------------------------------------------------
# the torch forms: each tensor is held against the shape beside it
# ---------------------------------------------------------------------------
class Given:
    """A stand-in for a CUDA tensor: what the checks look at, at an address that is never read."""

    def __init__(self, tensor, device=0):
        self.t, self.is_cuda, self.device = tensor, device >= 0, f"cuda:{device}" if device >= 0 else "cpu"
        self.dtype, self.shape, self.get_device = tensor.dtype, tensor.shape, lambda: device

    def __getattr__(self, name):
        return getattr(self.t, name)


class Reached(Exception):
    pass


@pytest.fixture
def calls(monkeypatch):
    """Calls that pass the checks end with Reached and not in the library."""
    def stop(*args):
        raise Reached

    class Lib:
        def __getattr__(self, name):
            return stop
    monkeypatch.setattr(A, "lib", Lib())
    monkeypatch.setattr(A, "_stream", lambda: 0)
    monkeypatch.setattr(A, "_device", lambda: 0)


def refused(call, given, bad, error):
    with pytest.raises(error) as e:
        call(**{**given, **bad})
    assert next(iter(bad)) in str(e.value), str(e.value)


def each_refused(call, given, optional=()):
    """Every tensor on its own: of another type, too short, on the host, on another GPU."""
    import torch
    with pytest.raises(Reached):
        call(**given)
    for name, g in given.items():
        other = torch.int64 if g.dtype == torch.int32 else torch.int32 if g.dtype == torch.int64 else torch.float64
        if name != "q" and name != "workspace":
            refused(call, given, {name: Given(g.t.to(other))}, TypeError)
        for device in (-1, 1):
            refused(call, given, {name: Given(g.t, device)}, ValueError)
        if name != "workspace":
            refused(call, given, {name: Given(g.t[:-1])}, ValueError)
            if g.numel() > 1:
                refused(call, given, {name: Given(torch.empty((2 * g.shape[0],) + g.shape[1:], dtype=g.dtype)[::2])}, ValueError)
        if name in optional:
            with pytest.raises(Reached):
                call(**{**given, name: None})


def ints(*shape, dtype=None):
    import torch
    return Given(torch.zeros(shape, dtype=dtype or torch.int32))


def test_page_plan_tensors(calls):
    import torch
    shape = A.PageShape(4, 16, 8, 32, 64, 0)
    given = dict(lens=ints(4), new_lens=ints(4), pos_base=ints(4), free_pages=ints(64), free_count=ints(1), block_table=ints(4, 8),
                 cu_new=ints(5), positions=ints(32), token_seq=ints(32), counts=ints(4), slot_map=ints(32, dtype=torch.int64), lens_out=ints(4))

    def call(**kw):
        out = {k: kw[k] for k in ("cu_new", "positions", "token_seq", "counts", "slot_map")}
        A.page_plan_t(shape, kw["lens"], kw["new_lens"], kw["free_pages"], kw["free_count"], kw["block_table"], {**out, "lens": kw["lens_out"]},
                      pos_base=kw["pos_base"])
    lens_out = given.pop("lens_out")
    each_refused(lambda **kw: call(lens_out=lens_out, **kw), given, optional=("pos_base", "token_seq"))
    with pytest.raises(TypeError, match="lens"):
        call(**given, lens_out=ints(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="lens"):
        call(**given, lens_out=ints(3))
    given["lens_out"], shape.table_stride = lens_out, 11  # a table inside a wider one
    with pytest.raises(ValueError, match="block_table"):
        call(**given)
    for table in (ints(4, 11), Given(torch.zeros((4, 11), dtype=torch.int32)[:, 2:10])):
        with pytest.raises(Reached):
            call(**{**given, "block_table": table})


def test_rope_tensors(calls):
    import torch
    shape = A.RopeShape(6, 0, 4, 2, 32, 32, 0, 16, 0, 0, 0, 0, 0)
    f = dict(dtype=torch.float32)
    given = dict(table=Given(torch.zeros((16, 16, 2))), positions=ints(6), q=ints(6, 128, **f), k=ints(6, 64, **f), q_out=ints(6, 128, **f),
                 k_out=ints(6, 64, **f))

    def call(**kw):
        A.rope_t(shape, kw["table"], kw["positions"], kw["q"], kw["k"], kw["q_out"], kw["k_out"])
    each_refused(call, given, optional=("positions", "k", "k_out"))
    refused(call, given, {"k": ints(6, 64, dtype=torch.bfloat16)}, TypeError)
    refused(call, given, {"q": Given(torch.zeros((6, 200))[:, :128])}, ValueError)          # its stride is not the shape's
    refused(call, given, {"q": ints(6, 256, **f)}, ValueError)
    for q in (ints(6, 4, 32, **f), ints(24, 32, **f), ints(9, 128, **f)):     # the same memory in other shapes, and more of it
        with pytest.raises(Reached):
            call(**{**given, "q": q})
    shape.q_row_stride = 200
    with pytest.raises(Reached):
        call(**{**given, "q": Given(torch.zeros((6, 200))[:, 30:158])})


def test_rope_append_tensors(calls):
    import torch
    shape = A.RopeShape(6, 0, 4, 2, 32, 32, 0, 16, 0, 0, 0, 0, 0)
    f = dict(dtype=torch.float32)
    given = dict(table=Given(torch.zeros((16, 16, 2))), positions=ints(6), slot_map=ints(6, dtype=torch.int64), q=ints(6, 128, **f),
                 k=ints(6, 64, **f), v=ints(6, 64, **f), q_out=ints(6, 128, **f))
    cache = A.PageCache.of(ints(32, 64, **f), ints(32, 64, **f))

    def call(kv=cache, **kw):
        A.rope_append_t(shape, kv, kw["table"], kw["positions"], kw["slot_map"], kw["q"], kw["k"], kw["v"], kw["q_out"])
    each_refused(call, given, optional=("positions",))
    narrow = A.PageCache.of(*(Given(torch.zeros((32, 96))[:, :32]) for _ in range(2)))
    codes = [ints(32, 64, dtype=torch.int8) for _ in range(2)]
    other = A.PageCache.of(*codes, *(Given(torch.zeros(32, 4)) for _ in range(2)))
    away = A.PageCache.of(*(Given(torch.zeros(32, 64), 1) for _ in range(2)))
    for kv, word in ((narrow, "rows of 32"), (other, "scales of 4"), (away, "device 1")):
        with pytest.raises(ValueError, match=word):
            call(kv=kv, **given)


def test_page_cache_tensors():
    import torch
    f = dict(dtype=torch.float32)
    k, scale, codes = ints(8, 64, **f), ints(8, 2, **f), ints(8, 64, dtype=torch.int8)
    A.PageCache.of(k, k)
    A.PageCache.of(codes, codes, scale, scale)
    for bad in ((k, ints(8, 64, dtype=torch.bfloat16)), (k, ints(7, 64, **f)), (k, Given(k.t, -1)), (k, Given(k.t, 1)), (ints(512, **f),) * 2,
                (codes, codes), (codes, codes, scale, None), (codes, codes, scale, ints(7, 2, **f)), (codes, codes, scale, ints(8, 3, **f))):
        with pytest.raises(ValueError):
            A.PageCache.of(*bad)
    for bad in ((codes, codes, scale, ints(8, 2, dtype=torch.float64)), (codes, codes, scale, Given(scale.t, 1)), (ints(8, 64, dtype=torch.float64),) * 2):
        with pytest.raises(TypeError):
            A.PageCache.of(*bad)


def test_prefix_decode_tensors(calls):
    import torch
    shape = A.PrefixShape(4, 2, 4, 2, 32, A.BF16, 16, 3, 5, 48, 80, 0, 0, 0.0)
    b = dict(dtype=torch.bfloat16)
    given = dict(q=ints(4, 128, **b), group_begin=ints(3), prefix_table=ints(2, 3), prefix_lens=ints(2), block_table=ints(4, 5), lens=ints(4),
                 out=ints(4, 128, **b), lse=ints(4, 4, dtype=torch.float32), workspace=ints(64, dtype=torch.uint8))
    cache = A.PageCache.of(ints(32, 64, **b), ints(32, 64, **b))

    def call(**kw):
        A.prefix_decode_t(shape, cache, kw["q"], kw["group_begin"], kw["prefix_table"], kw["prefix_lens"], kw["block_table"], kw["lens"],
                          kw["out"], lse=kw["lse"], workspace=kw["workspace"])
    each_refused(call, given, optional=("lse", "workspace"))
    refused(call, given, {"q": ints(4, 128, dtype=torch.float32)}, TypeError)
    refused(call, given, {"block_table": ints(4, 6)}, ValueError)                          # its lines are not max_pages apart
    with pytest.raises(ValueError, match="rows of 64"):
        shape.kv_heads = 4
        call(**given)
    shape.kv_heads, shape.n_groups = 2, 0
    with pytest.raises(Reached):
        call(**{**given, "group_begin": None, "prefix_table": None, "prefix_lens": None})
