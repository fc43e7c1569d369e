"""Refusals of the normed rotary calls, and of their torch forms; and the gradient's formula against differences."""
import numpy as np
import pytest

import attn_b200 as A
import norm_ref as N
import serve_ref as R
from test_serve_abi import Given, calls, each_refused, ints, kv, refused  # noqa: F401

P, Q = 1 << 20, 1 << 21
OK = dict(tokens=4, seq_len=0, heads=4, kv_heads=2, head_dim=64, rot_dim=64, interleaved=0, max_pos=16, q_row_stride=0,
          k_row_stride=0, v_row_stride=0, q_out_row_stride=0, k_out_row_stride=0)
NORM = A.HeadNormPtrs(P, P, 1e-6)


def test_forward_refusals():
    def call(shape, norm=NORM, dtype=A.F32, table=P, pos=P, q=P, k=P, q_out=Q, k_out=Q):
        return A.lib.attn_norm_rope_ex(shape, norm, dtype, table, pos, q, k, q_out, k_out, None)

    assert call(None) == A.ERR_INVALID
    for bad, status in ((dict(tokens=-1), A.ERR_INVALID), (dict(head_dim=48), A.ERR_UNSUPPORTED), (dict(rot_dim=3), A.ERR_INVALID),
                        (dict(rot_dim=66), A.ERR_INVALID), (dict(max_pos=0), A.ERR_INVALID), (dict(q_row_stride=255), A.ERR_INVALID),
                        (dict(k_out_row_stride=127), A.ERR_INVALID), (dict(kv_heads=0), A.ERR_INVALID)):
        assert call(A.RopeShape(**{**OK, **bad})) == status, bad
    shape = A.RopeShape(**OK)
    assert call(shape, dtype=A.I8) == A.ERR_UNSUPPORTED
    for bad in (dict(norm=None), dict(norm=A.HeadNormPtrs(P, P, -1.0)), dict(norm=A.HeadNormPtrs(P, P, float("nan"))),
                dict(norm=A.HeadNormPtrs(P + 2, P, 0.0)), dict(table=None), dict(table=P + 4), dict(pos=None), dict(q=None), dict(q_out=None),
                dict(k=None), dict(k_out=None), dict(q=P + 2)):
        assert call(shape, **bad) == A.ERR_INVALID, bad
    assert call(A.RopeShape(**{**OK, "q_row_stride": 512}), q=P, q_out=P) == A.ERR_INVALID and "in place" in A.last_error()
    assert call(A.RopeShape(**{**OK, "k_out_row_stride": 512}), k=P, k_out=P) == A.ERR_INVALID
    assert call(A.RopeShape(**{**OK, "tokens": 0})) == A.OK


def test_backward_refusals():
    def call(shape, norm=NORM, dtype=A.F32, table=P, pos=P, q=P, k=P, gq=P, gk=P, dq=Q, dk=Q, dqw=Q, dkw=Q, ws=P, ws_bytes=1 << 40):
        return A.lib.attn_norm_rope_bwd_ex(shape, norm, dtype, table, pos, q, k, gq, gk, dq, dk, dqw, dkw, 0, ws, ws_bytes, None)

    assert call(None) == A.ERR_INVALID
    shape = A.RopeShape(**OK)
    assert call(A.RopeShape(**{**OK, "head_dim": 80})) == A.ERR_UNSUPPORTED and call(shape, dtype=A.I8) == A.ERR_UNSUPPORTED
    for bad in (dict(norm=None), dict(table=None), dict(q=None), dict(gq=None), dict(dq=None), dict(k=None), dict(gk=None), dict(dk=None),
                dict(q=P + 2), dict(gk=P + 1), dict(dk=Q + 2), dict(dqw=Q + 2), dict(dkw=Q + 1)):
        assert call(shape, **bad) == A.ERR_INVALID, bad
    assert call(A.RopeShape(**{**OK, "q_out_row_stride": 512}), gq=Q, dq=Q) == A.ERR_INVALID and "in place" in A.last_error()
    need = A.norm_rope_bwd_workspace_bytes(shape)
    assert need >= 2 * 64 * 4 and need % 256 == 0
    for bad in (dict(ws=None), dict(ws=P + 16), dict(ws_bytes=need - 1)):
        assert call(shape, **bad) == A.ERR_WORKSPACE, bad
    assert A.norm_rope_bwd_workspace_bytes(A.RopeShape(**{**OK, "head_dim": 80})) == 0
    for dkw in (Q, Q + 4 * 63, Q - 4 * 63):                # one weight for q and k has two gradients
        assert call(shape, dkw=dkw) == A.ERR_INVALID and "overlap" in A.last_error()


def test_append_refusals():
    shape = A.RopeShape(**OK)

    def call(cache, norm=NORM, dtype=A.F32, slots=P, q=P, k=P, v=P, q_out=Q, shape=shape):
        return A.lib.attn_norm_rope_append_ex(shape, norm, cache, dtype, P, P, slots, q, k, v, q_out, None)

    assert call(None) == A.ERR_INVALID and call(kv(), norm=None) == A.ERR_INVALID
    assert call(kv(kv_dtype=A.BF16)) == A.ERR_UNSUPPORTED and call(kv(), dtype=A.BF16) == A.ERR_UNSUPPORTED
    for bad in (dict(k=None), dict(v=P + 8), dict(row_stride=127), dict(kv_dtype=A.I8), dict(rows=-1)):
        assert call(kv(**bad)) == A.ERR_INVALID, bad
    for bad in (dict(slots=None), dict(slots=P + 4), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(v=P + 2)):
        assert call(kv(), **bad) == A.ERR_INVALID, bad
    assert call(kv(), shape=A.RopeShape(**{**OK, "q_row_stride": 512}), q=Q) == A.ERR_INVALID
    assert call(kv(), shape=A.RopeShape(**{**OK, "tokens": 0})) == A.OK


def test_torch_forms(calls):  # noqa: F811
    import torch
    f = dict(dtype=torch.float32)
    shape = A.RopeShape(6, 0, 4, 2, 32, 32, 0, 16, 0, 0, 0, 0, 0)
    rope = dict(table=Given(torch.zeros((16, 16, 2))), positions=ints(6))
    weights = dict(q_weight=ints(32, **f), k_weight=ints(32, **f))
    rows = {n: ints(6, 128 if "q" in n else 64, **f) for n in ("q", "k", "v", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk")}
    pick = lambda *names: {n: rows[n] for n in names}  # noqa: E731

    def norm(kw):
        return A.HeadNorm.of(kw["q_weight"], kw["k_weight"], 1e-6)

    def forward(**kw):
        A.norm_rope_t(shape, norm(kw), kw["table"], kw["positions"], kw["q"], kw["k"], kw["q_out"], kw["k_out"])
    given = {**rope, **weights, **pick("q", "k", "q_out", "k_out")}
    each_refused(forward, given, optional=("positions", "k", "k_out", "q_weight", "k_weight"))
    refused(forward, given, {"q": Given(torch.zeros((6, 200))[:, :128])}, ValueError)

    def backward(**kw):
        A.norm_rope_bwd_t(shape, norm(kw), kw["table"], kw["positions"], kw["q"], kw["k"], kw["dq_out"], kw["dk_out"], kw["dq"], kw["dk"],
                          kw["dq_weight"], kw["dk_weight"], workspace=kw["workspace"])
    given = {**rope, **weights, **pick("q", "k", "dq_out", "dk_out", "dq", "dk"), "dq_weight": ints(32, **f), "dk_weight": ints(32, **f),
             "workspace": ints(64, dtype=torch.uint8)}
    each_refused(backward, given, optional=("positions", "q_weight", "dq_weight", "dk_weight"))

    cache = A.PageCache.of(ints(32, 64, **f), ints(32, 64, **f))

    def append(cache=cache, **kw):
        A.norm_rope_append_t(shape, norm(kw), cache, kw["table"], kw["positions"], kw["slot_map"], kw["q"], kw["k"], kw["v"], kw["q_out"])
    given = {**rope, **weights, **pick("q", "k", "v", "q_out"), "slot_map": ints(6, dtype=torch.int64)}
    each_refused(append, given, optional=("positions", "q_weight"))
    away = A.PageCache.of(*(Given(torch.zeros(32, 64), 1) for _ in range(2)))
    with pytest.raises(ValueError, match="device 1"):
        append(cache=away, **given)


@pytest.mark.parametrize("interleaved", [0, 1])
def test_gradient_formula_against_differences(interleaved):
    """Central differences in 64 bits: h^2 of a third derivative of order 1 (the inputs are), and rounding 2^-52 / h."""
    r = np.random.RandomState(3)
    n, heads, d, rot, h = 3, 2, 8, 6, 1e-4
    x, g, w = r.randn(n, heads * d), r.randn(n, heads * d), 1 + 0.3 * r.randn(d)
    table, pos = R.rope_table(rot, 20), np.array([0, 7, 19])

    def f(x, w):
        return (N.forward(x, heads, w, 1e-5, table, pos, rot, interleaved)[0] * g).sum()
    dx, dw, _, _ = N.backward(x, g, heads, w, 1e-5, table, pos, rot, interleaved)
    for i in range(n):
        for j in range(heads * d):
            e = np.zeros_like(x)
            e[i, j] = h
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx[i, j]) < 1e-6
    for j in range(d):
        e = np.zeros(d)
        e[j] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[j]) < 1e-6
