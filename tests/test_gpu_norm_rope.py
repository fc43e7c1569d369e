"""Normed and turned heads on the GPU against the 64-bit forms of norm_ref.py.

Tolerances, in roundings u = 2^-24 of fp32:
  forward   a sum of squares takes up to 8 fused steps in a lane, 5 between lanes and 3 for the mean and eps, 16 u, half of it
            in r, whose root adds 1 u; r w and its product with x add 2, the two products and the sum of the rotation 2: under
            16 u (|a c| + |b s|).  bf16: 2^-8 of the result more.
  backward  the gradient turned back is off by 2 u G, G = |a c| + |b s|; times w 3 u.  mean(g w x) is off by 3 u and 16 u of
            its sum of magnitudes, r^2 by 18 u, three products 3 u, the sum 1 u, r 9 u and its product 1 u: under
            64 u r (G |w| + |x| r^2 mean(G |w x|)).  bf16: 2^-8 of the result more.
  weights   a term is off by 13 u G |x| r, and a sum of n terms in fp32 by at most n u of the magnitudes.
  INT8      a code is the nearest: half a scale, and the scale's and value's own error, 2^-16 of 127 scales at most."""
import ctypes

import numpy as np
import pytest

import norm_ref as N
import synth

pytestmark = pytest.mark.gpu

U = N.U
EPS = 1e-5
# tokens, heads, kv_heads, d, rot
SHAPES = [(1, 1, 1, 32, 32), (5, 3, 1, 64, 26), (37, 12, 12, 128, 128), (130, 16, 4, 96, 48), (64, 8, 8, 64, 0), (9, 5, 5, 32, 2),
          (300, 32, 8, 128, 64), (2, 1, 1, 96, 96), (3, 7, 2, 128, 126), (11, 2, 2, 96, 6)]


@pytest.fixture(scope="module")
def A(cuda):
    import attn_b200
    return attn_b200


def dev(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def device_error(A):
    code = ctypes.c_int()
    A.check(A.lib.attn_device_error(0, ctypes.byref(code)))
    return code.value


class Case:
    """Inputs of a call: tensors, and what they hold in 64 bits."""

    def __init__(self, A, seed, tokens, heads, kv_heads, d, rot, interleaved, kind, max_pos=97, std=1.0):
        import torch
        self.A, self.tokens, self.heads, self.kv_heads, self.d, self.rot, self.interleaved = A, tokens, heads, kv_heads, d, rot, interleaved
        self.type = torch.bfloat16 if kind == "bf16" else torch.float32
        self.half = 2.0 ** -8 if kind == "bf16" else 0.0
        self.q, self.k, self.v, self.gq, self.gk = (
            dev(synth.normal(seed + i, (tokens, h * d), 0, std), self.type) for i, h in enumerate((heads, kv_heads, kv_heads, heads, kv_heads)))
        self.qw, self.kw = ((1 + 0.4 * synth.normal(seed + 7 + i, (d,))).astype(np.float32) for i in range(2))
        self.norm = A.HeadNorm.of(dev(self.qw), dev(self.kw), EPS)
        self.pos = np.random.RandomState(seed).randint(0, max_pos, tokens).astype(np.int32)
        import serve_ref as R
        self.table = R.rope_table(rot, max_pos, magnitude=1.1).astype(np.float32) if rot else np.zeros((max_pos, 0, 2), np.float32)
        self.max_pos = max_pos

    def shape(self, seq_len=0, **strides):
        s = self.A.RopeShape(self.tokens, seq_len, self.heads, self.kv_heads, self.d, self.rot, self.interleaved, self.max_pos, 0, 0, 0, 0, 0)
        for k, v in strides.items():
            setattr(s, k, v)
        return s

    def want(self, x, heads, weight, pos=None):
        return N.forward(host(x), heads, weight.astype(np.float64), np.float64(np.float32(EPS)), self.table, self.pos if pos is None else pos,
                         self.rot, self.interleaved)

    def check_forward(self, got, x, heads, weight, pos=None):
        want, most = self.want(x, heads, weight, pos)
        tol = 16 * U * most + self.half * np.abs(want) + 1e-37
        assert (np.abs(host(got) - want) <= tol).all(), (np.abs(host(got) - want) / tol).max()

    def check_backward(self, dx, dw, x, grad, heads, weight, pos=None, before=0.0):
        want, want_w, most, most_w = N.backward(host(x), host(grad), heads, weight.astype(np.float64), np.float64(np.float32(EPS)), self.table,
                                                self.pos if pos is None else pos, self.rot, self.interleaved)
        tol = 64 * U * most + self.half * np.abs(want) + 1e-37
        assert (np.abs(host(dx) - want) <= tol).all(), (np.abs(host(dx) - want) / tol).max()
        if dw is not None:
            tol = (13 + self.tokens * heads) * U * most_w + 2 * U * np.abs(want_w + before) + 1e-37
            assert (np.abs(host(dw) - before - want_w) <= tol).all(), (np.abs(host(dw) - before - want_w) / tol).max()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", SHAPES)
def test_norm_rope(A, tokens, heads, kv_heads, d, rot, interleaved, kind):
    import torch
    c = Case(A, tokens + d, tokens, heads, kv_heads, d, rot, interleaved, kind)
    qo, ko = torch.full_like(c.q, float("nan")), torch.full_like(c.k, float("nan"))
    A.norm_rope_t(c.shape(), c.norm, dev(c.table), dev(c.pos), c.q, c.k, qo, ko)
    c.check_forward(qo, c.q, heads, c.qw)
    c.check_forward(ko, c.k, kv_heads, c.kw)
    qi, ki = c.q.clone(), c.k.clone()             # in place, the same bits
    A.norm_rope_t(c.shape(), c.norm, dev(c.table), dev(c.pos), qi, ki, qi, ki)
    assert torch.equal(qi, qo) and torch.equal(ki, ko)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", SHAPES)
def test_norm_rope_gradients(A, tokens, heads, kv_heads, d, rot, interleaved, kind):
    import torch
    c = Case(A, tokens + d + 1, tokens, heads, kv_heads, d, rot, interleaved, kind)
    dq, dk = torch.full_like(c.q, float("nan")), torch.full_like(c.k, float("nan"))
    dqw, dkw = (torch.full((d,), float("nan"), device="cuda") for _ in range(2))
    args = (c.shape(), c.norm, dev(c.table), dev(c.pos), c.q, c.k)
    A.norm_rope_bwd_t(*args, c.gq, c.gk, dq, dk, dqw, dkw)
    c.check_backward(dq, dqw, c.q, c.gq, heads, c.qw)
    c.check_backward(dk, dkw, c.k, c.gk, kv_heads, c.kw)
    # in place of the outputs' gradients, adding to the weights', without them, and again: the same bits
    gq, gk, add = c.gq.clone(), c.gk.clone(), torch.full((d,), 3.0, device="cuda")
    A.norm_rope_bwd_t(*args, gq, gk, gq, gk, add, None, accumulate=True)
    assert torch.equal(gq, dq) and torch.equal(gk, dk)
    c.check_backward(gq, add, c.q, c.gq, heads, c.qw, before=3.0)
    qi, ki, again = c.q.clone(), c.k.clone(), torch.empty_like(dqw)
    A.norm_rope_bwd_t(c.shape(), c.norm, dev(c.table), dev(c.pos), qi, ki, c.gq, c.gk, qi, ki, again, None)
    assert torch.equal(qi, dq) and torch.equal(ki, dk) and torch.equal(again, dqw)


def test_gradients_against_differences(A):
    """Central differences of the 64-bit forward form, of steps h and h / 2; their own error, of order h^2, is at most
    4/3 of the change between the two, and what is left after that of order h^4."""
    import torch
    for interleaved, d, rot in ((0, 32, 20), (1, 32, 32)):
        c = Case(A, 17, 5, 2, 2, d, rot, interleaved, "f32")
        dq, dk = torch.empty_like(c.q), torch.empty_like(c.k)
        dqw = torch.empty(d, device="cuda")
        A.norm_rope_bwd_t(c.shape(), c.norm, dev(c.table), dev(c.pos), c.q, c.k, c.gq, c.gk, dq, dk, dqw)
        x, g, w = host(c.q), host(c.gq), c.qw.astype(np.float64)
        _, _, most, most_w = N.backward(x, g, 2, w, np.float64(np.float32(EPS)), c.table, c.pos, rot, interleaved)

        def f(x, w):
            return (N.forward(x, 2, w, np.float64(np.float32(EPS)), c.table, c.pos, rot, interleaved)[0] * g).sum()

        def slope(i, j, h):
            if i < 0:
                up, down = w.copy(), w.copy()
                up[j] += h
                down[j] -= h
                return (f(x, up) - f(x, down)) / (2 * h)
            up, down = x.copy(), x.copy()
            up[i, j] += h
            down[i, j] -= h
            return (f(up, w) - f(down, w)) / (2 * h)

        for i, j in [(i, j) for i in range(-1, 5) for j in range(0, d, 5)]:
            rough, fine = slope(i, j, 2.0 ** -8), slope(i, j, 2.0 ** -9)
            got, bound = (host(dqw)[j], 32 * U * most_w[j]) if i < 0 else (host(dq)[i, j], 64 * U * most[i, j])
            assert abs(got - fine) <= bound + 4 / 3 * abs(rough - fine) + 1e-9, (i, j)


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strided_views(A, kind, offset):
    """Column blocks of wider tensors at aligned and unaligned offsets, positions from seq_len, q alone; what lies beside
    the blocks is left as it was."""
    import torch
    c = Case(A, 3, 50, 4, 2, 64, 64, 0, kind)
    pos = np.arange(50) % 13

    def wide(*blocks):
        t = torch.full((50, 600 + offset), 5.0, dtype=c.type, device="cuda")
        views = [t[:, offset + 300 * i:offset + 300 * i + b.shape[1]] for i, b in enumerate(blocks)]
        for v, b in zip(views, blocks):
            v.copy_(b)
        return (t, *views)

    _, q, k = wide(c.q, c.k)
    _, gq, gk = wide(c.gq, c.gk)
    out, qo, ko = wide(torch.zeros_like(c.q), torch.zeros_like(c.k))
    grads, dq, dk = wide(torch.zeros_like(c.q), torch.zeros_like(c.k))
    st = q.stride(0)
    shape = c.shape(13, q_row_stride=st, k_row_stride=st, q_out_row_stride=st, k_out_row_stride=st)
    A.norm_rope_t(shape, c.norm, dev(c.table), None, q, k, qo, ko)
    c.check_forward(qo, c.q, 4, c.qw, pos)
    c.check_forward(ko, c.k, 2, c.kw, pos)
    dqw = torch.empty(64, device="cuda")
    A.norm_rope_bwd_t(shape, c.norm, dev(c.table), None, q, k, gq, gk, dq, dk, dqw)
    c.check_backward(dq, dqw, c.q, c.gq, 4, c.qw, pos)
    c.check_backward(dk, None, c.k, c.gk, 2, c.kw, pos)
    for t in (out, grads):
        assert (t[:, :offset] == 5).all() and (t[:, offset + 256:offset + 300] == 5).all() and (t[:, offset + 428:] == 5).all()
    alone, daw, none = torch.empty_like(c.q), torch.empty_like(dqw), torch.full_like(dqw, 2.0)
    shape = c.shape(13, q_row_stride=st)
    A.norm_rope_t(shape, c.norm, dev(c.table), None, q, None, alone, None)
    c.check_forward(alone, c.q, 4, c.qw, pos)     # (aligned rows may go another way than unaligned ones: not the same bits)
    g = c.gq
    dw = wide(torch.zeros_like(c.q))[1]
    A.norm_rope_bwd_t(shape, c.norm, dev(c.table), None, q, None, g, None, dw, None, daw, none)
    c.check_backward(dw, daw, c.q, c.gq, 4, c.qw, pos)
    assert (none == 0).all()                      # the sum over no tokens


def test_without_weights_and_other_inputs(A):
    """Weights of None are ones; rows of zeros, of large and of small values; a value that is no number stays in its head."""
    import torch
    c = Case(A, 29, 6, 3, 2, 64, 64, 0, "f32")
    c.q[0] = 0
    c.q[1] *= 1e15
    c.q[2] *= 1e-15
    c.q[3, 70] = float("nan")
    c.q[4, 3] = float("inf")
    ones = np.ones(64, np.float32)
    out = torch.empty_like(c.q)
    A.norm_rope_t(c.shape(), A.HeadNorm.of(eps=EPS), dev(c.table), dev(c.pos), c.q, None, out, None)
    want, most = c.want(torch.nan_to_num(c.q, nan=0.0, posinf=0.0), 3, ones)
    good = np.ones((6, 3 * 64), bool)
    good[3, 64:128] = good[4, :64] = False
    got = host(out)
    assert (np.abs(got - want) <= 16 * U * most + 1e-37)[good].all()
    assert np.isnan(got[3, 64:128]).all() and np.isnan(got[4, 3])
    dq, dw = torch.empty_like(c.q), torch.empty(64, device="cuda")
    keep = [0, 1, 2, 5]
    q, g, pos = c.q[keep].contiguous(), c.gq[keep].contiguous(), c.pos[keep]
    c.tokens = 4
    A.norm_rope_bwd_t(c.shape(), A.HeadNorm.of(eps=EPS), dev(c.table), dev(pos), q, None, g, None, dq[:4], None, dw)
    c.check_backward(dq[:4], dw, q, g, 3, ones, pos)


def test_no_tokens(A):
    import torch
    c = Case(A, 1, 2, 2, 2, 32, 32, 0, "f32")
    c.tokens = 0
    out, dw = torch.full_like(c.q, 7.0), torch.full((32,), 7.0, device="cuda")
    kept = dw.clone()
    A.norm_rope_t(c.shape(1), c.norm, dev(c.table), None, c.q, c.k, out, out)
    A.norm_rope_bwd_t(c.shape(1), c.norm, dev(c.table), None, c.q, c.k, c.gq, c.gk, out, out, dw, None)
    A.norm_rope_bwd_t(c.shape(1), c.norm, dev(c.table), None, c.q, c.k, c.gq, c.gk, out, out, kept, None, accumulate=True)
    assert (out == 7).all() and (dw == 0).all() and (kept == 7).all()


@pytest.mark.parametrize("kind,cache", [("f32", "f32"), ("bf16", "bf16"), ("f32", "int8")])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", SHAPES)
def test_norm_rope_append(A, tokens, heads, kv_heads, d, rot, interleaved, kind, cache):
    import torch
    c = Case(A, tokens + 2 * d, tokens, heads, kv_heads, d, rot, interleaved, kind)
    rows, width = tokens * 2 + 5, kv_heads * d
    stride = width + 32
    dt = torch.int8 if cache == "int8" else c.type
    kc, vc = (torch.full((rows, stride), 9, dtype=dt, device="cuda")[:, :width] for _ in range(2))
    ks, vs = ((torch.full((rows, kv_heads), 9.0, device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
    r = np.random.RandomState(tokens)
    slots = r.permutation(rows)[:tokens].astype(np.int64)
    skip = r.rand(tokens) < 0.2
    slots[skip] = r.choice([-1, rows, 2 ** 40], skip.sum())
    pos = c.pos.copy()
    pos[skip] = 10 ** 6                           # (not reported: the token has no slot)
    device_error(A)
    out = torch.full_like(c.q, float("nan"))
    A.norm_rope_append_t(c.shape(), c.norm, A.PageCache.of(kc, vc, ks, vs), dev(c.table), dev(pos), dev(slots), c.q, c.k, c.v, out)
    assert device_error(A) == 0
    c.check_forward(out, c.q, heads, c.qw, np.minimum(pos, c.max_pos - 1))
    there = np.flatnonzero(~skip)
    left = np.setdiff1d(np.arange(rows), slots[there])
    assert (kc[left] == 9).all() and (vc[left] == 9).all()
    assert (kc._base[:, width:] == 9).all() and (vc._base[:, width:] == 9).all()
    if not len(there):
        return
    at, rows_there = dev(slots[there]), dev(there)
    if cache != "int8":
        c.pos, keep = c.pos[there], c.pos
        c.check_forward(kc[at], c.k[rows_there], kv_heads, c.kw)
        c.pos = keep
        assert torch.equal(vc[at], c.v[rows_there])
        return
    codes, scales = A.quantize_int8_t(c.v, kv_heads)
    assert torch.equal(vc[at], codes[rows_there]) and torch.equal(vs[at], scales[rows_there])
    want, _ = N.forward(host(c.k)[there], kv_heads, c.kw.astype(np.float64), np.float64(np.float32(EPS)), c.table, c.pos[there], rot, interleaved)
    want = want.reshape(len(there), kv_heads, d)
    scale = host(ks[at])
    np.testing.assert_allclose(scale, np.abs(want).max(-1) / 127, rtol=2.0 ** -18)
    got = host(kc[at]).reshape(want.shape)
    assert (np.abs(got * scale[..., None] - want) <= scale[..., None] * (0.5 + 127 * 2.0 ** -16)).all()
    assert (ks[dev(left)] == 9).all() and (vs[dev(left)] == 9).all()


def test_position_outside_the_table(A):
    import torch
    c = Case(A, 1, 4, 2, 2, 32, 32, 0, "f32", max_pos=10)
    out, ko = torch.empty_like(c.q), torch.empty_like(c.k)
    device_error(A)
    for pos in ([0, 10, 1, 9], [0, 3, -1, 9]):
        A.norm_rope_t(c.shape(), c.norm, dev(c.table), dev(np.array(pos, np.int32)), c.q, c.k, out, ko)
        assert device_error(A) == 0x701
        c.check_forward(out, c.q, 2, c.qw, np.clip(pos, 0, 9))
        A.norm_rope_bwd_t(c.shape(), c.norm, dev(c.table), dev(np.array(pos, np.int32)), c.q, c.k, c.gq, c.gk, out, ko)
        assert device_error(A) == 0x701
        c.check_backward(out, None, c.q, c.gq, 2, c.qw, np.clip(pos, 0, 9))
    assert device_error(A) == 0


def test_captured_with_two_streams(A):
    """Forward and gradients captured together and replayed on new inputs, another call running beside on a stream of its
    own with a workspace of its own: the bits of plain calls."""
    import torch
    a, b = (Case(A, s, 200, 8, 4, 64, 64, 0, "bf16") for s in (41, 42))
    outs = []
    for c in (a, b):
        o = [torch.zeros_like(c.q), torch.zeros_like(c.k), torch.zeros_like(c.q), torch.zeros_like(c.k),
             torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")]
        w = torch.empty(A.norm_rope_bwd_workspace_bytes(c.shape()), dtype=torch.uint8, device="cuda")
        outs.append((c, o, w, dev(c.table), dev(c.pos)))

    def step(c, o, w, table, pos):
        A.norm_rope_t(c.shape(), c.norm, table, pos, c.q, c.k, o[0], o[1])
        A.norm_rope_bwd_t(c.shape(), c.norm, table, pos, c.q, c.k, c.gq, c.gk, o[2], o[3], o[4], o[5], workspace=w)

    want = []
    for x in outs:
        step(*x)
        torch.cuda.synchronize()
        want.append([t.clone() for t in x[1]])
        for t in x[1]:
            t.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(*outs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        g.replay()
        with torch.cuda.stream(side):
            step(*outs[1])
    torch.cuda.synchronize()
    for w, x in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(w, x[1]))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved,rot", [(0, 32), (1, 32), (0, 2)])
def test_weight_gradients_do_not_lose_bits_with_the_tokens(A, interleaved, rot, kind):
    """2^17 tokens of eight heads, all one row, so that every rounding of a sum that is kept in fp32 falls on the same side:
    a term is off by at most 13 u as above, chains of at most 4 terms in fp32 add 4 u, the result's rounding 1 u, however
    many tokens there are."""
    import torch
    tokens, heads, d = 2 ** 17, 8, 128
    dt = torch.bfloat16 if kind == "bf16" else torch.float32
    table = np.zeros((1, rot // 2, 2), np.float32)
    table[..., 0] = 1.0
    x = dev(1 + synth.uniform(71, d), dt)
    g = dev(1 + synth.uniform(72, d), dt)
    q, dq = x.repeat(tokens, heads), g.repeat(tokens, heads)
    dw = torch.empty(d, device="cuda")
    shape = A.RopeShape(tokens, tokens, heads, heads, d, rot, interleaved, tokens, 0, 0, 0, 0, 0)
    A.norm_rope_bwd_t(shape, A.HeadNorm.of(eps=EPS), dev(np.repeat(table, tokens, 0)), None, q, None, dq, None, dq, None, dw)
    x, g = host(x), host(g)
    want = tokens * heads * g * x / np.sqrt((x * x).mean() + np.float64(np.float32(EPS)))
    assert (np.abs(host(dw) - want) <= (13 + 4 + 1) * U * want).all(), np.abs(host(dw) / want - 1).max() / U


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved,rot", [(0, 64), (1, 64), (0, 26)])
@pytest.mark.parametrize("seq_len", [13, 700, 4999, 9000])
def test_positions_of_many_tokens(A, seq_len, interleaved, rot, kind):
    """Positions by seq_len over several of a group's tokens: sequences shorter than the stride between them, longer, and
    longer than the tokens there are."""
    import torch
    tokens = 5003
    c = Case(A, seq_len + rot, tokens, 12, 4, 64, rot, interleaved, kind, max_pos=seq_len)
    pos = np.arange(tokens) % seq_len
    table = dev(c.table)
    qo, ko = torch.empty_like(c.q), torch.empty_like(c.k)
    device_error(A)
    A.norm_rope_t(c.shape(seq_len), c.norm, table, None, c.q, c.k, qo, ko)
    c.check_forward(qo, c.q, 12, c.qw, pos)
    c.check_forward(ko, c.k, 4, c.kw, pos)
    dqw, dkw = (torch.empty(64, device="cuda") for _ in range(2))
    A.norm_rope_bwd_t(c.shape(seq_len), c.norm, table, None, c.q, c.k, c.gq, c.gk, qo, ko, dqw, dkw)
    c.check_backward(qo, dqw, c.q, c.gq, 12, c.qw, pos)
    c.check_backward(ko, dkw, c.k, c.gk, 4, c.kw, pos)
    assert device_error(A) == 0
