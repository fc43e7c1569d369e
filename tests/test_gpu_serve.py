"""The serving operators over a paged cache and the rotary embedding on the GPU, against 64-bit forms (serve_ref.py).

Tolerances, from the arithmetic:
  pages     whole numbers: equal.
  rope      fp32: two products and a sum, 2^-23 (|a| + |b|) per element; bf16: half a unit in the last place of the
            result, 2^-8 of it at most (2^-9 and the fp32 error before it).
  prefix    a score is off by at most delta = 2^-21 (1 + scale sum|q k|) (products off by 2^-22 where an operand is
            split in parts, fp32 sums, the exponential's argument), so a probability by the factor 1 +- 2 delta and
            the output by 4 delta sum p|v| (numerator and denominator); for bf16 2^-8 sum p|v| more, the most that rounding
            the output can take (probabilities rounded to bf16 err at random, so over many keys they stay far below it;
            over few keys the kernel keeps what the rounding drops).  A probability under 2^-126, the smallest normal
            fp32 number, may count as 0: 2^-126 max|v| more for each key.  lse: delta + 2^-22 |lse|."""
import ctypes

import numpy as np
import pytest

import serve_ref as R
import synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A(cuda):
    import attn_b200
    return attn_b200


def dev(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def device_error(A):
    code = ctypes.c_int()
    A.check(A.lib.attn_device_error(0, ctypes.byref(code)))
    return code.value


# ---------------------------------------------------------------------------
# page plan
# ---------------------------------------------------------------------------
def plan_case(seed, n, page, max_len, most_new, ended=0.0, room=1.0, extra_columns=0):
    r = np.random.RandomState(seed)
    lens = r.randint(0, max_len + 1, n).astype(np.int32)
    new = r.randint(0, most_new + 1, n).astype(np.int32)
    new[r.rand(n) < ended] = -1
    max_pages = max(1, -(-(max_len + most_new) // page)) + extra_columns
    ids = r.permutation(n * max_pages + 5).astype(np.int32)
    table = np.full((n, max_pages), -7, np.int32)
    at = 0
    for s in range(n):
        k = -(-int(lens[s]) // page)
        table[s, :k] = ids[at:at + k]
        at += k
    need = sum(-(-(int(l) + int(k)) // page) - -(-int(l) // page) for l, k in zip(lens, new) if k > 0)
    count = min(len(ids) - at, int(need * room + 0.5))
    free = np.full(len(ids), -9, np.int32)
    free[:count] = ids[at:at + count]
    return lens, new, r.randint(0, 100, n).astype(np.int32), free, count, table


def run_plan(A, case, page, max_tokens, base=True):
    lens, new, pos_base, free, count, table = case
    shape = A.PageShape(len(lens), page, table.shape[1], max_tokens, len(free), 0)
    out = A.page_outputs(shape)
    for t in out.values():
        t.fill_(-99)
    d_free, d_table = dev(free), dev(table)
    A.page_plan_t(shape, dev(lens), dev(new), d_free, dev(np.array([count], np.int32)), d_table, out,
                  pos_base=dev(pos_base) if base else None)
    got = {k: v.cpu().numpy() for k, v in out.items()}
    return got, d_table.cpu().numpy(), d_free.cpu().numpy()


def check_plan(A, case, page, max_tokens, base=True):
    lens, new, pos_base, free, count, table = case
    got, g_table, g_free = run_plan(A, case, page, max_tokens, base)
    want = R.page_plan(lens, new, pos_base if base else 0 * pos_base, free, count, table, page, max_tokens)
    for name, w in zip(("lens", "cu_new", "slot_map", "positions", "token_seq", "counts"), want):
        np.testing.assert_array_equal(got[name], w, err_msg=name)
    np.testing.assert_array_equal(g_table, want[6])
    np.testing.assert_array_equal(g_free, want[7])


@pytest.mark.parametrize("n,page,max_len,most_new,ended,room", [
    (1, 16, 0, 1, 0.0, 1.0), (1, 1, 3, 2, 0.0, 1.0), (7, 16, 100, 1, 0.0, 1.0), (64, 8, 500, 4, 0.3, 0.3),
    (33, 1024, 3000, 2047, 0.2, 0.5), (1025, 32, 300, 3, 0.1, 0.9), (300, 64, 0, 700, 0.0, 0.6), (40, 2, 50, 9, 0.5, 0.0),
])
@pytest.mark.parametrize("slack", [0, 37, -5])
def test_page_plan(A, n, page, max_len, most_new, ended, room, slack):
    """slack: token rows beyond the tokens there are, or too few of them."""
    case = plan_case(n + page, n, page, max_len, most_new, ended, room)
    max_tokens = max(0, int(np.maximum(case[1], 0).sum()) + slack)
    check_plan(A, case, page, max_tokens, base=slack != 37)


def test_page_plan_no_requests_and_no_rows(A):
    case = plan_case(3, 5, 16, 40, 0)
    check_plan(A, case, 16, 0)
    shape = A.PageShape(0, 16, 4, 8, 2, 0)
    out = A.page_outputs(shape)
    free, count = dev(np.array([4, 5], np.int32)), dev(np.array([2], np.int32))
    A.page_plan_t(shape, free, free, free, count, free, out)
    assert out["counts"].tolist() == [2, 0, 0, 0] and out["cu_new"].tolist() == [0]
    assert out["slot_map"].tolist() == [-1] * 8 and out["token_seq"].tolist() == [-1] * 8


def test_page_plan_lengths_past_the_table(A):
    """A request past its table's width is refused, lengths outside [0, width] are clamped, and sums saturate."""
    page, table = 4, np.arange(12, dtype=np.int32).reshape(4, 3)
    lens = np.array([12, 11, 99, -3], np.int32)
    new = np.array([1, 1, 0, 2], np.int32)
    case = (lens, new, np.zeros(4, np.int32), np.array([20, 21, 22], np.int32), 3, table)
    check_plan(A, case, page, 16)
    big = np.full(4, 2 ** 30, np.int32)
    got, _, _ = run_plan(A, (lens, big, np.zeros(4, np.int32), case[3], 3, table), page, 16)
    assert got["cu_new"].tolist() == [0, 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
    assert got["counts"].tolist() == [3, 2 ** 31 - 1, 4, 0] and (got["slot_map"] == -1).all()


def test_page_plan_row_stride_and_steps_in_turn(A):
    """Ten steps fed from one another's outputs, with a table inside a wider one, keep every page owned once."""
    import torch
    r = np.random.RandomState(5)
    n, page, max_pages, total = 12, 8, 6, 50
    wide = torch.full((n, max_pages + 3), -1, dtype=torch.int32, device="cuda")
    shape = A.PageShape(n, page, max_pages, 200, total, max_pages + 3)
    free = dev(r.permutation(total).astype(np.int32))
    lens, count = torch.zeros(n, dtype=torch.int32, device="cuda"), dev(np.array([total], np.int32))
    outs = [A.page_outputs(shape) for _ in range(2)]
    for step in range(10):
        new = r.randint(-1, 12, n).astype(np.int32)
        before = [x.cpu().numpy() for x in (lens, free, wide, count)]
        out = A.page_plan_t(shape, lens, dev(new), free, count, wide, outs[step % 2])
        want = R.page_plan(before[0], new, np.zeros(n, np.int32), before[1], int(before[3][0]), before[2][:, :max_pages], page, 200)
        np.testing.assert_array_equal(out["slot_map"].cpu().numpy(), want[2])
        np.testing.assert_array_equal(wide[:, :max_pages].cpu().numpy(), want[6])
        assert (wide[:, max_pages:] == -1).all()
        lens, count = out["lens"], out["counts"][:1]
        held = [int(wide[s, j]) for s in range(n) for j in range(-(-int(lens[s]) // page))]
        assert sorted(held + free[:int(count)].tolist()) == list(range(total))


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def rope_case(A, seed, tokens, heads, kv_heads, d, rot, kind, max_pos=97):
    import torch
    dt = torch.bfloat16 if kind == "bf16" else torch.float32
    q, k, v = (dev(synth.normal(seed + i, (tokens, h * d)), dt) for i, h in enumerate((heads, kv_heads, kv_heads)))
    pos = np.random.RandomState(seed).randint(0, max_pos, tokens).astype(np.int32)
    table = R.rope_table(rot, max_pos).astype(np.float32) if rot else np.zeros((max_pos, 0, 2), np.float32)
    return q, k, v, pos, table


def rope_close(got, x, want, heads, rot, kind):
    """got, x: tensors (output and input); want float64."""
    g = got.float().cpu().numpy().astype(np.float64)
    if kind == "bf16":
        tol = 2.0 ** -8 * np.abs(want) + 1e-30
        tol = np.maximum(tol, 2.0 ** -22 * np.abs(x.float().cpu().numpy()).max())
    else:
        tol = np.full_like(want, 2.0 ** -23 * 2 * float(x.abs().max()))
    assert (np.abs(g - want) <= tol).all(), np.abs(g - want).max()


ROPE = [(1, 1, 1, 32, 32), (5, 3, 1, 64, 26), (37, 12, 12, 128, 128), (130, 16, 4, 96, 48), (64, 8, 8, 64, 0), (9, 5, 5, 32, 2),
        (300, 32, 8, 128, 64), (2, 1, 1, 96, 96)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", ROPE)
def test_rope(A, tokens, heads, kv_heads, d, rot, interleaved, kind):
    import torch
    q, k, _, pos, table = rope_case(A, tokens + d, tokens, heads, kv_heads, d, rot, kind)
    shape = A.RopeShape(tokens, 0, heads, kv_heads, d, rot, interleaved, len(table), 0, 0, 0, 0, 0)
    for transpose in (False, True):
        q_out, k_out = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
        A.rope_t(shape, dev(table), dev(pos), q, k, q_out, k_out, transpose=transpose)
        for x, got, h in ((q, q_out, heads), (k, k_out, kv_heads)):
            rope_close(got, x, R.rope(x.float().cpu().numpy(), h, table, pos, rot, interleaved, transpose), h, rot, kind)
    # in place, the same bits
    qi, ki = q.clone(), k.clone()
    A.rope_t(shape, dev(table), dev(pos), qi, ki, qi, ki, transpose=True)
    assert torch.equal(qi, q_out) and torch.equal(ki, k_out)


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rope_strided_views(A, kind, offset):
    """Column blocks of wider tensors, at aligned and unaligned offsets; positions from seq_len; q alone."""
    import torch
    tokens, heads, kv_heads, d, rot = 50, 4, 2, 64, 64
    q, k, _, _, table = rope_case(A, 3, tokens, heads, kv_heads, d, rot, kind)
    wide = torch.zeros((tokens, 600 + offset), dtype=q.dtype, device="cuda")
    qv, kv = wide[:, offset:offset + heads * d], wide[:, 300 + offset:300 + offset + kv_heads * d]
    qv.copy_(q)
    kv.copy_(k)
    out = torch.full((tokens, 700), 5.0, dtype=q.dtype, device="cuda")
    qo, ko = out[:, offset:offset + heads * d], out[:, 400:400 + kv_heads * d]
    shape = A.RopeShape(tokens, 13, heads, kv_heads, d, rot, 0, len(table), wide.stride(0), wide.stride(0), 0, 700, 700)
    A.rope_t(shape, dev(table), None, qv, kv, qo, ko)
    pos = np.arange(tokens) % 13
    rope_close(qo, q, R.rope(q.float().cpu().numpy(), heads, table, pos, rot, 0), heads, rot, kind)
    rope_close(ko, k, R.rope(k.float().cpu().numpy(), kv_heads, table, pos, rot, 0), kv_heads, rot, kind)
    assert (out[:, offset + heads * d:400] == 5).all() and (out[:, 400 + kv_heads * d:] == 5).all()
    alone = torch.empty_like(q)
    shape.q_out_row_stride = 0
    A.rope_t(shape, dev(table), None, qv, None, alone, None)
    assert torch.equal(alone, qo)


def test_rope_gradient_against_differences(A):
    """<g, J e_i> by central differences of the forward equals the transposed rotation of g: the map is linear, so a
    difference over a step of 1 is exact up to rounding (2^-23 of the largest output, over 2 outputs)."""
    import torch
    tokens, heads, d, rot = 6, 2, 32, 20
    for interleaved in (0, 1):
        q, k, _, pos, table = rope_case(A, 11, tokens, heads, heads, d, rot, "f32")
        table = (table * 1.3).astype(np.float32)          # a magnitude: the transpose is not the inverse
        shape = A.RopeShape(tokens, 0, heads, heads, d, rot, interleaved, len(table), 0, 0, 0, 0, 0)
        g = dev(synth.normal(12, (tokens, heads * d)))
        grad = torch.empty_like(g)
        A.rope_t(shape, dev(table), dev(pos), g, None, grad, None, transpose=True)
        for col in range(0, heads * d, 3):
            up, down = q.clone(), q.clone()
            up[:, col] += 0.5
            down[:, col] -= 0.5
            outs = []
            for x in (up, down):
                y = torch.empty_like(x)
                A.rope_t(shape, dev(table), dev(pos), x, None, y, None)
                outs.append(y.double())
            diff = ((outs[0] - outs[1]) * g.double()).sum(1)
            assert (diff - grad[:, col].double()).abs().max() < 2.0 ** -21 * 1.3 * float(q.abs().max() * g.abs().max())


def test_rope_position_outside_the_table(A):
    import torch
    q, k, _, pos, table = rope_case(A, 1, 4, 2, 2, 32, 32, "f32", max_pos=10)
    pos = np.array([0, 10, -1, 9], np.int32)
    shape = A.RopeShape(4, 0, 2, 2, 32, 32, 0, 10, 0, 0, 0, 0, 0)
    out, ko = torch.empty_like(q), torch.empty_like(k)
    device_error(A)
    A.rope_t(shape, dev(table), dev(pos), q, k, out, ko)
    assert device_error(A) == 0x701
    rope_close(out, q, R.rope(q.cpu().numpy(), 2, table, np.array([0, 9, 0, 9]), 32, 0), 2, 32, "f32")
    assert device_error(A) == 0


@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "ramp"])
@pytest.mark.parametrize("rot", [4, 64, 128])
def test_rope_table(A, scaling, rot):
    """Angles in fp64, so an entry is off by fp32 rounding (2^-24) and the fp64 angle's error (position x 2^-50)."""
    number = {"plain": A.ROPE_PLAIN, "linear": A.ROPE_LINEAR, "base": A.ROPE_BASE, "ramp": A.ROPE_RAMP}[scaling]
    cfg = A.RopeConfig(rot, 40007, number, 4096, 10000.0, 8.0, 32.0, 1.0, 1.25)
    got = A.rope_table_t(cfg).cpu().numpy()
    want = R.rope_table(rot, 40007, 10000.0, scaling, 8.0, 4096, 32.0, 1.0, 1.25)
    assert np.abs(got - want).max() < 1.25 * (2.0 ** -24 + 40007 * 2.0 ** -50) + 2.0 ** -24


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind,cache", [("f32", "f32"), ("bf16", "bf16"), ("f32", "int8")])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", ROPE)
def test_rope_append(A, tokens, heads, kv_heads, d, rot, interleaved, kind, cache):
    """K and V land in their slots and nowhere else; an INT8 cache holds what the quantiser makes of the turned rows."""
    import torch
    q, k, v, pos, table = rope_case(A, tokens + 3 * d, tokens, heads, kv_heads, d, rot, kind)
    rows, stride = 2 * tokens + 11, kv_heads * d + 32
    dt = torch.int8 if cache == "int8" else q.dtype
    kc, vc = (torch.full((rows, stride), 77, dtype=dt, device="cuda")[:, :kv_heads * d] for _ in range(2))
    ks, vs = ((torch.full((rows, kv_heads), -1.0, device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
    slots = np.random.RandomState(tokens).permutation(rows)[:tokens].astype(np.int64)
    if tokens > 3:
        slots[1], slots[2] = -1, rows                     # outside the cache: not written
    shape = A.RopeShape(tokens, 0, heads, kv_heads, d, rot, interleaved, len(table), 0, 0, 0, 0, 0)
    q_out, k_want = torch.empty_like(q), torch.empty_like(k)
    paged = A.PageCache.of(kc, vc, ks, vs)
    A.rope_append_t(shape, paged, dev(table), dev(pos), dev(slots), q, k, v, q_out)
    rope_close(q_out, q, R.rope(q.float().cpu().numpy(), heads, table, pos, rot, interleaved), heads, rot, kind)
    A.rope_t(shape, dev(table), dev(pos), q, k, torch.empty_like(q), k_want)
    rope_close(k_want, k, R.rope(k.float().cpu().numpy(), kv_heads, table, pos, rot, interleaved), kv_heads, rot, kind)
    keep = (slots >= 0) & (slots < rows)
    at = dev(slots[keep])
    mask = torch.ones(rows, dtype=torch.bool, device="cuda")
    mask[at] = False
    for c, s, x in ((kc, ks, k_want), (vc, vs, v)):
        if cache == "int8":
            codes, scales = A.quantize_int8_t(x, kv_heads)
            assert torch.equal(c[at], codes[dev(keep)]) and torch.equal(s[at], scales[dev(keep)])
            assert (s[mask] == -1).all()
        else:
            assert torch.equal(c[at], x[dev(keep)])
        assert (c[mask] == 77).all()


@pytest.mark.parametrize("kind,cache", [("f32", "f32"), ("bf16", "bf16"), ("f32", "int8")])
@pytest.mark.parametrize("rot", [32, 6])
def test_rope_append_after_a_refusal(A, kind, cache, rot):
    """A request at the end of its table is refused one token more, whose position is past a rotary table of the cache's
    length: no error is reported, and the other requests' tokens go where they should.  A token that has a slot and
    such a position is reported."""
    import torch
    page, d, heads = 4, 32, 2
    lens, new = np.array([8, 2, 0, 7], np.int32), np.array([2, 1, 3, 1], np.int32)
    table = np.array([[0, 1], [2, -1], [-1, -1], [3, 4]], np.int32)
    shape = A.PageShape(4, page, 2, 8, 8, 0)
    plan = A.page_outputs(shape)
    A.page_plan_t(shape, dev(lens), dev(new), dev(np.array([5, 6, 7, 0, 0, 0, 0, 0], np.int32)), dev(np.array([3], np.int32)), dev(table), plan)
    slots, positions = plan["slot_map"].cpu().numpy(), plan["positions"].cpu().numpy()
    assert slots.tolist() == [-1, -1, 10, 28, 29, 30, 19, -1] and positions.tolist() == [8, 9, 2, 0, 1, 2, 7, 0]
    q, k, v, _, angles = rope_case(A, 5, 8, heads, heads, d, rot, kind, max_pos=8)
    dt = torch.int8 if cache == "int8" else q.dtype
    kc, vc = (torch.full((32, heads * d), 77, dtype=dt, device="cuda") for _ in range(2))
    ks, vs = ((torch.full((32, heads), -1.0, device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
    rshape = A.RopeShape(8, 0, heads, heads, d, rot, 0, 8, 0, 0, 0, 0, 0)
    paged, q_out = A.PageCache.of(kc, vc, ks, vs), torch.empty_like(q)
    device_error(A)
    A.rope_append_t(rshape, paged, dev(angles), plan["positions"], plan["slot_map"], q, k, v, q_out)
    assert device_error(A) == 0
    at = slots[slots >= 0]
    want = R.rope(k.float().cpu().numpy(), heads, angles, np.minimum(positions, 7), rot, 0)[slots >= 0]
    got = kc[dev(at)].float().cpu().numpy().astype(np.float64)
    if cache == "int8":
        step = np.repeat(ks[dev(at)].cpu().numpy().astype(np.float64), d, 1)
        assert (np.abs(got * step - want) <= 0.5 * step * (1 + 2.0 ** -12)).all()      # half a code, and rounding
        assert torch.equal(vc[dev(at)], A.quantize_int8_t(v, heads)[0][dev(slots >= 0)])
    else:
        rope_close(kc[dev(at)], k, want, heads, rot, kind)
        assert torch.equal(vc[dev(at)], v[dev(slots >= 0)])
    others = np.setdiff1d(np.arange(32), at)
    assert (kc[dev(others)] == 77).all() and (vc[dev(others)] == 77).all()
    plan["positions"][3] = 8
    A.rope_append_t(rshape, paged, dev(angles), plan["positions"], plan["slot_map"], q, k, v, q_out)
    assert device_error(A) == 0x701


# ---------------------------------------------------------------------------
# shared-prefix decode
# ---------------------------------------------------------------------------
def torch_equal(a, b):
    import torch
    return torch.equal(a, b)


class PrefixCase:
    """Random tables over a cache whose unused rows are NaN (INT8: extreme scales) and whose unused table entries lie
    outside the cache."""

    def __init__(self, A, seed, kind, d, heads, kv_heads, page, group_sizes, prefix_lens, lens, q_std=1.0, extra_stride=0, no_group=0):
        import torch
        r = np.random.RandomState(seed)
        self.A, self.kind, self.d, self.heads, self.kv_heads, self.page = A, kind, d, heads, kv_heads, page
        self.n = n = sum(group_sizes) + no_group
        assert len(lens) == n
        self.begin = np.concatenate([[0], np.cumsum(group_sizes)]).astype(np.int32)
        self.plens, self.lens = np.array(prefix_lens, np.int32), np.array(lens, np.int32)
        mp, mo = (max([1] + [-(-int(x) // page) for x in v]) for v in (prefix_lens, lens))
        need = sum(-(-int(x) // page) for x in list(prefix_lens) + list(lens))
        n_pages = need + 4
        ids = r.permutation(n_pages)
        self.ptable, self.table = np.full((max(1, len(group_sizes)), mp), 2 ** 30, np.int32), np.full((n, mo), -5, np.int32)
        at, used = 0, np.zeros(n_pages * page, bool)
        for table, ls in ((self.ptable, prefix_lens), (self.table, lens)):
            for i, x in enumerate(ls):
                for j in range(-(-int(x) // page)):
                    table[i, j] = ids[at]
                    used[ids[at] * page:ids[at] * page + min(page, int(x) - j * page)] = True
                    at += 1
        rows, w = n_pages * page, kv_heads * d
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.float32}[kind]
        self.q = dev(synth.normal(seed + 1, (n, heads * d), 0, q_std), dt)
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
        self.shape = A.PrefixShape(n, len(group_sizes), heads, kv_heads, d, A.BF16 if kind == "bf16" else A.F32, page, mp, mo,
                                   max([0] + list(prefix_lens)), max([0] + list(lens)), 0, 0, 0.0)

    def run(self, q=None, out=None, workspace="own", lse=True):
        import torch
        A = self.A
        q = self.q if q is None else q
        out = torch.full_like(self.q, float("nan")) if out is None else out
        ls = torch.full((self.n, self.heads), float("nan"), device="cuda") if lse else None
        ws = None
        if workspace == "own":
            ws = torch.full((A.prefix_decode_workspace_bytes(self.shape, self.cache),), 0xff, dtype=torch.uint8, device="cuda")
        groups = (dev(self.begin), dev(self.ptable), dev(self.plens)) if self.shape.n_groups else (None, None, None)
        A.prefix_decode_t(self.shape, self.cache, q, *groups, dev(self.table), dev(self.lens), out, lse=ls, workspace=ws)
        return out, ls

    def rows_of(self, s):
        rows = []
        for g in range(len(self.plens)):
            if self.begin[g] <= s < self.begin[g + 1]:
                rows += [int(self.ptable[g, t // self.page]) * self.page + t % self.page for t in range(self.plens[g])]
        return rows + [int(self.table[s, t // self.page]) * self.page + t % self.page for t in range(self.lens[s])]

    def check(self, out, lse, only=None, absent=None):
        scale = 1.0 / np.sqrt(self.d)
        q64 = self.q.float().cpu().numpy().astype(np.float64)
        out, lse = out.float().cpu().numpy().astype(np.float64), None if lse is None else lse.cpu().numpy().astype(np.float64)
        for s in range(self.n) if only is None else only:
            rows = [x for x in self.rows_of(s) if absent is None or x not in absent]
            want, wl, weight, reach = R.prefix_decode(q64[s], self.k64[rows], self.v64[rows], self.heads, self.kv_heads, scale)
            delta = 2.0 ** -21 * (1 + reach)
            tol = 4 * np.repeat(delta, self.d) * weight + (2.0 ** -8 * weight if self.kind == "bf16" else 0)
            tol = tol + len(rows) * 2.0 ** -126 * (np.abs(self.v64[rows]).max() if rows else 0)
            assert (np.abs(out[s] - want) <= tol).all(), (s, np.nanmax(np.abs(out[s] - want) / np.maximum(tol, 1e-300)))
            if lse is not None:
                finite = np.isfinite(wl)
                assert np.array_equal(lse[s][~finite], wl[~finite])
                assert (np.abs(lse[s][finite] - wl[finite]) <= (delta + 2.0 ** -22 * np.abs(wl))[finite]).all(), s


KINDS = ["f32", "bf16", "int8"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,heads,kv_heads,page", [(32, 4, 4, 16), (64, 6, 2, 8), (96, 3, 3, 32), (128, 8, 1, 64), (64, 2, 2, 1), (128, 4, 4, 1024)])
def test_prefix_small(A, kind, d, heads, kv_heads, page):
    """Lengths 0 and 1, tiles' edges, empty prefixes, requests of no group, a request with no rows."""
    c = PrefixCase(A, d + heads, kind, d, heads, kv_heads, page, [3, 2, 4], [129, 0, 1], [0, 1, 77, 0, 33, 128, 64, 0, 2, 0, 5], no_group=2)
    out, lse = c.run()
    c.check(out, lse)
    assert (out[3] == 0).all() and (out[9] == 0).all() and (lse[9] == -float("inf")).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,plen", [(1, 1), (2, 300), (17, 1000), (33, 127), (65, 513), (130, 260)])
def test_prefix_group_sizes(A, kind, n, plen):
    """One group of n requests: one tile of query rows, several, ragged ones."""
    r = np.random.RandomState(n)
    c = PrefixCase(A, n, kind, 64, 4, 2, 16, [n], [plen], r.randint(0, 40, n))
    c.check(*c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("ratio", [1, 2, 3, 8, 16])
def test_prefix_shared_heads(A, kind, d, ratio):
    c = PrefixCase(A, d + ratio, kind, d, 2 * ratio, 2, 16, [5, 9], [200, 70], np.random.RandomState(ratio).randint(0, 150, 14))
    c.check(*c.run())


@pytest.mark.parametrize("d,heads,kv_heads,page", [(64, 8, 2, 16), (128, 8, 2, 64), (128, 4, 4, 4), (64, 16, 1, 8), (128, 16, 1, 128), (64, 4, 4, 1024)])
@pytest.mark.parametrize("sizes,plens", [([70], [900]), ([33, 90], [385, 128]), ([2, 64, 1], [1, 2000, 127])])
def test_prefix_tiles(A, d, heads, kv_heads, page, sizes, plens):
    """bf16 groups of many query rows (the tensor-core tiles): blocks of 256 rows and of fewer than 128, steps that end
    inside a tile, pages below and above a tile's rows."""
    lens = np.random.RandomState(d + page).randint(0, 30, sum(sizes))
    c = PrefixCase(A, d + sum(sizes), "bf16", d, heads, kv_heads, page, sizes, plens, lens)
    out, lse = c.run()
    c.check(out, lse)
    again, l2 = c.run()
    assert torch_equal(again, out) and torch_equal(l2, lse)


@pytest.mark.parametrize("d,heads,kv_heads", [(32, 4, 4), (64, 4, 4), (96, 6, 2), (128, 4, 2)])
@pytest.mark.parametrize("n,plen", [(3, 50), (12, 700), (20, 3), (40, 9), (70, 900), (140, 65)])
def test_prefix_bf16_error_is_the_outputs_rounding(A, d, heads, kv_heads, n, plen):
    """The same precision whatever the group's size: rounding the output (2^-8 of it), a probability's second part (2^-17 of
    it) and the scores (4 delta) are all there is between a bf16 result and the 64-bit one."""
    c = PrefixCase(A, d + n, "bf16", d, heads, kv_heads, 16, [n], [plen], np.random.RandomState(n).randint(0, 20, n))
    out, _ = c.run()
    for s in range(0, n, 3):
        rows = c.rows_of(s)
        want, _, weight, reach = R.prefix_decode(c.q[s].double().cpu().numpy(), c.k64[rows], c.v64[rows], heads, kv_heads, 1 / np.sqrt(d))
        tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -17 + 4 * 2.0 ** -21 * (1 + np.repeat(reach, d))) * weight
        err = np.abs(out[s].double().cpu().numpy() - want)
        assert (err <= tol).all(), (s, (err / tol).max())


def test_prefix_tiles_bad_page(A):
    """A page outside the cache in the middle of a tile's keys: its rows are absent, and nothing is read there."""
    c = PrefixCase(A, 21, "bf16", 128, 4, 1, 16, [40], [600], [3] * 40)
    lost = set(range(int(c.ptable[0, 20]) * 16, int(c.ptable[0, 20]) * 16 + 16))
    c.ptable = c.ptable.copy()
    c.ptable[0, 20], keep = 2 ** 20, c.ptable[0, 20]
    out, lse = c.run()
    assert device_error(A) == 0x702
    c.ptable[0, 20] = keep
    c.check(out, lse, absent=lost)


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_long(A, kind):
    """Long prefixes and own rows: many pieces, joined."""
    c = PrefixCase(A, 9, kind, 64, 2, 2, 16, [3, 2], [5001, 9000], [3000, 1, 0, 7000, 4095])
    c.check(*c.run())


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_none(A, kind):
    c = PrefixCase(A, 10, kind, 64, 4, 4, 16, [], [], [3, 0, 200, 1000], no_group=4)
    c.check(*c.run(workspace=None))


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("ratio", [1, 2, 4])
def test_prefix_int8_largest_codes(A, d, ratio):
    """Codes of -128 and 127 and equal scores over many rows: the largest sums a piece can hold."""
    import torch
    c = PrefixCase(A, d, "int8", d, ratio, 1, 64, [], [], [50000, 4097], no_group=2)
    c.q.fill_(-1.0)
    for x, s, x64, code in ((c.kc, c.ks, c.k64, -128), (c.vc, c.vs, c.v64, 127)):
        x.fill_(code)
        x[::3, 1::2] = -code - 1
        s.copy_(torch.where(s.isnan(), s, torch.full_like(s, 2.0 ** -9)))
        x64[:] = x.cpu().numpy().astype(np.float64) * 2.0 ** -9
    c.check(*c.run())


def scores_bound(c, s):
    """out of request s in 64 bits and its bound, key by key: with delta_j = 2^-21 (1 + scale sum|q k_j|) a probability is
    off by the factor 1 +- 2 delta_j, and so is the sum it is divided by: 2 sum p delta |v| + 2 sum p delta . sum p |v|.
    (A key without a probability adds nothing, however wide its value is.)"""
    rows, d, r = c.rows_of(s), c.d, c.heads // c.kv_heads
    q = c.q[s].double().cpu().numpy().reshape(c.heads, d)
    out, tol = np.zeros((c.heads, d)), np.zeros((c.heads, d))
    for h in range(c.heads):
        k, v = (x[rows][:, h // r * d:(h // r + 1) * d] for x in (c.k64, c.v64))
        x = k @ q[h] / np.sqrt(d)
        p = np.exp(x - x.max())
        p /= p.sum()
        delta = 2.0 ** -21 * (1 + np.abs(k) @ np.abs(q[h]) / np.sqrt(d))
        out[h] = p @ v
        tol[h] = 2 * (p * delta) @ np.abs(v) + 2 * (p @ delta) * (p @ np.abs(v)) + len(rows) * 2.0 ** -126 * np.abs(v).max()
    return out.ravel(), tol.ravel()


@pytest.mark.parametrize("spread", [1e3, 1e4, 1e6])
@pytest.mark.parametrize("d,ratio", [(32, 1), (64, 1), (64, 2), (96, 2), (128, 1), (64, 4), (128, 4), (32, 8), (64, 8)])
@pytest.mark.parametrize("sizes,plen,mixed", [([], 0, False), ([3], 300, False), ([20], 300, False), ([6], 300, True)])
def test_prefix_int8_wide_value_scales(A, d, ratio, sizes, plen, mixed, spread):
    """Value scales far apart: every 16th row's is `spread` times the others' and its scores are too low to count, so it may
    not cost the others their bits; `mixed` spreads the scales evenly in their logarithm instead."""
    n = max(5, sum(sizes))
    c = PrefixCase(A, d + ratio, "int8", d, 2 * ratio, 2, 16, sizes, [plen] * len(sizes), ([70, 200, 40, 33, 64] * n)[:n], no_group=n - sum(sizes))
    r = np.random.RandomState(d)
    if mixed:
        wide = np.exp(r.uniform(0, np.log(spread), c.v64.shape[0]))
    else:
        wide = np.where(np.arange(c.v64.shape[0]) % 16 == 5, spread, 1.0)
        c.q[:, ::d] = 300.0                       # dim 0 of every head: code -127 in a wide row, 0 in the others
        codes = np.where(wide > 1, -127, 0).astype(np.int8)
        for j in range(2):
            c.kc[:, j * d] = dev(codes)
            c.k64[:, j * d] = codes * np.nan_to_num(c.ks[:, j].double().cpu().numpy())
    c.vs *= dev(wide.astype(np.float32))[:, None]
    c.v64 = c.vc.double().cpu().numpy() * np.repeat(np.nan_to_num(c.vs.double().cpu().numpy()), d, 1)
    out, _ = c.run()
    for s in range(n):
        want, tol = scores_bound(c, s)
        err = np.abs(out[s].double().cpu().numpy() - want)
        assert (err <= tol).all(), (s, (err / tol).max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ratio", [1, 2, 4])
@pytest.mark.parametrize("sizes,plen,no_group", [([], 0, 5), ([5], 300, 0), ([40], 300, 0)])
def test_prefix_not_numbers(A, kind, ratio, sizes, plen, no_group):
    """What is no number in a query, a key or a value shows in its own outputs, and only there."""
    n = sum(sizes) + no_group
    c = PrefixCase(A, 14, kind, 64, 3 * ratio, 3, 16, sizes, [plen] * len(sizes), ([70, 200, 40, 33, 64] * n)[:n], no_group=no_group)
    row = [c.rows_of(s)[plen:] for s in range(5)]
    c.q[0, 5] = float("nan")                      # head 0
    c.q[1, 64 * (3 * ratio - 1)] = float("inf")   # the last head
    if kind == "int8":
        c.ks[row[2][7], 1] = float("nan")         # key head 1
        c.vs[row[3][32], 2] = float("nan")        # key head 2
    else:
        c.kc[row[2][7], 64 + 9] = float("nan")
        c.vc[row[3][32], 128:192] = float("nan")
    out, lse = c.run()
    o = out.view(n, 3 * ratio, 64)
    bad = {(0, 0), (1, 3 * ratio - 1)} | {(2, ratio + i) for i in range(ratio)} | {(3, 2 * ratio + i) for i in range(ratio)}
    for s in range(n):
        for h in range(3 * ratio):
            assert (not o[s, h].isfinite().any()) if (s, h) in bad else o[s, h].isfinite().all(), (s, h)
            assert bool(lse[s, h].isfinite()) == ((s, h) not in bad or s == 3), (s, h)
    c.check(out, lse, only=[4])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ratio", [1, 4])
@pytest.mark.parametrize("n", [5, 40])
def test_prefix_value_not_a_number_without_weight(A, kind, ratio, n):
    """A prefix of one row whose value is no number, and whose score is so low that its weight is 0 beside the own rows':
    it shows all the same, in its own key head alone."""
    c = PrefixCase(A, 16, kind, 64, 2 * ratio, 2, 16, [n], [1], ([70, 0, 40, 33, 300] * n)[:n])
    c.q.fill_(4.0)
    row = c.rows_of(0)[0]
    if kind == "int8":
        c.kc[row] = -127
        c.ks[row], c.vs[row, 1] = 0.5, float("nan")
    else:
        c.kc[row], c.vc[row, 64:] = -60.0, float("nan")
    out, lse = c.run()
    o = out.view(n, 2, ratio, 64).isfinite()
    assert o[:, 0].all() and not o[:, 1].any() and lse.isfinite().all()


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_sharp_scores(A, kind):
    """Scores of many hundreds: the largest key alone counts, and nothing overflows."""
    c = PrefixCase(A, 11, kind, 64, 4, 4, 16, [6], [700], [0, 10, 300, 1, 64, 65], q_std=300.0)
    c.check(*c.run())


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_strides_streams_and_repeats(A, kind):
    """q and out as column blocks, a cache with a wider row, another stream, no lse: the same bits."""
    import torch
    c = PrefixCase(A, 12, kind, 96, 4, 2, 32, [4, 3], [400, 130], [10, 0, 200, 31, 32, 33, 90], extra_stride=48)
    out, lse = c.run()
    c.check(out, lse)
    wide = torch.zeros((c.n, 600), dtype=c.q.dtype, device="cuda")
    q, o = wide[:, 16:16 + c.q.shape[1]], torch.full((c.n, 800), 3.0, dtype=c.q.dtype, device="cuda")
    q.copy_(c.q)
    c.shape.q_row_stride, c.shape.out_row_stride = 600, 800
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = c.run(q=q, out=o[:, 8:8 + c.q.shape[1]], lse=False)
    side.synchronize()
    assert torch.equal(got, out)
    assert (o[:, :8] == 3).all() and (o[:, 8 + c.q.shape[1]:] == 3).all()
    c.shape.q_row_stride = c.shape.out_row_stride = 0
    for _ in range(3):
        again, l2 = c.run()
        assert torch.equal(again, out) and torch.equal(l2, lse)


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_bad_pages_and_lengths(A, kind):
    """A page outside the cache: its rows are absent and the error word says 0x702; a length past its bound: 0x703."""
    c = PrefixCase(A, 13, kind, 64, 2, 2, 16, [4], [100], [40, 0, 50, 3])
    lost = set(range(int(c.ptable[0, 2]) * 16, int(c.ptable[0, 2]) * 16 + 16))
    out, lse = c.run()
    c.check(out, lse)
    assert device_error(A) == 0
    good = c.ptable.copy()
    c.ptable[0, 2] = -1
    out, lse = c.run()
    assert device_error(A) == 0x702
    c.ptable = good
    c.check(out, lse, absent=lost)
    c.shape.max_len = 49
    out, _ = c.run()
    assert device_error(A) == 0x703
    c.lens[2] = 49
    c.check(out, None)


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_lengths_past_a_bound_of_zero(A, kind):
    """A part whose bound is 0 has no rows, and lengths above the bound are reported all the same: own rows, a prefix,
    and neither of them; not the prefix of a group without requests."""
    c = PrefixCase(A, 15, kind, 64, 2, 2, 16, [2, 0, 1], [40, 7, 0], [9, 0, 30])
    device_error(A)
    full, lens, plens = (c.shape.max_len, c.shape.max_prefix_len), c.lens, c.plens
    for own, prefix, code in ((0, full[1], 0x703), (full[0], 0, 0x703), (0, 0, 0x703), (full[0], full[1], 0)):
        c.shape.max_len, c.shape.max_prefix_len = own, prefix
        c.lens, c.plens = lens, plens
        out, lse = c.run()
        assert device_error(A) == code, (own, prefix)
        c.lens, c.plens = np.minimum(lens, own), np.minimum(plens, prefix)
        c.check(out, lse)
    c.shape.max_len, c.shape.max_prefix_len, c.lens, c.plens = full[0], 0, lens, np.array([0, 7, 0], np.int32)
    out, lse = c.run()
    assert device_error(A) == 0
    c.plens = 0 * plens
    c.check(out, lse)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_prefix_cache_past_32_bits(A, kind):
    """Rows whose element offsets pass 2^31."""
    import torch
    page, w = 64, 2 * 128
    n_pages = 2 ** 31 // (page * w) + 40
    dt = torch.bfloat16 if kind == "bf16" else torch.int8
    kc, vc = (torch.zeros((n_pages * page, w), dtype=dt, device="cuda") for _ in range(2))
    c = PrefixCase(A, 14, kind, 128, 2, 2, page, [3], [200], [70, 5, 0])
    small = c.kc.shape[0] // page
    kc[-small * page:].copy_(c.kc)
    vc[-small * page:].copy_(c.vc)
    want, wl = c.run()
    shift = n_pages - small
    c.ptable[:, :4] += shift                # pages in use; the entries past them stay outside
    c.table = np.where(c.table >= 0, c.table + shift, c.table).astype(np.int32)
    ks = vs = None
    if kind == "int8":
        ks, vs = (torch.full((n_pages * page, 2), float("nan"), device="cuda") for _ in range(2))
        ks[-small * page:].copy_(c.ks)
        vs[-small * page:].copy_(c.vs)
    c.cache = A.PageCache.of(kc, vc, ks, vs)
    out, lse = c.run()
    assert torch.equal(out, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[224] + [1] * 32, [0, 1, 2, 0, 3, 5] * 15, [1] * 70])
def test_prefix_many_groups(A, kind, sizes):
    """More groups than a warp looks through at once, empty ones and one that has most of the requests."""
    r = np.random.RandomState(len(sizes))
    n = sum(sizes) + 3
    c = PrefixCase(A, 18, kind, 32, 4, 2, 16, sizes, r.randint(0, 90, len(sizes)), r.randint(0, 20, n), no_group=3)
    c.check(*c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [6, 70])
def test_prefix_call_in_a_graph(A, kind, n):
    """A call with a prefix (own rows' launch beside the prefix's) between other work on the stream, captured and replayed
    with other queries and lengths: the same bits as the calls one by one."""
    import torch
    c = PrefixCase(A, 19, kind, 64, 4, 2, 16, [n // 2, n - n // 2], [300, 90], np.random.RandomState(n).randint(0, 60, n))
    queries = [dev(synth.normal(40 + i, tuple(c.q.shape)), c.q.dtype) for i in range(3)]
    lengths = [dev(np.minimum(c.lens, m).astype(np.int32)) for m in (60, 31, 7)]
    q, lens, out = torch.empty_like(c.q), torch.empty_like(lengths[0]), torch.empty_like(c.q)
    lse, twice = torch.empty((n, 4), device="cuda"), torch.empty_like(c.q)
    work = torch.empty(A.prefix_decode_workspace_bytes(c.shape, c.cache), dtype=torch.uint8, device="cuda")
    group, table, given = (dev(c.begin), dev(c.ptable), dev(c.plens)), dev(c.table), (torch.empty_like(c.q), torch.empty_like(lens))

    def step():
        q.copy_(given[0])
        lens.copy_(given[1])
        A.prefix_decode_t(c.shape, c.cache, q, *group, table, lens, out, lse=lse, workspace=work)
        torch.mul(out, 2, out=twice)
        q.zero_()                         # the next call's inputs may be written as soon as this one is over
        lens.zero_()

    want = []
    for x in zip(queries, lengths):
        for to, src in zip(given, x):
            to.copy_(src)
        step()
        want.append((twice.clone(), lse.clone()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
        step()
    for x, (w, wl) in zip(zip(queries, lengths), want):
        for to, src in zip(given, x):
            to.copy_(src)
        twice.zero_()
        lse.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(twice, w) and torch.equal(lse, wl)
    c.q, c.lens = queries[0], lengths[0].cpu().numpy()
    c.check(want[0][0] / 2, want[0][1])


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_calls_on_two_streams(A, kind):
    """Two calls at a time, each on its stream with its workspace: the same bits as alone."""
    import torch
    cases = [PrefixCase(A, 20 + i, kind, 64, 4, 2, 16, [n], [plen], np.random.RandomState(n).randint(0, 300, n))
             for i, (n, plen) in enumerate(((40, 700), (9, 2000)))]
    want = [c.run() for c in cases]
    outs = [(torch.empty_like(w), torch.empty_like(l)) for w, l in want]
    calls = [prefix_call(A, c, c.q, *o, torch.empty(A.prefix_decode_workspace_bytes(c.shape, c.cache), dtype=torch.uint8, device="cuda"))
             for c, o in zip(cases, outs)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o[0].fill_(float("nan"))
        torch.cuda.synchronize()
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                call()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_serving_calls_are_captured_in_a_graph(A):
    """plan, append and decode in one CUDA graph, replayed: the same results as the calls."""
    import torch
    n, heads, d, page, total = 4, 2, 64, 8, 40
    shape = A.PageShape(n, page, 8, 16, total, 0)
    lens, new = dev(np.array([3, 8, 0, 20], np.int32)), dev(np.array([1, 1, 1, 1], np.int32))
    table = torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    table[:, :3] = torch.arange(12, dtype=torch.int32, device="cuda").view(4, 3)
    free, count = torch.arange(12, total, dtype=torch.int32, device="cuda"), dev(np.array([total - 12], np.int32))
    free = torch.cat([free, torch.full((12,), -1, dtype=torch.int32, device="cuda")])
    kc, vc = (torch.randn((total * page, heads * d), device="cuda") for _ in range(2))
    cache = A.PageCache.of(kc, vc)
    q, k, v = (torch.randn((16, heads * d), device="cuda") for _ in range(3))
    rope = A.rope_table_t(A.RopeConfig(d, 64, A.ROPE_PLAIN, 0, 10000.0, 1.0, 0.0, 0.0, 1.0))
    rshape = A.RopeShape(16, 0, heads, heads, d, d, 0, 64, 0, 0, 0, 0, 0)
    pshape = A.PrefixShape(n, 0, heads, heads, d, A.F32, page, 0, 8, 0, 64, 0, 0, 0.0)
    work = torch.empty(A.prefix_decode_workspace_bytes(pshape, cache), dtype=torch.uint8, device="cuda")
    out, plan, q_out = torch.empty((n, heads * d), device="cuda"), A.page_outputs(shape), torch.empty_like(q)

    def step():
        A.page_plan_t(shape, lens, new, free, count, table, plan)
        A.rope_append_t(rshape, cache, rope, plan["positions"], plan["slot_map"], q, k, v, q_out)
        A.prefix_decode_t(pshape, cache, q_out, None, None, None, table, plan["lens"], out, workspace=work)

    step()
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and float(out.abs().sum()) > 0


def prefix_call(A, c, q, out, lse, workspace):
    """A call on device arrays made beforehand, as a captured one needs."""
    group = (dev(c.begin), dev(c.ptable), dev(c.plens))
    own = (dev(c.table), dev(c.lens))
    return lambda: A.prefix_decode_t(c.shape, c.cache, q, *group, *own, out, lse=lse, workspace=workspace)


def test_prefix_without_a_workspace_is_refused_in_a_graph(A):
    """The library's buffer may move, and a graph would keep its address: refused while capturing, and the capture goes on."""
    import torch
    c = PrefixCase(A, 17, "f32", 64, 4, 2, 16, [3], [100], [20, 0, 40])
    want, wl = c.run(workspace=None)
    out, lse = torch.zeros_like(want), torch.zeros_like(wl)
    work = torch.empty(A.prefix_decode_workspace_bytes(c.shape, c.cache), dtype=torch.uint8, device="cuda")
    refused, taken = (prefix_call(A, c, c.q, out, lse, w) for w in (None, work))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(A.AttnError, match="workspace") as e:
            refused()
        taken()
    assert e.value.status == A.ERR_WORKSPACE
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wl)
    again, _ = c.run(workspace=None)
    assert torch.equal(again, want)


@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_serving_example(A, cache):
    """The example's loop: projection, plan, append and decode together; fp32 arithmetic, the repository's 1e-5."""
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("serve_shared_prefix", os.path.join(ROOT, "examples", "serve_shared_prefix.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(requests=6, prompt=130, steps=21, cache=cache) < 1e-5


def test_serving_example_uses_the_prompts_attention(A, monkeypatch):
    """What the prompt attends to reaches the requests, and an output that is no number reaches the example's result."""
    import runpy
    import os
    from conftest import ROOT
    m = runpy.run_path(os.path.join(ROOT, "examples", "serve_shared_prefix.py"))
    forward = A.forward_t
    monkeypatch.setattr(A, "forward_t", lambda *a, **kw: (forward(*a, **kw)[0] * float("nan"), None))
    assert not m["main"](requests=2, prompt=20, steps=3) < 1e-5
