"""Measured cases of the paged serving operators and of the rotary embedding:

  pages    attn_page_plan_ex: a step's slot map, positions, block-table entries and free list from the
           requests' lengths
  rope     attn_rope_ex: rotation of Q and K by their positions (forward, or transposed for gradients)
  append   attn_rope_append_ex: the serving form, Q rotated and K (rotated) and V written to their cache slots
  prefix   attn_prefix_decode_ex: one query token per request over a prefix that the request's group shares
           and the request's own rows, both in a paged cache

A case names its operator in "op".  With `own` false `run` computes the operators from elementary torch
operations in 32 bits; with `own` true it makes the library's calls.
"""
import math
import os
import sys

import torch

own = False

INTS = torch.int32


def listed():
    return [
        # a decode step of a lightly loaded server: latency alone
        {"name": "pages-few", "op": "pages", "n_seq": 8, "page": 16, "max_len": 2048, "new": 1, "ended": 0.0, "room": 1.0},
        # a decode step of a full server: one token each, some requests end and hand their pages back
        {"name": "pages-step", "op": "pages", "n_seq": 2048, "page": 16, "max_len": 8192, "new": 1, "ended": 0.05, "room": 1.0},
        # admission of many ragged prompts, with too few free pages for the last ones
        {"name": "pages-prompts", "op": "pages", "n_seq": 301, "page": 64, "max_len": 0, "new": 2047, "ended": 0.0, "room": 0.9},
        # the reference trainer's attention inputs: 4 x 1024 tokens, 12 heads of 128, as column blocks of the
        # fused projection's output, halves layout
        {"name": "rope-train-f32", "op": "rope", "tokens": 4096, "seq_len": 1024, "heads": 12, "kv_heads": 12, "d": 128,
         "rot": 128, "interleaved": False, "transpose": False, "type": "f32", "fused": True},
        # the gradient of the 16 x 64 prefill shape in bf16, interleaved pairs on half of each head
        {"name": "rope-grad-bf16", "op": "rope", "tokens": 8192, "seq_len": 1024, "heads": 16, "kv_heads": 16, "d": 64,
         "rot": 32, "interleaved": True, "transpose": True, "type": "bf16", "fused": False},
        # a decode step: one new token for each of 64 requests, fp32 cache
        {"name": "append-step-f32", "op": "append", "tokens": 64, "heads": 16, "kv_heads": 16, "d": 64, "rot": 64,
         "interleaved": False, "type": "f32", "slots": 65536, "max_pos": 8192},
        # long prompts into a bf16 cache with shared key heads
        {"name": "append-prompts-bf16", "op": "append", "tokens": 32749, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "interleaved": False, "type": "bf16", "slots": 49152, "max_pos": 131072},
        # few requests of the small model on a short shared prompt: latency
        {"name": "prefix-few-f32", "op": "prefix", "n_seq": 4, "groups": 1, "prefix": 500, "tail": 60, "heads": 16, "kv_heads": 16,
         "d": 32, "page": 16, "type": "f32", "cache": "f32"},
        # a chat batch on one system prompt, every head with its own keys
        {"name": "prefix-chat-bf16", "op": "prefix", "n_seq": 64, "groups": 1, "prefix": 8192, "tail": 1024, "heads": 16,
         "kv_heads": 16, "d": 64, "page": 16, "type": "bf16", "cache": "bf16"},
        # the trainer's head shape in fp32, odd lengths
        {"name": "prefix-f32", "op": "prefix", "n_seq": 33, "groups": 2, "prefix": 2047, "tail": 511, "heads": 12, "kv_heads": 12,
         "d": 128, "page": 32, "type": "f32", "cache": "f32"},
        # the ragged-decode batch (64 requests, up to 8192 own rows, 16 x 64) behind a prefix, INT8 cache
        {"name": "prefix-int8", "op": "prefix", "n_seq": 64, "groups": 1, "prefix": 16384, "tail": 8192, "heads": 16,
         "kv_heads": 16, "d": 64, "page": 64, "type": "f32", "cache": "int8"},
        # a full server on two long documents, four query heads to a key head
        {"name": "prefix-documents-bf16", "op": "prefix", "n_seq": 256, "groups": 2, "prefix": 32768, "tail": 2000, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "type": "bf16", "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["pages", "rope", "append", "prefix", "prefix"])
    if op == "pages":
        if rng.random() < 0.5:
            return {"op": op, "n_seq": _log(rng, 1, 4096), "page": rng.choice([8, 16, 32, 64, 128]), "max_len": _log(rng, 64, 8192),
                    "new": rng.randint(1, 4), "ended": rng.choice([0.0, 0.02, 0.3]), "room": rng.choice([1.0, 0.5])}
        return {"op": op, "n_seq": _log(rng, 2, 400), "page": rng.choice([8, 16, 32, 64, 128]), "max_len": rng.choice([0, 700]),
                "new": _log(rng, 64, 2047), "ended": rng.choice([0.0, 0.1]), "room": rng.choice([1.0, 0.7])}
    d = rng.choice([32, 64, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([r for r in (1, 1, 2, 4, 8) if r * kv_heads <= 32 and r * kv_heads * d != 3072])
    if kv_heads * d == 3072:
        kv_heads = heads = 8
    kind = rng.choice(["f32", "bf16"])
    if op in ("rope", "append"):
        rot = rng.choice([d, d // 2, 2 * rng.randint(1, d // 2)])
        case = {"op": op, "tokens": _log(rng, 1, 32749), "heads": heads, "kv_heads": kv_heads, "d": d, "rot": rot,
                "interleaved": rng.random() < 0.5, "type": kind}
        if op == "rope":
            case.update(seq_len=rng.choice([1024, 777]), transpose=rng.random() < 0.5, fused=rng.random() < 0.5)
            if case["fused"] and (heads + 2 * kv_heads) * d == 3072:
                case["fused"] = False
        else:
            case.update(slots=case["tokens"] * 2 + rng.randint(0, 999), max_pos=_log(rng, 1024, 131072))
        return case
    cache = rng.choice([kind, "int8"])
    n_seq = _log(rng, 1, 256)
    case = {"op": op, "n_seq": n_seq, "groups": rng.choice([g for g in (1, 1, 2, 3, 5) if g <= n_seq]), "prefix": _log(rng, 1, 32768),
            "tail": _log(rng, 1, 2000), "heads": heads, "kv_heads": kv_heads, "d": d, "page": rng.choice([8, 16, 32, 64, 128]),
            "type": "f32" if cache == "int8" else kind, "cache": cache}
    most = _prefix_numbers(listed()[-1])
    while True:
        now = _prefix_numbers(case)
        if now["flops"] <= most["flops"] and now["bytes"] <= most["bytes"]:
            return case
        case["prefix"], case["tail"] = max(1, case["prefix"] // 2), max(1, case["tail"] * 3 // 4)


TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "int8": 1}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, n, lo, hi):
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda", dtype=INTS)


def _normal(g, shape, kind, std=1.0):
    x = torch.empty(shape, dtype=torch.float32, device="cuda")
    x.normal_(0.0, std, generator=g)
    return x.to(TYPES[kind])


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    {"pages": _prepare_pages, "rope": _prepare_rope, "append": _prepare_append, "prefix": _prepare_prefix}[case["op"]](case, g, s)
    return s


def _prepare_pages(case, g, s):
    n, page = case["n_seq"], case["page"]
    most = case["max_len"] + case["new"]
    s["max_pages"] = max_pages = -(-most // page)
    s["max_tokens"] = n * case["new"]
    lens = _ints(g, n, 1, case["max_len"]) if case["max_len"] else torch.zeros(n, dtype=INTS, device="cuda")
    new = _ints(g, n, 1, case["new"])
    ends = torch.rand(n, generator=g, device="cuda") < case["ended"]
    have = (lens + page - 1) // page
    pages = torch.randperm(n * max_pages, generator=g, device="cuda", dtype=torch.int64).to(INTS)
    column = torch.arange(max_pages, device="cuda", dtype=INTS)[None, :]
    held = column < have[:, None]
    table = torch.full((n, max_pages), -1, dtype=INTS, device="cuda")
    taken = int(held.sum())
    table[held] = pages[:taken]
    free = torch.full((n * max_pages,), -1, dtype=INTS, device="cuda")
    need = int(((lens + new + page - 1) // page - have).sum())
    free_count = min(n * max_pages - taken, max(1, int(need * case["room"] + 0.5)))
    free[:free_count] = pages[taken:taken + free_count]
    s.update(lens=lens, new=torch.where(ends, -1, new).to(INTS), free=free, table=table,
             free_count=torch.tensor([free_count], dtype=INTS, device="cuda"), base=_ints(g, n, 0, 4000))
    out = {"lens": (n,), "cu_new": (n + 1,), "positions": (s["max_tokens"],), "token_seq": (s["max_tokens"],), "counts": (4,)}
    s["out"] = {k: torch.empty(shape, dtype=INTS, device="cuda") for k, shape in out.items()}
    s["out"]["slot_map"] = torch.empty(s["max_tokens"], dtype=torch.int64, device="cuda")


def _table(rot, max_pos):
    """cos and sin of position x frequency, [max_pos][rot / 2][2], angles taken in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * freq[None, :]
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


def _prepare_rope(case, g, s):
    n, d, qw, kw = case["tokens"], case["d"], case["heads"] * case["d"], case["kv_heads"] * case["d"]
    if case["fused"]:      # Q and K are column blocks of one projection output [Q | K | V]
        x = _normal(g, (n, qw + 2 * kw), case["type"])
        s["q"], s["k"] = x[:, :qw], x[:, qw:qw + kw]
    else:
        s["q"], s["k"] = _normal(g, (n, qw), case["type"]), _normal(g, (n, kw), case["type"])
    s["table"] = _table(case["rot"], case["seq_len"])
    s["q_out"], s["k_out"] = torch.empty((n, qw), dtype=s["q"].dtype, device="cuda"), torch.empty((n, kw), dtype=s["q"].dtype, device="cuda")


def _prepare_append(case, g, s):
    n, qw, kw = case["tokens"], case["heads"] * case["d"], case["kv_heads"] * case["d"]
    s["q"], s["k"], s["v"] = (_normal(g, (n, w), case["type"]) for w in (qw, kw, kw))
    s["table"] = _table(case["rot"], case["max_pos"])
    s["positions"] = _ints(g, n, 0, case["max_pos"] - 1)
    s["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:n].contiguous()
    if n > 8:
        s["slots"][3::97] = -1          # padding rows: nothing is written for them
    s["q_out"] = torch.empty_like(s["q"])
    s["kcache"], s["vcache"] = (torch.zeros((case["slots"], kw), dtype=s["q"].dtype, device="cuda") for _ in range(2))


def _prepare_prefix(case, g, s):
    n, groups, page, d = case["n_seq"], case["groups"], case["page"], case["d"]
    kw = case["kv_heads"] * d
    pp, po = -(-case["prefix"] // page), -(-case["tail"] // page)
    s["lens"] = _ints(g, n, 0 if n > 16 else 1, case["tail"])
    s["lens"][0] = case["tail"]
    s["prefix_lens"] = _ints(g, groups, max(1, case["prefix"] - case["prefix"] // 8), case["prefix"])
    s["prefix_lens"][0] = case["prefix"]
    # groups of about equal size
    s["group_begin"] = torch.tensor([i * n // groups for i in range(groups + 1)], dtype=INTS, device="cuda")
    n_pages = groups * pp + n * po + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(INTS)
    s["prefix_table"] = ids[:groups * pp].view(groups, pp).contiguous()
    s["block_table"] = ids[groups * pp:groups * pp + n * po].view(n, po).contiguous()
    s["n_pages"] = n_pages
    rows = n_pages * page
    s["q"] = _normal(g, (n, case["heads"] * d), case["type"])
    s["kscale"] = s["vscale"] = None
    if case["cache"] == "int8":
        for x in ("k", "v"):
            s[x + "cache"] = torch.randint(-127, 128, (rows, kw), generator=g, device="cuda", dtype=torch.int8)
            s[x + "scale"] = torch.rand((rows, case["kv_heads"]), generator=g, device="cuda") * 0.01 + 0.012
    else:
        s["kcache"], s["vcache"] = (_normal(g, (rows, kw), case["cache"]) for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((n, case["heads"]), dtype=torch.float32, device="cuda")


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"pages": _own_pages, "rope": _own_rope, "append": _own_append, "prefix": _own_prefix}[op](s, _library())
    return {"pages": _plain_pages, "rope": _plain_rope, "append": _plain_append, "prefix": _plain_prefix}[op](s)


def _library():
    if "attn_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "pure-c-llm_b200"))
    import attn_b200
    return attn_b200


def _own_pages(s, A):
    if "shape" not in s:
        s["shape"] = A.PageShape(s["case"]["n_seq"], s["case"]["page"], s["max_pages"], s["max_tokens"], s["free"].numel(), 0)
    out = s["out"]
    A.page_plan_t(s["shape"], s["lens"], s["new"], s["free"], s["free_count"], s["table"], out, pos_base=s["base"])
    return {**out, "table": s["table"], "free": s["free"]}


def _rope_shape(s, A, seq_len, max_pos):
    c = s["case"]
    return A.RopeShape(c["tokens"], seq_len, c["heads"], c["kv_heads"], c["d"], c["rot"], int(c["interleaved"]), max_pos,
                       s["q"].stride(0), s["k"].stride(0), 0, 0, 0)


def _own_rope(s, A):
    if "shape" not in s:
        s["shape"] = _rope_shape(s, A, s["case"]["seq_len"], s["case"]["seq_len"])
    A.rope_t(s["shape"], s["table"], None, s["q"], s["k"], s["q_out"], s["k_out"], transpose=s["case"]["transpose"])
    return s["q_out"], s["k_out"]


def _own_append(s, A):
    if "shape" not in s:
        s["shape"] = _rope_shape(s, A, 0, s["case"]["max_pos"])
        s["cache"] = A.PageCache.of(s["kcache"], s["vcache"])
    A.rope_append_t(s["shape"], s["cache"], s["table"], s["positions"], s["slots"], s["q"], s["k"], s["v"], s["q_out"])
    return s["q_out"], s["kcache"], s["vcache"]


def _own_prefix(s, A):
    if "shape" not in s:
        c = s["case"]
        s["cache"] = A.PageCache.of(s["kcache"], s["vcache"], s["kscale"], s["vscale"])
        s["shape"] = A.PrefixShape(c["n_seq"], c["groups"], c["heads"], c["kv_heads"], c["d"], A.BF16 if c["type"] == "bf16" else A.F32,
                                   c["page"], s["prefix_table"].shape[1], s["block_table"].shape[1], c["prefix"], c["tail"], 0, 0, 0.0)
        s["work"] = torch.empty(A.prefix_decode_workspace_bytes(s["shape"], s["cache"]), dtype=torch.uint8, device="cuda")
    A.prefix_decode_t(s["shape"], s["cache"], s["q"], s["group_begin"], s["prefix_table"], s["prefix_lens"], s["block_table"], s["lens"],
                      s["out"], lse=s["lse"], workspace=s["work"])
    return s["out"], s["lse"]


def _plain_pages(s):
    page, max_pages, max_tokens = s["case"]["page"], s["max_pages"], s["max_tokens"]
    out, table, free, count = s["out"], s["table"], s["free"], s["free_count"].long()
    lens, new = s["lens"].clamp(0, max_pages * page).long(), s["new"].clamp(min=0).long()
    ended = s["new"] < 0
    have, end = (lens + page - 1) // page, lens + new
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    fits = ~ended & ((new == 0) | ((end <= max_pages * page) & (cu[1:] <= max_tokens)))
    need = torch.where(fits, (end + page - 1) // page - have, 0)
    back = torch.where(ended, have, 0)
    # the list pages are taken from, last entry first: the free pages, then those of the ended requests
    column = torch.arange(max_pages, device="cuda")[None, :]
    pool = torch.cat([free[:1].new_full((1,), -1), free, table[column < back[:, None]]])      # [0] stands for "none"
    returned = back.sum()
    avail = count + returned
    taken = need.cumsum(0)
    ok = fits & ((need == 0) | (taken <= avail))
    used = torch.where(ok, need, 0).sum()
    at = torch.arange(pool.numel() - 1, device="cuda")
    stack = torch.where(at < count, at, at - count + free.numel())                             # place in the list -> place in pool - 1
    i = column - have[:, None]
    fresh = ok[:, None] & (i >= 0) & (i < need[:, None])
    place = (avail - 1 - (taken - need)[:, None] - i).clamp(0, stack.numel() - 1)
    pages = torch.where(fresh, pool[1 + stack[place].clamp(max=pool.numel() - 2)], table)
    table.copy_(pages)
    kept = (at >= count) & (at < avail - used)
    at_free = at[:free.numel()]
    free.copy_(torch.where(kept[:free.numel()], pool[1 + stack[at_free].clamp(max=pool.numel() - 2)], free))
    t = torch.arange(max_tokens, device="cuda")
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=new.numel() - 1)
    real = t < cu[-1]
    p = lens[seq] + t - cu[seq]
    entry = table[seq, (p // page).clamp(0, max_pages - 1)].long()
    out["slot_map"].copy_(torch.where(real & ok[seq], entry * page + p % page, -1))
    out["positions"].copy_(torch.where(real, s["base"][seq] + p, 0))
    out["token_seq"].copy_(torch.where(real, seq, -1))
    out["cu_new"].copy_(cu)
    out["lens"].copy_(torch.where(ended, 0, torch.where(ok, end, lens)))
    out["counts"].copy_(torch.cat([(avail - used).view(1), cu[-1:], (~ok & ~ended).sum().view(1), used.view(1)]))
    return {**out, "table": table, "free": free}


def _rotate(x, case, heads, cs, transpose):
    """x: (tokens, heads * d); cs: (tokens, rot / 2, 2)."""
    rot = case["rot"]
    x = x.float().reshape(x.shape[0], heads, case["d"])
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    if transpose:
        sin = -sin
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1).flatten(1)


def _plain_rope(s):
    c = s["case"]
    cs = s["table"][torch.arange(c["tokens"], device="cuda") % c["seq_len"]]
    s["q_out"].copy_(_rotate(s["q"], c, c["heads"], cs, c["transpose"]))
    s["k_out"].copy_(_rotate(s["k"], c, c["kv_heads"], cs, c["transpose"]))
    return s["q_out"], s["k_out"]


def _plain_append(s):
    c = s["case"]
    cs = s["table"][s["positions"].long()]
    s["q_out"].copy_(_rotate(s["q"], c, c["heads"], cs, False))
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["kcache"][at] = _rotate(s["k"], c, c["kv_heads"], cs, False)[keep].to(s["k"].dtype)
    s["vcache"][at] = s["v"][keep]
    return s["q_out"], s["kcache"], s["vcache"]


def _rows(table, page, most):
    """Cache rows of tokens 0 .. most - 1 of each line of a block table."""
    t = torch.arange(most, device="cuda")
    return table.long()[:, t // page] * page + t % page


def _values(s, x, rows):
    """Cache values of the rows (a, b) in 32 bits: (a, kv_heads, b, d)."""
    c = s["case"]
    v = s[x + "cache"][rows.flatten()].float().view(*rows.shape, c["kv_heads"], c["d"])
    if s[x + "scale"] is not None:
        v = v * s[x + "scale"][rows.flatten()].view(*rows.shape, c["kv_heads"], 1)
    return v.transpose(1, 2)


def _plain_prefix(s):
    c = s["case"]
    n, groups, h, hk, d, page = c["n_seq"], c["groups"], c["heads"], c["kv_heads"], c["d"], c["page"]
    r = h // hk
    q = s["q"].float().view(n, hk, r, d) * (1.0 / math.sqrt(d))
    begin = s["group_begin"].long()
    group = torch.searchsorted(begin, torch.arange(n, device="cuda"), right=True) - 1
    place = torch.arange(n, device="cuda") - begin[group]
    most = -(-n // groups)
    # queries of a group side by side, (groups, hk, most * r, d): the prefix is read once for all of them
    qg = q.new_zeros(groups, most, hk, r, d)
    qg[group, place] = q
    qg = qg.transpose(1, 2).reshape(groups, hk, most * r, d)
    rows = _rows(s["prefix_table"], page, c["prefix"])
    sp = qg @ _values(s, "k", rows).transpose(-1, -2)
    sp = sp.masked_fill((torch.arange(c["prefix"], device="cuda")[None, :] >= s["prefix_lens"][:, None])[:, None, None, :], -math.inf)
    mp = sp.amax(-1).clamp(min=-3e38)
    sp = torch.exp(sp - mp[..., None])
    lp, op = sp.sum(-1), sp @ _values(s, "v", rows)
    mp, lp, op = (x.view(groups, hk, most, r, -1).transpose(1, 2)[group, place] for x in (mp, lp, op))
    rows = _rows(s["block_table"], page, c["tail"])
    so = q @ _values(s, "k", rows).transpose(-1, -2)
    masked = torch.arange(c["tail"], device="cuda")[None, :] >= s["lens"][:, None]
    so = so.masked_fill(masked[:, None, None, :], -math.inf)
    mo = so.amax(-1, keepdim=True).clamp(min=-3e38)
    so = torch.exp(so - mo)
    lo, oo = so.sum(-1, keepdim=True), so @ _values(s, "v", rows)
    m = torch.maximum(mp, mo)
    wp, wo = torch.exp(mp - m), torch.exp(mo - m)
    total = lp * wp + lo * wo
    s["out"].copy_(((op * wp + oo * wo) / total).reshape(n, h * d))
    s["lse"].copy_((m + torch.log(total)).reshape(n, h))
    return s["out"], s["lse"]


# ---------------------------------------------------------------------------
# exact: the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)

    def attention():
        n, h, hk, d, page = case["n_seq"], case["heads"], case["kv_heads"], case["d"], case["page"]
        r = h // hk
        out = torch.zeros(n, hk, r, d, dtype=torch.float64, device="cuda")
        lse = torch.full((n, hk, r), -math.inf, dtype=torch.float64, device="cuda")
        q = s["q"].double().view(n, hk, r, d)
        begin, plens, lens = s["group_begin"].tolist(), s["prefix_lens"].tolist(), s["lens"].tolist()

        def fetch(x, table, count, j):
            t = torch.arange(count, device="cuda")
            at = table[t // page].long() * page + t % page
            v = s[x + "cache"][at, j * d:(j + 1) * d].double()
            return v if s[x + "scale"] is None else v * s[x + "scale"][at, j].double()[:, None]

        for g in range(case["groups"]):
            for j in range(hk):
                k0, v0 = (fetch(x, s["prefix_table"][g], plens[g], j) for x in ("k", "v"))
                members = range(begin[g], begin[g + 1])
                s0 = (q[begin[g]:begin[g + 1], j].reshape(-1, d) @ k0.T / math.sqrt(d)).view(len(members), r, -1)
                peak, rest = s0.amax(-1), []
                for a, i in enumerate(members):
                    k1, v1 = (fetch(x, s["block_table"][i], lens[i], j) for x in ("k", "v"))
                    s1 = q[i, j] @ k1.T / math.sqrt(d)
                    rest.append((s1, v1))
                    if lens[i]:
                        peak[a] = torch.maximum(peak[a], s1.amax(-1))
                p0 = torch.exp(s0 - peak[..., None])
                o, total = (p0.view(-1, p0.shape[-1]) @ v0).view(len(members), r, d), p0.sum(-1)
                for a, (s1, v1) in enumerate(rest):
                    p1 = torch.exp(s1 - peak[a][:, None])
                    o[a] += p1 @ v1
                    total[a] += p1.sum(-1)
                out[begin[g]:begin[g + 1], j] = o / total[..., None]
                lse[begin[g]:begin[g + 1], j] = peak + torch.log(total)
        return out.view(n, h * d), lse.view(n, h)

    if case["op"] == "prefix":
        return attention()
    n, d, rot = case["tokens"], case["d"], case["rot"]
    # each pair is one complex number, turned by multiplication with cos + i sin
    position = torch.arange(n, device="cuda") % case["seq_len"] if case["op"] == "rope" else s["positions"].long()
    turn = torch.view_as_complex(s["table"].double())[position][:, None, :]
    if case.get("transpose"):
        turn = turn.conj()

    def turned(x, heads):
        y = x.double().view(n, heads, d).clone()
        first = torch.arange(0, rot, 2) if case["interleaved"] else torch.arange(0, rot // 2)
        second = first + (1 if case["interleaved"] else rot // 2)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y.view(n, heads * d)

    q, k = turned(s["q"].contiguous(), case["heads"]), turned(s["k"].contiguous(), case["kv_heads"])
    if case["op"] == "rope":
        return q, k
    kc, vc = s["kcache"].double(), s["vcache"].double()
    keep = (s["slots"] >= 0).nonzero().flatten()
    kc[s["slots"][keep]], vc[s["slots"][keep]] = k[keep], s["v"].double()[keep]
    return q, kc, vc


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def _prefix_numbers(c):
    """Prefix and own rows at their expected lengths: every K and V row once, q, out and lse once."""
    prefix, own_rows = c["groups"] * c["prefix"] * (15 / 16 if c["groups"] > 1 else 1.0), c["n_seq"] * (c["tail"] + 1) / 2
    row = 2 * c["kv_heads"] * (c["d"] * BYTES[c["cache"]] + (4 if c["cache"] == "int8" else 0))
    table = 4 * (prefix + own_rows) / c["page"]
    act = c["n_seq"] * c["heads"] * (2 * c["d"] * BYTES[c["type"]] + 4)
    scores = c["n_seq"] * c["heads"] * (prefix / c["groups"] + (c["tail"] + 1) / 2)
    return {"bytes": (prefix + own_rows) * row + table + act, "flops": 4 * c["d"] * scores}


def work(case):
    c = case
    if c["op"] == "prefix":
        return _prefix_numbers(c)
    if c["op"] == "pages":
        tokens = c["n_seq"] * (c["new"] + 1) / 2 * (1 - c["ended"])
        rows = c["n_seq"] * c["new"]
        fresh = tokens / c["page"]
        back = c["n_seq"] * c["ended"] * c["max_len"] / 2 / c["page"]
        # lengths in and out, one table entry for each request's open page, new and returned pages, four words a token row
        return {"bytes": c["n_seq"] * 4 * 6 + 8 * (fresh + back) + rows * 16, "flops": 0}
    e, width = BYTES[c["type"]], (c["heads"] + c["kv_heads"]) * c["d"]
    pairs = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rot"] // 2
    if c["op"] == "rope":
        rows = min(c["tokens"], c["seq_len"])
        return {"bytes": 2 * c["tokens"] * width * e + rows * c["rot"] * 4, "flops": 6 * pairs}
    rows = min(c["tokens"], c["max_pos"])
    return {"bytes": 2 * c["tokens"] * (width + c["kv_heads"] * c["d"]) * e + rows * c["rot"] * 4 + c["tokens"] * 12, "flops": 6 * pairs}
