"""Measured cases of the normed rotary embedding and of drafted token trees over a paged cache:

  norm     attn_norm_rope_ex, attn_norm_rope_bwd_ex: each head of Q and K divided by its root mean square, weighted
           and turned by its position; or the gradients of Q, K and the weights
  append   attn_norm_rope_append_ex: the serving form, Q to its rows, K and V to their cache slots
  plan     attn_tree_plan_ex: positions and visibility masks of drafted tokens from their parents
  tree     attn_tree_decode_ex: every drafted token of a request over a shared prefix, the request's context and
           the drafted tokens it descends from, all in a paged cache
  commit   attn_tree_commit_ex: the cache rows of an accepted path moved together in all layers, lengths after it, the
           pages behind it handed back

A case names its operator in "op".  With `own` false `run` computes the operators from elementary torch
operations in 32 bits; with `own` true it makes the library's calls.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

INTS = torch.int32
EPS = 1e-6


def listed():
    return [
        # the reference trainer's attention inputs: 4 x 1024 tokens, 12 heads of 128, as column blocks of the fused
        # projection's output
        {"name": "norm-train-f32", "op": "norm", "grad": False, "tokens": 4096, "seq_len": 1024, "heads": 12, "kv_heads": 12, "d": 128,
         "rot": 128, "interleaved": False, "type": "f32", "fused": True},
        # its gradients
        {"name": "norm-grad-f32", "op": "norm", "grad": True, "tokens": 4096, "seq_len": 1024, "heads": 12, "kv_heads": 12, "d": 128,
         "rot": 128, "interleaved": False, "type": "f32", "fused": True},
        # gradients of a 64-dim bf16 model with shared key heads, interleaved pairs on half of each head
        {"name": "norm-grad-bf16", "op": "norm", "grad": True, "tokens": 8192, "seq_len": 1024, "heads": 16, "kv_heads": 4, "d": 64,
         "rot": 32, "interleaved": True, "type": "bf16", "fused": False},
        # the drafted tokens of 64 requests, eight each, into an fp32 cache
        {"name": "append-drafts-f32", "op": "append", "tokens": 512, "heads": 16, "kv_heads": 16, "d": 64, "rot": 64,
         "interleaved": False, "type": "f32", "slots": 65536, "max_pos": 8192},
        # long prompts into a bf16 cache with shared key heads
        {"name": "append-prompts-bf16", "op": "append", "tokens": 32749, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "interleaved": False, "type": "bf16", "slots": 49152, "max_pos": 131072},
        # small trees of few requests: latency alone
        {"name": "plan-few", "op": "plan", "n_seq": 8, "nodes": 16},
        # a full server's trees
        {"name": "plan-full", "op": "plan", "n_seq": 2048, "nodes": 64},
        # few requests of the small model, short drafts: latency
        {"name": "tree-few-f32", "op": "tree", "n_seq": 4, "nodes": 8, "groups": 0, "prefix": 0, "context": 500, "heads": 16,
         "kv_heads": 16, "d": 32, "page": 16, "type": "f32", "cache": "f32"},
        # the ragged-decode batch (64 requests of up to 8192 rows, 16 x 64) with trees of up to 16 tokens, INT8 cache
        {"name": "tree-int8", "op": "tree", "n_seq": 64, "nodes": 16, "groups": 0, "prefix": 0, "context": 8192, "heads": 16,
         "kv_heads": 16, "d": 64, "page": 64, "type": "f32", "cache": "int8"},
        # a full server on two documents, trees of up to 32 tokens, four query heads to a key head
        {"name": "tree-documents-bf16", "op": "tree", "n_seq": 256, "nodes": 32, "groups": 2, "prefix": 8192, "context": 2000, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # few requests of the small model, all of its 16 layers
        {"name": "commit-few-f32", "op": "commit", "n_seq": 4, "nodes": 8, "layers": 16, "kv_heads": 16, "d": 32, "page": 16, "type": "f32"},
        # a full server's large trees
        {"name": "commit-full-bf16", "op": "commit", "n_seq": 256, "nodes": 64, "layers": 4, "kv_heads": 8, "d": 128, "page": 64, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "plan", "tree", "tree", "commit"])
    if op == "plan":
        return {"op": op, "n_seq": _log(rng, 1, 2048), "nodes": _log(rng, 1, 64)}
    d = rng.choice([32, 64, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([r for r in (1, 1, 2, 4, 8) if r * kv_heads <= 32])
    kind = rng.choice(["f32", "bf16"])
    if op == "commit":
        while True:
            case = {"op": op, "n_seq": _log(rng, 1, 256), "nodes": _log(rng, 1, 64), "layers": rng.randint(1, 16), "kv_heads": kv_heads,
                    "d": d, "page": rng.choice([8, 16, 32, 64, 128]), "type": kind}
            if _commit_cache(case) <= _commit_cache(listed()[-1]):
                return case
    if op in ("norm", "append"):
        rot = rng.choice([d, d // 2, 2 * rng.randint(0, d // 2)])
        case = {"op": op, "tokens": _log(rng, 1, 32749 if op == "append" else 8192), "heads": heads, "kv_heads": kv_heads, "d": d, "rot": rot,
                "interleaved": rng.random() < 0.5, "type": kind}
        if op == "norm":
            case.update(seq_len=rng.choice([1024, 777]), grad=rng.random() < 0.5, fused=rng.random() < 0.5)
        else:
            case.update(slots=case["tokens"] * 2 + rng.randint(0, 999), max_pos=_log(rng, 1024, 131072))
        return case
    cache = rng.choice([kind, "int8"])
    n_seq = _log(rng, 1, 256)
    groups = rng.choice([g for g in (0, 0, 1, 2, 3) if g <= n_seq])
    case = {"op": op, "n_seq": n_seq, "nodes": _log(rng, 1, 64), "groups": groups, "prefix": _log(rng, 1, 8192) if groups else 0,
            "context": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "d": d, "page": rng.choice([8, 16, 32, 64, 128]),
            "type": "f32" if cache == "int8" else kind, "cache": cache}
    most = _tree_numbers(next(c for c in listed() if c["name"] == "tree-documents-bf16"))
    while True:
        now = _tree_numbers(case)
        if now["flops"] <= most["flops"] and now["bytes"] <= most["bytes"] and now["scores"] <= most["scores"]:
            return case
        case["prefix"], case["context"] = case["prefix"] // 2 + (groups > 0), max(1, case["context"] * 2 // 3)


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
    {"norm": _prepare_norm, "append": _prepare_append, "plan": _prepare_plan, "tree": _prepare_tree, "commit": _prepare_commit}[case["op"]](
        case, g, s, seed)
    return s


def _table(rot, max_pos):
    """cos and sin of position x frequency, [max_pos][rot / 2][2], angles taken in 64 bits."""
    if not rot:
        return torch.zeros((max_pos, 0, 2), device="cuda")
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * freq[None, :]
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


def _weights(case, g, s):
    """Norm weights as training leaves them: around one, of either sign now and then."""
    s["q_weight"], s["k_weight"] = (1.0 + 0.3 * _normal(g, (case["d"],), "f32") for _ in range(2))


def _prepare_norm(case, g, s, _):
    n, d, qw, kw, kind = case["tokens"], case["d"], case["heads"] * case["d"], case["kv_heads"] * case["d"], case["type"]
    if case["fused"]:      # Q and K are column blocks of one projection output [Q | K | V]
        x = _normal(g, (n, qw + 2 * kw), kind)
        s["q"], s["k"] = x[:, :qw], x[:, qw:qw + kw]
    else:
        s["q"], s["k"] = _normal(g, (n, qw), kind), _normal(g, (n, kw), kind)
    _weights(case, g, s)
    s["table"] = _table(case["rot"], case["seq_len"])
    if case["grad"]:
        s["dq_out"], s["dk_out"] = _normal(g, (n, qw), kind), _normal(g, (n, kw), kind)
        grads = torch.empty_like(x) if case["fused"] else None
        s["dq"], s["dk"] = (grads[:, :qw], grads[:, qw:qw + kw]) if case["fused"] else (torch.empty_like(s["q"]), torch.empty_like(s["k"]))
        s["dq_weight"], s["dk_weight"] = (torch.empty(d, device="cuda") for _ in range(2))
    else:
        s["q_out"], s["k_out"] = torch.empty((n, qw), dtype=s["q"].dtype, device="cuda"), torch.empty((n, kw), dtype=s["q"].dtype, device="cuda")


def _prepare_append(case, g, s, _):
    n, qw, kw = case["tokens"], case["heads"] * case["d"], case["kv_heads"] * case["d"]
    s["q"], s["k"], s["v"] = (_normal(g, (n, w), case["type"]) for w in (qw, kw, kw))
    _weights(case, g, s)
    s["table"] = _table(case["rot"], case["max_pos"])
    s["positions"] = _ints(g, n, 0, case["max_pos"] - 1)
    s["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:n].contiguous()
    if n > 8:
        s["slots"][3::97] = -1          # padding rows: nothing is written for them
    s["q_out"] = torch.empty_like(s["q"])
    s["kcache"], s["vcache"] = (torch.zeros((case["slots"], kw), dtype=s["q"].dtype, device="cuda") for _ in range(2))


def _trees(case, g, s):
    """Drafts of 1 .. nodes tokens: token 0 is the one sampled last, each other one descends from one of the eight
    before it.  Rows of the requests one after another, with rows to spare behind the last."""
    n, nodes = case["n_seq"], case["nodes"]
    count = _ints(g, n, 1, nodes)
    count[0] = nodes
    s["words"] = (nodes + 31) // 32
    s["rows"] = n * nodes
    s["cu"] = torch.cat([count.new_zeros(1), count.cumsum(0).to(INTS)])
    i = torch.arange(nodes, device="cuda")[None, :].expand(n, nodes)
    back = (torch.rand((n, nodes), generator=g, device="cuda") * i.clamp(max=8)).long().clamp(max=7)
    parent = torch.where(i > 0, i - 1 - torch.minimum(back, (i - 1).clamp(min=0)), -1).to(INTS)
    s["parents"] = torch.full((s["rows"],), -1, dtype=INTS, device="cuda")
    s["parents"][:int(s["cu"][-1])] = parent[i < count[:, None]]
    return count


def _prepare_plan(case, g, s, _):
    n = case["n_seq"]
    count = _trees(case, g, s)
    first = _ints(g, n, 0, 8192)
    row = torch.arange(s["rows"], device="cuda")
    seq = (torch.searchsorted(s["cu"].long(), row, right=True) - 1).clamp(max=n - 1)
    s["positions"] = torch.where(row < s["cu"][-1], first[seq] + row - s["cu"][seq], 0).to(INTS)      # as the page plan leaves them
    s["tree_positions"] = torch.zeros(s["rows"], dtype=INTS, device="cuda")
    s["masks"] = torch.zeros((s["rows"], s["words"]), dtype=INTS, device="cuda")


def _prepare_tree(case, g, s, _):
    n, groups, page, d, nodes = case["n_seq"], case["groups"], case["page"], case["d"], case["nodes"]
    kw = case["kv_heads"] * d
    count = _trees(case, g, s)
    s["masks"] = _plain_masks(s)[0]
    s["ctx"] = _ints(g, n, 0 if n > 16 else 1, case["context"])
    s["ctx"][0] = case["context"]
    refused = torch.rand(n, generator=g, device="cuda") < (0.04 if n > 16 else 0.0)     # no pages were left for these drafts
    s["lens"] = torch.where(refused, s["ctx"], s["ctx"] + count).to(INTS)
    most = case["context"] + nodes
    pp, po = -(-case["prefix"] // page), -(-most // page)
    s["group_begin"] = s["prefix_table"] = s["prefix_lens"] = None
    n_pages = groups * pp + n * po + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(INTS)
    if groups:
        s["prefix_lens"] = _ints(g, groups, max(1, case["prefix"] - case["prefix"] // 8), case["prefix"])
        s["prefix_lens"][0] = case["prefix"]
        s["group_begin"] = torch.tensor([i * n // groups for i in range(groups + 1)], dtype=INTS, device="cuda")
        s["prefix_table"] = ids[:groups * pp].view(groups, pp).contiguous()
    s["block_table"] = ids[groups * pp:groups * pp + n * po].view(n, po).contiguous()
    rows = n_pages * page
    s["q"] = _normal(g, (s["rows"], case["heads"] * d), case["type"])
    s["kscale"] = s["vscale"] = None
    if case["cache"] == "int8":
        for x in ("k", "v"):
            s[x + "cache"] = torch.randint(-127, 128, (rows, kw), generator=g, device="cuda", dtype=torch.int8)
            s[x + "scale"] = torch.rand((rows, case["kv_heads"]), generator=g, device="cuda") * 0.01 + 0.012
    else:
        s["kcache"], s["vcache"] = (_normal(g, (rows, kw), case["cache"]) for _ in range(2))
    s["out"] = torch.zeros_like(s["q"])                   # rows behind the last draft stay as they are
    s["lse"] = torch.zeros((s["rows"], case["heads"]), dtype=torch.float32, device="cuda")


COMMIT_CONTEXT = 64


def _commit_pages(case):
    return -(-(COMMIT_CONTEXT + case["nodes"]) // case["page"])


def _commit_cache(case):
    return case["n_seq"] * _commit_pages(case) * case["page"] * case["layers"] * 2 * case["kv_heads"] * case["d"] * BYTES[case["type"]]


def _commit_trees(case, seed):
    """Drafts whose first half (rounded up) is the likeliest chain and whose rest are shorter ways that leave it, each
    no deeper than the chain is long; an accepted node (-1: none) for each request.  Lists of parents, and leaves."""
    r = random.Random(seed)
    parents, leaves = [], []
    for _ in range(case["n_seq"]):
        n = r.randint(1, case["nodes"])
        chain = (n + 1) // 2
        depth, tree = list(range(chain)), [i - 1 for i in range(chain)]
        for i in range(chain, n):
            on = i > chain and r.random() < 0.6 and depth[i - 1] + 1 < chain
            parent = i - 1 if on else r.randrange(max(1, chain - 1))
            tree.append(parent)
            depth.append(depth[parent] + 1)
        parents.append(tree)
        leaves.append(r.randrange(n) if r.random() < 0.95 else -1)
    return parents, leaves


def _prepare_commit(case, g, s, seed):
    n, page, kw = case["n_seq"], case["page"], case["kv_heads"] * case["d"]
    parents, leaves = _commit_trees(case, seed)
    count = torch.tensor([len(t) for t in parents], dtype=INTS)
    s["rows"], s["words"] = n * case["nodes"], (case["nodes"] + 31) // 32
    s["cu"] = torch.cat([count.new_zeros(1), count.cumsum(0).to(INTS)]).cuda()
    s["parents"] = torch.full((s["rows"],), -1, dtype=INTS, device="cuda")
    s["parents"][:int(count.sum())] = torch.tensor([p for t in parents for p in t], dtype=INTS).cuda()
    s["leaf"] = torch.tensor(leaves, dtype=INTS).cuda()
    s["masks"] = _plain_masks(s)[0]
    s["ctx"] = _ints(g, n, 0, COMMIT_CONTEXT)
    s["lens"] = (s["ctx"] + count.cuda()).to(INTS)
    most = _commit_pages(case)
    ids = torch.randperm(n * most, generator=g, device="cuda").to(INTS)
    s["block_table"] = ids.view(n, most).contiguous()
    s["free"] = torch.full((n * most + 5,), -1, dtype=INTS, device="cuda")
    s["free_count"] = torch.tensor([5], dtype=INTS, device="cuda")
    s["free"][:5] = torch.arange(n * most, n * most + 5, device="cuda")
    rows = (n * most + 5) * page
    s["caches"] = [tuple(_normal(g, (rows, kw), case["type"]) for _ in range(2)) for _ in range(case["layers"])]
    s["lens_out"], s["counts"] = torch.empty(n, dtype=INTS, device="cuda"), torch.empty(4, dtype=INTS, device="cuda")


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "plan": _own_plan, "tree": _own_tree, "commit": _own_commit}[op](s, _library())
    return {"norm": _plain_norm, "append": _plain_append, "plan": _plain_plan, "tree": _plain_tree, "commit": _plain_commit}[op](s)


def _library():
    if "attn_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "pure-c-llm_b200"))
    import attn_b200
    return attn_b200


def _rope_shape(s, A, seq_len, max_pos):
    c = s["case"]
    return A.RopeShape(c["tokens"], seq_len, c["heads"], c["kv_heads"], c["d"], c["rot"], int(c["interleaved"]), max_pos,
                       s["q"].stride(0), s["k"].stride(0), 0, 0, 0)


def _own_norm(s, A):
    if "shape" not in s:
        s["shape"] = _rope_shape(s, A, s["case"]["seq_len"], s["case"]["seq_len"])
        s["norm"] = A.HeadNorm.of(s["q_weight"], s["k_weight"], EPS)
        if s["case"]["grad"]:
            s["work"] = torch.empty(A.norm_rope_bwd_workspace_bytes(s["shape"]), dtype=torch.uint8, device="cuda")
    if not s["case"]["grad"]:
        A.norm_rope_t(s["shape"], s["norm"], s["table"], None, s["q"], s["k"], s["q_out"], s["k_out"])
        return s["q_out"], s["k_out"]
    A.norm_rope_bwd_t(s["shape"], s["norm"], s["table"], None, s["q"], s["k"], s["dq_out"], s["dk_out"], s["dq"], s["dk"],
                      dq_weight=s["dq_weight"], dk_weight=s["dk_weight"], workspace=s["work"])
    return s["dq"], s["dk"], s["dq_weight"], s["dk_weight"]


def _own_append(s, A):
    if "shape" not in s:
        s["shape"] = _rope_shape(s, A, 0, s["case"]["max_pos"])
        s["norm"] = A.HeadNorm.of(s["q_weight"], s["k_weight"], EPS)
        s["cache"] = A.PageCache.of(s["kcache"], s["vcache"])
    A.norm_rope_append_t(s["shape"], s["norm"], s["cache"], s["table"], s["positions"], s["slots"], s["q"], s["k"], s["v"], s["q_out"])
    return s["q_out"], s["kcache"], s["vcache"]


def _own_plan(s, A):
    A.tree_plan_t(s["cu"], s["parents"], s["positions"], s["tree_positions"], s["masks"])
    return s["tree_positions"], s["masks"]


def _own_tree(s, A):
    if "shape" not in s:
        c = s["case"]
        s["cache"] = A.PageCache.of(s["kcache"], s["vcache"], s["kscale"], s["vscale"])
        s["shape"] = A.TreeShape(c["n_seq"], s["rows"], c["groups"], c["heads"], c["kv_heads"], c["d"], A.BF16 if c["type"] == "bf16" else A.F32,
                                 c["page"], s["prefix_table"].shape[1] if c["groups"] else 0, s["block_table"].shape[1], c["prefix"],
                                 c["context"] + c["nodes"], c["nodes"], s["words"], 0, 0, 0.0)
        s["work"] = torch.empty(A.tree_decode_workspace_bytes(s["shape"], s["cache"]), dtype=torch.uint8, device="cuda")
    A.tree_decode_t(s["shape"], s["cache"], s["q"], s["cu"], s["ctx"], s["lens"], s["masks"], s["block_table"], s["out"], lse=s["lse"],
                    group_begin=s["group_begin"], prefix_table=s["prefix_table"], prefix_lens=s["prefix_lens"], workspace=s["work"])
    return s["out"], s["lse"]


def _own_commit(s, A):
    if "shape" not in s:
        c = s["case"]
        s["shape"] = A.PageShape(c["n_seq"], c["page"], s["block_table"].shape[1], s["rows"], s["free"].numel(), 0)
        s["kv"] = A.cache_array([A.PageCache.of(k, v) for k, v in s["caches"]])
    c = s["case"]
    A.tree_commit_t(s["shape"], s["kv"], c["kv_heads"], c["d"], s["cu"], s["ctx"], s["lens"], s["leaf"], s["masks"], s["block_table"], s["free"],
                    s["free_count"], s["lens_out"], s["counts"])
    return [s["lens_out"], s["counts"], s["free"]] + [x for pair in s["caches"] for x in pair]


def _turn(x, case, cs, transpose=False):
    """x: (tokens, heads, d); cs: (tokens, rot / 2, 2)."""
    rot = case["rot"]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    if transpose:
        sin = -sin
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _heads(x, d):
    return x.float().reshape(x.shape[0], -1, d)


def _plain_normed(x, weight, case, cs):
    x = _heads(x, case["d"])
    return _turn(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight, case, cs).flatten(1)


def _plain_norm(s):
    c = s["case"]
    cs = s["table"][torch.arange(c["tokens"], device="cuda") % c["seq_len"]]
    if not c["grad"]:
        s["q_out"].copy_(_plain_normed(s["q"], s["q_weight"], c, cs))
        s["k_out"].copy_(_plain_normed(s["k"], s["k_weight"], c, cs))
        return s["q_out"], s["k_out"]
    for x in ("q", "k"):
        v, g = _heads(s[x], c["d"]), _turn(_heads(s["d" + x + "_out"], c["d"]), c, cs, transpose=True)
        r = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
        s["d" + x + "_weight"].copy_((g * v * r).sum((0, 1), dtype=torch.float64))
        g = g * s[x + "_weight"]
        s["d" + x].copy_((r * (g - v * (r * r * (g * v).mean(-1, keepdim=True)))).flatten(1))
    return s["dq"], s["dk"], s["dq_weight"], s["dk_weight"]


def _plain_append(s):
    c = s["case"]
    cs = s["table"][s["positions"].long()]
    s["q_out"].copy_(_plain_normed(s["q"], s["q_weight"], c, cs))
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["kcache"][at] = _plain_normed(s["k"], s["k_weight"], c, cs)[keep].to(s["k"].dtype)
    s["vcache"][at] = s["v"][keep]
    return s["q_out"], s["kcache"], s["vcache"]


def _plain_masks(s):
    """Masks (rows, words) and depths (rows) from the parents; zeros behind the last draft."""
    rows, words, cu = s["rows"], s["words"], s["cu"].long()
    row = torch.arange(rows, device="cuda")
    seq = (torch.searchsorted(cu, row, right=True) - 1).clamp(max=cu.numel() - 2)
    index = row - cu[seq]
    real = row < cu[-1]
    bits = torch.zeros((rows, 32 * words), dtype=torch.bool, device="cuda")
    at, depth = torch.where(real, index, -1), torch.zeros(rows, dtype=torch.int64, device="cuda")
    for _ in range(32 * words):                   # one generation up a turn; no draft is deeper than its nodes
        there = at >= 0
        bits[row, at.clamp(min=0)] |= there
        at = torch.where(there, s["parents"].long()[(cu[seq] + at).clamp(0, rows - 1)], -1)
        depth += (at >= 0)
    word = (bits.view(rows, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(INTS), depth


def _plain_plan(s):
    masks, depth = _plain_masks(s)
    cu = s["cu"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = (torch.searchsorted(cu, row, right=True) - 1).clamp(max=cu.numel() - 2)
    real = row < cu[-1]
    s["tree_positions"].copy_(torch.where(real, s["positions"].long()[cu[seq]] + depth, s["tree_positions"].long()))
    s["masks"].copy_(torch.where(real[:, None], masks, s["masks"]))
    return s["tree_positions"], s["masks"]


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


def _softmax_parts(scores, hidden, values):
    """Maximum, sum and weighted values of the scores that are not hidden."""
    scores = scores.masked_fill(hidden, -math.inf)
    m = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - m).masked_fill(hidden, 0.0)
    return m, p.sum(-1, keepdim=True), p @ values


def _plain_tree(s):
    c = s["case"]
    n, groups, h, hk, d, page, nodes = c["n_seq"], c["groups"], c["heads"], c["kv_heads"], c["d"], c["page"], c["nodes"]
    r, cu, words = h // hk, s["cu"].long(), s["words"]
    index = torch.arange(nodes, device="cuda")[None, :]
    there = index < (cu[1:] - cu[:-1])[:, None]                                     # (n, nodes)
    row = torch.where(there, cu[:-1, None] + index, 0)
    q = (s["q"].float() * (1.0 / math.sqrt(d))).view(-1, hk, r, d)[row]             # (n, nodes, hk, r, d)
    own_q = q.permute(0, 2, 1, 3, 4).reshape(n, hk, nodes * r, d)
    rows = _rows(s["block_table"], page, c["context"] + nodes)
    t = torch.arange(c["context"] + nodes, device="cuda")
    bit = t[None, :] - s["ctx"].long()[:, None]                                     # (n, T): place behind the context
    word = s["masks"][row]                                                          # (n, nodes, words)
    at = bit.clamp(0, 32 * words - 1)
    seen = torch.gather(word, 2, (at // 32)[:, None, :].expand(n, nodes, -1)) >> (at % 32)[:, None, :].to(INTS) & 1
    seen = (seen.bool() | (bit < 0)[:, None, :]) & (t[None, :] < s["lens"].long()[:, None])[:, None, :]
    hidden = ~seen[:, None, :, None, :].expand(n, 1, nodes, r, -1).reshape(n, 1, nodes * r, -1)
    mo, lo, oo = _softmax_parts(own_q @ _values(s, "k", rows).transpose(-1, -2), hidden, _values(s, "v", rows))
    if groups:
        begin = s["group_begin"].long()
        group = torch.searchsorted(begin, torch.arange(n, device="cuda"), right=True) - 1
        place = torch.arange(n, device="cuda") - begin[group]
        most = -(-n // groups)
        # queries of a group side by side: the prefix is read once for all of them
        qg = q.new_zeros(groups, most, hk, nodes * r, d)
        qg[group, place] = own_q
        qg = qg.transpose(1, 2).reshape(groups, hk, most * nodes * r, d)
        rows = _rows(s["prefix_table"], page, c["prefix"])
        hidden = (torch.arange(c["prefix"], device="cuda")[None, :] >= s["prefix_lens"][:, None])[:, None, None, :]
        parts = _softmax_parts(qg @ _values(s, "k", rows).transpose(-1, -2), hidden, _values(s, "v", rows))
        mp, lp, op = (x.view(groups, hk, most, nodes * r, -1).transpose(1, 2)[group, place] for x in parts)
        m = torch.maximum(mp, mo)
        wp, wo = torch.exp(mp - m), torch.exp(mo - m)
        mo, lo, oo = m, lp * wp + lo * wo, op * wp + oo * wo
    out = torch.where(lo > 0, oo / lo, 0.0).view(n, hk, nodes, r, d).transpose(1, 2).reshape(n, nodes, h * d)
    lse = torch.where(lo > 0, mo + torch.log(lo), -math.inf).view(n, hk, nodes, r).transpose(1, 2).reshape(n, nodes, h)
    s["out"][row[there]] = out[there].to(s["out"].dtype)
    s["lse"][row[there]] = lse[there]
    return s["out"], s["lse"]


def _plain_commit(s):
    c = s["case"]
    n, page, words = c["n_seq"], c["page"], s["words"]
    cu, ctx, lens, leaf = (s[x].long() for x in ("cu", "ctx", "lens", "leaf"))
    line = s["masks"][(cu[:-1] + leaf.clamp(min=0))]                                # (n, words)
    bit = torch.arange(32 * words, device="cuda")
    on = (line[:, bit // 32] >> (bit % 32).to(INTS)[None, :] & 1).bool() & (bit[None, :] <= leaf[:, None])
    count = on.sum(-1)
    place = on.cumsum(-1) - 1                                                       # of an accepted node behind the context
    table = s["block_table"].long()
    t_from, t_to = ctx[:, None] + bit[None, :], ctx[:, None] + place
    last = table.shape[1] - 1
    row = lambda t: table.gather(1, (t // page).clamp(0, last)) * page + t % page   # noqa: E731
    src, dst = row(t_from)[on], row(t_to.clamp(min=0))[on]
    for k, v in s["caches"]:
        k[dst] = k[src]
        v[dst] = v[src]
    after = ctx + count
    keep, held = (after + page - 1) // page, (lens + page - 1) // page
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    back = s["block_table"][(column >= keep[:, None]) & (column < held[:, None])]
    base = s["free_count"].long()
    s["free"][base + torch.arange(back.numel(), device="cuda")] = back
    s["lens_out"].copy_(after)
    returned = (held - keep).sum().view(1)
    s["counts"].copy_(torch.cat([base + returned, count.sum().view(1), (leaf < 0).sum().view(1), returned]))
    return [s["lens_out"], s["counts"], s["free"]] + [x for pair in s["caches"] for x in pair]


# ---------------------------------------------------------------------------
# exact: the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None                     # whole numbers
    s = prepare(case, seed)
    return {"tree": _exact_tree, "commit": _exact_commit}.get(case["op"], _exact_norm)(case, s)


def _exact_norm(case, s):
    n, d, rot = case["tokens"], case["d"], case["rot"]
    position = torch.arange(n, device="cuda") % case["seq_len"] if case["op"] == "norm" else s["positions"].long()
    turn = torch.view_as_complex(s["table"].double())[position][:, None, :] if rot else None
    first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(0, rot // 2, device="cuda")
    second = first + (1 if case["interleaved"] else rot // 2)

    def forward(x, weight):
        y = x.reshape(n, -1, d)
        y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * weight
        if not rot:
            return y.reshape(n, -1)
        # each pair is one complex number, turned by multiplication with cos + i sin
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.index_copy(2, first, z.real).index_copy(2, second, z.imag)
        return y.reshape(n, -1)

    if case["op"] == "norm" and case["grad"]:
        grads = []
        for x in ("q", "k"):
            v, w = s[x].double().requires_grad_(), s[x + "_weight"].double().requires_grad_()
            grads.append(torch.autograd.grad(forward(v, w), (v, w), s["d" + x + "_out"].double()))
        return grads[0][0], grads[1][0], grads[0][1], grads[1][1]
    q, k = forward(s["q"].double(), s["q_weight"].double()), forward(s["k"].double(), s["k_weight"].double())
    if case["op"] == "norm":
        return q, k
    kc, vc = s["kcache"].double(), s["vcache"].double()
    keep = (s["slots"] >= 0).nonzero().flatten()
    kc[s["slots"][keep]], vc[s["slots"][keep]] = k[keep], s["v"].double()[keep]
    return q, kc, vc


def _exact_tree(case, s):
    h, hk, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    r = h // hk
    out, lse = s["out"].double(), s["lse"].double()
    cu, ctx, lens, parents = (s[x].tolist() for x in ("cu", "ctx", "lens", "parents"))
    begin = s["group_begin"].tolist() if case["groups"] else []
    prefixes = s["prefix_lens"].tolist() if case["groups"] else []
    t = torch.arange(case["prefix"] + case["context"] + case["nodes"], device="cuda")

    def fetch(x, at):
        v = s[x + "cache"][at].double().view(-1, hk, d)
        return (v if s[x + "scale"] is None else v * s[x + "scale"][at].double()[..., None]).transpose(0, 1)

    def slots(line, count):
        return line.long()[t[:count] // page] * page + t[:count] % page

    for i in range(case["n_seq"]):
        n = cu[i + 1] - cu[i]
        sees = np.zeros((n, max(lens[i] - ctx[i], 0)), bool)
        for a in range(n):
            b = a
            while b >= 0:
                if b < sees.shape[1]:
                    sees[a, b] = True
                b = parents[cu[i] + b]
        at = slots(s["block_table"][i], lens[i])
        before = 0
        for g in range(case["groups"]):
            if begin[g] <= i < begin[g + 1]:
                at, before = torch.cat([slots(s["prefix_table"][g], prefixes[g]), at]), prefixes[g]
        k, v = fetch("k", at), fetch("v", at)
        q = s["q"][cu[i]:cu[i + 1]].double().view(n, hk, r, d).permute(1, 0, 2, 3).reshape(hk, n * r, d)
        x = (q @ k.transpose(1, 2) / math.sqrt(d)).view(hk, n, r, -1)
        x[..., before + ctx[i]:].masked_fill_(~torch.from_numpy(sees).cuda()[None, :, None, :], -math.inf)
        if x.shape[-1] == 0:
            o, e = q.new_zeros(hk, n, r, d), q.new_full((hk, n, r), -math.inf)
        else:
            e = torch.logsumexp(x, -1)
            p = torch.where(torch.isneginf(e)[..., None], 0.0, torch.exp(x - e[..., None]))
            o = (p.view(hk, n * r, -1) @ v).view(hk, n, r, d)
        out[cu[i]:cu[i + 1]] = o.permute(1, 0, 2, 3).reshape(n, h * d)
        lse[cu[i]:cu[i + 1]] = e.permute(1, 0, 2).reshape(n, h)
    return out, lse


def _exact_commit(case, s):
    cu, ctx, parents, leaf, table, page = *(s[x].tolist() for x in ("cu", "ctx", "parents", "leaf", "block_table")), case["page"]
    src, dst = [], []
    for i in range(case["n_seq"]):
        path, at = [], leaf[i]
        while at >= 0:
            path.insert(0, at)
            at = parents[cu[i] + at]
        for to, at in enumerate(path):
            a, b = ctx[i] + at, ctx[i] + to
            src.append(table[i][a // page] * page + a % page)
            dst.append(table[i][b // page] * page + b % page)
    after = []
    for x in (x for pair in s["caches"] for x in pair):
        moved = x.double()
        moved[torch.tensor(dst, dtype=torch.int64, device="cuda")] = x.double()[torch.tensor(src, dtype=torch.int64, device="cuda")]
        after.append(moved)
    return [None, None, None] + after


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def _tree_numbers(c):
    """Drafts, contexts and prefixes at their expected lengths: every K and V row once, q, out and lse once."""
    rows = c["n_seq"] * (c["nodes"] + 1) / 2
    prefix, own_rows = c["groups"] * c["prefix"] * (15 / 16 if c["groups"] > 1 else 1.0), c["n_seq"] * (c["context"] + 1) / 2 + rows
    row = 2 * c["kv_heads"] * (c["d"] * BYTES[c["cache"]] + (4 if c["cache"] == "int8" else 0))
    act = rows * (c["heads"] * (2 * c["d"] * BYTES[c["type"]] + 4) + 4 * ((c["nodes"] + 31) // 32))
    scores = rows * c["heads"] * (prefix / max(c["groups"], 1) + (c["context"] + 1) / 2 + math.log2(c["nodes"] + 1))
    padded = c["n_seq"] * c["nodes"] * c["heads"] * (c["prefix"] + c["context"] + c["nodes"])       # the plain form's
    return {"bytes": (prefix + own_rows) * row + 4 * (prefix + own_rows) / c["page"] + act, "flops": 4 * c["d"] * scores, "scores": padded}


def work(case):
    c = case
    if c["op"] == "tree":
        w = _tree_numbers(c)
        return {"bytes": w["bytes"], "flops": w["flops"]}
    if c["op"] == "plan":
        rows = c["n_seq"] * (c["nodes"] + 1) / 2
        return {"bytes": rows * (4 + 4 + 4 * ((c["nodes"] + 31) // 32)) + c["n_seq"] * 8, "flops": 0}
    if c["op"] == "commit":
        parents, leaves = _commit_trees(c, 0)
        moved = 0
        for tree, leaf in zip(parents, leaves):
            path = []
            while leaf >= 0:
                path.append(leaf)
                leaf = tree[leaf]
            moved += sum(a != b for a, b in enumerate(reversed(path)))
        row = 2 * c["kv_heads"] * c["d"] * BYTES[c["type"]] * c["layers"]
        return {"bytes": 2 * moved * row + c["n_seq"] * (20 + 4 * ((c["nodes"] + 31) // 32)), "flops": 0}
    e, width, heads = BYTES[c["type"]], (c["heads"] + c["kv_heads"]) * c["d"], c["tokens"] * (c["heads"] + c["kv_heads"])
    flops = heads * (4 * c["d"] + 3 * c["rot"])
    if c["op"] == "norm":
        rows = min(c["tokens"], c["seq_len"])
        return {"bytes": (3 if c["grad"] else 2) * c["tokens"] * width * e + rows * c["rot"] * 4, "flops": flops * (3 if c["grad"] else 1)}
    rows = min(c["tokens"], c["max_pos"])
    return {"bytes": 2 * c["tokens"] * (width + c["kv_heads"] * c["d"]) * e + rows * c["rot"] * 4 + c["tokens"] * 12, "flops": flops}
