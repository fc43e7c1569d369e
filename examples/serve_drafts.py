"""One attention layer of a server that checks drafted token trees, on the library's paged entry points.

    python examples/serve_drafts.py [--requests 6] [--prompt 200] [--steps 8] [--nodes 12] [--cache f32|int8]

All requests share a prompt, whose keys and values lie in pages that no request owns.  A step gives every request a tree of
drafted tokens: the page plan finds cache rows for them, the tree plan their positions and who sees whom, the projection
and the normed rotary append put their keys and values there, and the tree decode attends from every draft to the prompt,
the request's context and the drafts it descends from.  (A real server would compare the model's answers with the drafts;
here a random draft is the last right one.)  The commit moves its path's rows together and hands pages back.  The outputs
of every step and the cache after the last are checked against 64-bit forms that know only the accepted tokens.
"""
import argparse
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "pure-c-llm_b200"))
import attn_b200 as A  # noqa: E402

HEADS, D = 8, 64
DIM = HEADS * D
PAGE = 8
EPS = 1e-6


def normed(x, weight, turn):
    """64-bit heads of rows (n, DIM), normed, weighted and turned (turn: (n, D / 2) complex)."""
    y = x.double().view(-1, HEADS, D)
    y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * turn[:, None]
    return torch.cat([z.real, z.imag], -1)


def main(requests=6, prompt=200, steps=8, nodes=12, cache="f32", seed=0):
    """Runs the loop and returns the largest error of outputs and cache rows, relative to the largest value."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    ints = dict(dtype=torch.int32, device="cuda")

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)

    wq, wk, wv = (normal(DIM, DIM, std=1 / math.sqrt(DIM)) for _ in range(3))
    q_weight, k_weight = (1 + normal(D, std=0.2) for _ in range(2))
    norm = A.HeadNorm.of(q_weight, k_weight, EPS)
    most = prompt + steps * nodes
    table = A.rope_table_t(A.RopeConfig(D, most, A.ROPE_PLAIN, 0, 10000.0, 1.0, 0.0, 0.0, 1.0))
    turn = torch.view_as_complex(table.double())

    # the cache: pages 0 .. prompt_pages - 1 hold the prompt, the others are free
    prompt_pages, own_pages = -(-prompt // PAGE), -(-(steps * nodes) // PAGE)
    total = prompt_pages + requests * own_pages
    dtype = torch.int8 if cache == "int8" else torch.float32
    kc, vc = (torch.zeros((total * PAGE, DIM), dtype=dtype, device="cuda") for _ in range(2))
    ks, vs = ((torch.zeros((total * PAGE, HEADS), device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
    kv = A.PageCache.of(kc, vc, ks, vs)
    text = normal(prompt, DIM)
    q, k, v = A.qkv_proj_t(text, wq, wk, wv)
    A.norm_rope_append_t(A.RopeShape(prompt, prompt, HEADS, HEADS, D, D, 0, most, 0, 0, 0, 0, 0), norm, kv, table, None,
                         torch.arange(prompt, device="cuda"), q, k, v, torch.empty_like(q))

    rows = requests * nodes
    lens, block_table = torch.zeros(requests, **ints), torch.full((requests, own_pages), -1, **ints)
    free_pages, free_count = torch.arange(prompt_pages, total, **ints), torch.tensor([total - prompt_pages], **ints)
    pos_base = torch.full((requests,), prompt, **ints)
    pages = A.PageShape(requests, PAGE, own_pages, rows, free_pages.numel(), 0)
    plans = [A.page_outputs(pages) for _ in range(2)]
    after = [(torch.empty(requests, **ints), torch.empty(4, **ints)) for _ in range(2)]
    words = -(-nodes // 32)
    tree = A.TreeShape(requests, rows, 1, HEADS, HEADS, D, A.F32, PAGE, prompt_pages, own_pages, prompt, own_pages * PAGE, nodes, words, 0, 0, 0.0)
    group_begin, prefix_lens = torch.tensor([0, requests], **ints), torch.tensor([prompt], **ints)
    prefix_table = torch.arange(prompt_pages, **ints).view(1, -1)
    work = torch.empty(A.tree_decode_workspace_bytes(tree, kv), dtype=torch.uint8, device="cuda")
    shape = A.RopeShape(rows, 0, HEADS, HEADS, D, D, 0, most, 0, 0, 0, 0, 0)

    # what the check knows: the prompt's and each request's accepted keys and values
    if cache == "f32":
        known_k, known_v = normed(k, k_weight, turn[:prompt]), v.double().view(-1, HEADS, D)
    else:
        known_k, known_v = (x[:prompt].double().view(-1, HEADS, D) * s[:prompt].double()[..., None] for x, s in ((kc, ks), (vc, vs)))
    history = [([], []) for _ in range(requests)]
    worst = 0.0

    def compare(got, want):
        nonlocal worst
        err = float((got.double() - want).abs().max() / want.abs().max())
        worst = worst if err <= worst else err            # (also an error that is no number)

    out = torch.empty((rows, DIM), device="cuda")
    for step in range(steps):
        trees = []
        for _ in range(requests):
            n = rnd.randint(1, nodes)
            trees.append([-1] + [rnd.randrange(max(0, i - 4), i) for i in range(1, n)])
        flat = [p for t in trees for p in t]
        parents = torch.tensor(flat + [-1] * (rows - len(flat)), **ints)
        new = torch.tensor([len(t) for t in trees], **ints)
        plan = A.page_plan_t(pages, lens, new, free_pages, free_count, block_table, plans[step % 2], pos_base=pos_base)
        masks = torch.empty((rows, words), **ints)
        A.tree_plan_t(plan["cu_new"], parents, plan["positions"], plan["positions"], masks)
        x = normal(rows, DIM)
        q, k, v = A.qkv_proj_t(x, wq, wk, wv)
        turned = A.norm_rope_append_t(shape, norm, kv, table, plan["positions"], plan["slot_map"], q, k, v, torch.empty_like(q))
        A.tree_decode_t(tree, kv, turned, plan["cu_new"], lens, plan["lens"], masks, block_table, out, group_begin=group_begin,
                        prefix_table=prefix_table, prefix_lens=prefix_lens, workspace=work)
        leaves = [rnd.randrange(len(t)) for t in trees]
        lens_out, counts = after[step % 2]
        first = 0
        for s, (t, leaf) in enumerate(zip(trees, leaves)):
            path, at = [], leaf
            while at >= 0:
                path.insert(0, at)
                at = t[at]
            r = [first + i for i in path]
            positions = torch.tensor([prompt + len(history[s][0]) + i for i in range(len(path))], device="cuda")
            if cache == "f32":
                new_k, new_v = normed(k[r], k_weight, turn[positions]), v[r].double().view(-1, HEADS, D)
            else:                         # what the cache holds for them, before the commit moves it
                slots = plan["slot_map"][r]
                new_k, new_v = (c[slots].double().view(-1, HEADS, D) * z[slots].double()[..., None] for c, z in ((kc, ks), (vc, vs)))
            history[s][0].extend(new_k)
            history[s][1].extend(new_v)
            all_k, all_v = torch.cat([known_k, torch.stack(history[s][0])]), torch.cat([known_v, torch.stack(history[s][1])])
            query = normed(q[r[-1:]], q_weight, turn[positions[-1:]])[0]
            p = torch.softmax(torch.einsum("hd,nhd->hn", query, all_k) / math.sqrt(D), dim=-1)
            compare(out[r[-1]], torch.einsum("hn,nhd->hd", p, all_v).flatten())
            first += len(t)
        A.tree_commit_t(pages, A.cache_array([kv]), HEADS, D, plan["cu_new"], lens, plan["lens"], torch.tensor(leaves, **ints), masks, block_table,
                        free_pages, plan["counts"][:1], lens_out, counts)
        lens, free_count = lens_out, counts[:1]

    for s in range(requests):             # the cache holds the accepted tokens, in order, and every page has one owner
        n = len(history[s][0])
        if int(lens[s]) != n:
            return math.inf
        t = torch.arange(n, device="cuda")
        at = block_table[s].long()[t // PAGE] * PAGE + t % PAGE
        for c, z, want in ((kc, ks, history[s][0]), (vc, vs, history[s][1])):
            held = c[at].double().view(-1, HEADS, D) * (1 if z is None else z[at].double()[..., None])
            compare(held, torch.stack(want))
    held = [int(block_table[s, j]) for s in range(requests) for j in range(-(-int(lens[s]) // PAGE))]
    if sorted(held + free_pages[:int(free_count)].tolist()) != list(range(prompt_pages, total)):
        return math.inf
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--nodes", type=int, default=12)
    ap.add_argument("--cache", choices=("f32", "int8"), default="f32")
    a = ap.parse_args()
    print(f"largest relative error of outputs and cache: {main(a.requests, a.prompt, a.steps, a.nodes, a.cache):.2e}")
