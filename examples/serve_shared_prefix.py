"""One attention layer of a server whose requests share a system prompt, on the library's paged entry points.

    python examples/serve_shared_prefix.py [--requests 8] [--prompt 300] [--steps 40] [--cache f32|int8]

The prompt is projected, turned and attended once: its keys and values go to pages that no request owns, and what its last
row attends to is where every request begins, with a token of its own.  Then every step decodes one token per request: the page plan says where its key and value go, the projection and the rotary append
put them there, and the shared-prefix decode attends to the prompt's rows and the request's own.  Halfway, two requests
end and hand their pages back.  The last step is checked against attention in 64 bits over each request's rows.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "pure-c-llm_b200"))
import attn_b200 as A  # noqa: E402

HEADS, D = 16, 64
DIM = HEADS * D
PAGE = 16


def main(requests=8, prompt=300, steps=40, cache="f32", seed=0):
    """Runs the loop and returns the largest error of the last step, relative to the largest output."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)

    wq, wk, wv, wo = (normal(DIM, DIM, std=1 / math.sqrt(DIM)) for _ in range(4))
    most = prompt + steps
    table = A.rope_table_t(A.RopeConfig(D, most, A.ROPE_PLAIN, 0, 10000.0, 1.0, 0.0, 0.0, 1.0))

    # the cache: pages 0 .. prompt_pages - 1 hold the prompt, the others are free
    prompt_pages, own_pages = -(-prompt // PAGE), -(-steps // PAGE)
    total = prompt_pages + requests * own_pages
    dtype = torch.int8 if cache == "int8" else torch.float32
    kc, vc = (torch.zeros((total * PAGE, DIM), dtype=dtype, device="cuda") for _ in range(2))
    ks, vs = ((torch.zeros((total * PAGE, HEADS), device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
    kv = A.PageCache.of(kc, vc, ks, vs)

    # the prompt: rows 0 .. prompt - 1 of the cache, its own causal attention from the turned projections
    text = normal(prompt, DIM)
    q, k, v = A.qkv_proj_t(text, wq, wk, wv)
    shape = A.RopeShape(prompt, prompt, HEADS, HEADS, D, D, 0, most, 0, 0, 0, 0, 0)
    A.rope_append_t(shape, kv, table, None, torch.arange(prompt, device="cuda"), q, k, v, torch.empty_like(q))
    A.rope_t(shape, table, None, q, k, q, k)
    begin = text[-1] + A.forward_t(q, k, v, HEADS, 1, want_lse=False)[0][-1] @ wo

    # requests: tables, lengths and free pages on the GPU, the plan's outputs of two steps in turn
    ints = dict(dtype=torch.int32, device="cuda")
    lens, block_table = torch.zeros(requests, **ints), torch.full((requests, own_pages), -1, **ints)
    free_pages = torch.arange(prompt_pages, total, **ints)
    free_count = torch.tensor([total - prompt_pages], **ints)
    pos_base = torch.full((requests,), prompt, **ints)
    pages = A.PageShape(requests, PAGE, own_pages, requests, free_pages.numel(), 0)
    plans = [A.page_outputs(pages) for _ in range(2)]
    group_begin, prefix_lens = torch.tensor([0, requests], **ints), torch.tensor([prompt], **ints)
    prefix_table = torch.arange(prompt_pages, **ints).view(1, -1)
    decode = A.PrefixShape(requests, 1, HEADS, HEADS, D, A.F32, PAGE, prompt_pages, own_pages, prompt, steps, 0, 0, 0.0)
    work = torch.empty(A.prefix_decode_workspace_bytes(decode, kv), dtype=torch.uint8, device="cuda")
    shape = A.RopeShape(requests, 0, HEADS, HEADS, D, D, 0, most, 0, 0, 0, 0, 0)

    x, out = begin + normal(requests, DIM), torch.empty((requests, DIM), device="cuda")
    one, end_two = torch.ones(requests, **ints), torch.ones(requests, **ints)
    end_two[:2] = -1
    for step in range(steps):
        plan = A.page_plan_t(pages, lens, end_two if step == steps // 2 else one, free_pages, free_count, block_table,
                             plans[step % 2], pos_base=pos_base)
        lens, free_count = plan["lens"], plan["counts"][:1]
        # a token row per planned token (an ended request has none this step, and begins anew with the next)
        rows = plan["token_seq"].long()
        there = (rows >= 0)[:, None]
        q, k, v = A.qkv_proj_t(x[rows.clamp(min=0)], wq, wk, wv)
        turned = A.rope_append_t(shape, kv, table, plan["positions"], plan["slot_map"], q, k, v, torch.empty_like(q))
        query = torch.zeros((requests + 1, DIM), device="cuda")
        query[torch.where(there[:, 0], rows, requests)] = turned
        A.prefix_decode_t(decode, kv, query, group_begin, prefix_table, prefix_lens, block_table, lens, out, workspace=work)
        if step + 1 < steps:
            x = x + out @ wo
            x = x / x.square().mean(-1, keepdim=True).sqrt()

    # 64-bit attention over the rows that each request sees
    worst = 0.0
    for s in range(requests):
        t = torch.arange(int(lens[s]), device="cuda")
        at = torch.cat([torch.arange(prompt, device="cuda"), block_table[s].long()[t // PAGE] * PAGE + t % PAGE])
        kr, vr = ((c[at].double().view(-1, HEADS, D) * (1 if z is None else z[at].double()[..., None])) for c, z in ((kc, ks), (vc, vs)))
        p = torch.softmax(torch.einsum("hd,nhd->hn", query[s].double().view(HEADS, D), kr) / math.sqrt(D), dim=-1)
        want = torch.einsum("hn,nhd->hd", p, vr).flatten()
        err = float((out[s].double() - want).abs().max() / want.abs().max())
        worst = worst if err <= worst else err            # (also an error that is no number)
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--cache", choices=("f32", "int8"), default="f32")
    a = ap.parse_args()
    print(f"largest relative error of the last step: {main(a.requests, a.prompt, a.steps, a.cache):.2e}")
