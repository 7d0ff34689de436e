"""The operators of one step of tree-speculative decoding over the paged KV
cache, as timed cases.

A drafter proposes a small tree of tokens per request; the target model runs
all of them in one pass.  Four operators, in the order a step calls them:

* ``attn``: one layer's attention of every tree token over its request's pages
  and its own ancestors in the tree,
* ``accept``: the longest path of the tree that the target's greedy picks
  follow,
* ``commit``: that path's K/V moved together behind the committed tokens, in
  every layer,
* ``copy``: pages copied in every layer (a request forked for another
  continuation).

``own`` False computes them from elementary torch operations, True through the
package's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

HEAD_DIM = 128
VOCAB = 151936
# (q heads, kv heads): the GQA ratios and the MHA that the decode and prefill cases have
HEADS = {"gqa4": (32, 8), "mha": (32, 32), "gqa7": (28, 4)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one chat, a draft of 8 tokens: latency and launches
        {"name": "attn_1x8_2048_gqa4_bf16", "kind": "attn", "heads": "gqa4", "requests": 1, "min_tree": 8,
         "max_tree": 8, "min_len": 2048, "max_len": 2048, "page": 16, "dtype": "bf16"},
        # one request with a long context and a wide tree: the work split over the kv axis
        {"name": "attn_1x64_32768_gqa4_bf16", "kind": "attn", "heads": "gqa4", "requests": 1, "min_tree": 64,
         "max_tree": 64, "min_len": 32768, "max_len": 32768, "page": 16, "dtype": "bf16"},
        # a medium batch of ragged chats and ragged trees, a GQA ratio that is no power of two
        {"name": "attn_23_ragged_gqa7_bf16", "kind": "attn", "heads": "gqa7", "requests": 23, "min_tree": 1,
         "max_tree": 27, "min_len": 33, "max_len": 4099, "page": 16, "dtype": "bf16"},
        # no GQA: the most cache per query
        {"name": "attn_8x32_4096_mha_fp16", "kind": "attn", "heads": "mha", "requests": 8, "min_tree": 32,
         "max_tree": 32, "min_len": 4001, "max_len": 4096, "page": 16, "dtype": "fp16"},
        # a full batch of long chats, the largest call
        {"name": "attn_64x16_8192_gqa4_bf16", "kind": "attn", "heads": "gqa4", "requests": 64, "min_tree": 16,
         "max_tree": 16, "min_len": 2048, "max_len": 8192, "page": 16, "dtype": "bf16"},
        # the verification of one small tree and of a large batch of large ones
        {"name": "accept_1x8", "kind": "accept", "requests": 1, "min_tree": 8, "max_tree": 8},
        {"name": "accept_256x64", "kind": "accept", "requests": 256, "min_tree": 33, "max_tree": 64},
        # one request's accepted tokens, and a full batch's, through 36 layers
        {"name": "commit_1x8_36_bf16", "kind": "commit", "heads": "gqa4", "requests": 1, "min_tree": 8, "max_tree": 8,
         "max_path": 4, "min_len": 77, "max_len": 77, "layers": 36, "page": 16, "dtype": "bf16"},
        {"name": "commit_64x32_36_bf16", "kind": "commit", "heads": "gqa4", "requests": 64, "min_tree": 17,
         "max_tree": 32, "max_path": 8, "min_len": 33, "max_len": 130, "layers": 36, "page": 16, "dtype": "bf16"},
        # the partial page of one forked request; many forks at once; the pages of long prompts moved (no GQA)
        {"name": "copy_1_36_bf16", "kind": "copy", "heads": "gqa4", "pages": 1, "layers": 36, "page": 16,
         "dtype": "bf16"},
        {"name": "copy_32_32_mha_fp16", "kind": "copy", "heads": "mha", "pages": 32, "layers": 32, "page": 16,
         "dtype": "fp16"},
        {"name": "copy_256_36_bf16", "kind": "copy", "heads": "gqa4", "pages": 256, "layers": 36, "page": 16,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "accept", "commit", "copy"))
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(sorted(DTYPES))
    hq, hkv = HEADS[heads]
    requests, tree = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
    page = rng.choice((16, 16, 16, 32, 8, 1))
    trees = {"min_tree": max(1, tree // rng.choice((1, 1, 2, 16))), "max_tree": tree}
    if kind == "attn":
        hi = _log_int(rng, 1, 32768)
        # no more cache and no more products than the largest listed call
        hi = min(hi, 64 * 5120 * 8 // (requests * hkv), 64 * 5120 * 16 * 32 // (requests * tree * hq))
        return {"kind": kind, "heads": heads, "requests": requests, **trees, "min_len": max(1, hi // rng.choice((1, 2, 64))),
                "max_len": hi, "page": page, "dtype": dtype}
    if kind == "accept":
        return {"kind": kind, "requests": _log_int(rng, 1, 256), **trees}
    layers = rng.choice((1, 28, 32, 36))
    if kind == "commit":
        # as much cache at the most as the largest listed call's
        hi = _log_int(rng, 1, 130)
        hi = min(hi, 64 * 130 * 36 * 8 // (requests * layers * hkv))
        return {"kind": kind, "heads": heads, "requests": requests, **trees, "max_path": rng.choice((1, 3, 8)),
                "min_len": max(1, hi // 2), "max_len": max(1, hi), "layers": layers, "page": page, "dtype": dtype}
    most = 256 * 36 * 8 * 16 // (layers * hkv * page)
    return {"kind": kind, "heads": heads, "pages": _log_int(rng, 1, min(most, 1500)), "layers": layers, "page": page,
            "dtype": dtype}


# ------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers evenly over lo .. hi, in no order."""
    at = sorted(range(n), key=lambda i: (i * 7919 + 13) % (n + 1))
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in at]


def _sizes(case):
    """(tree tokens, committed tokens) of each request."""
    n = case["requests"]
    return _spread(n, case["min_tree"], case["max_tree"]), _spread(n, case["min_len"], case["max_len"])[::-1]


def _tables(trees, lens, page, gen, extra=0):
    """Host tables of requests of ``lens`` committed tokens and ``trees`` tree
    tokens behind them, pages in no order; (tables, pages of the pool)."""
    totals = torch.tensor([a + b for a, b in zip(trees, lens)])
    pages = (totals + page - 1) // page
    pool = int(pages.sum()) + extra
    zero = torch.zeros(1, dtype=torch.int64)
    return {"qo_indptr": torch.cat((zero, torch.tensor(trees).cumsum(0))).int(),
            "paged_kv_indptr": torch.cat((zero, pages.cumsum(0))).int(),
            "paged_kv_indices": torch.randperm(pool, generator=gen)[: pool - extra].int(),
            "paged_kv_last_page_len": (totals - (pages - 1) * page).int()}, pool


def _parents(trees, gen):
    """A random tree per request: node 0 is the root, every other node's parent an earlier node; parents [requests, widest], -2 past a tree."""
    width = max(trees)
    at = torch.arange(width)
    up = (torch.rand((len(trees), width), generator=gen) * at).long().clamp(max=width - 1)
    up[:, 0] = -1
    return torch.where(at[None, :] < torch.tensor(trees)[:, None], up, -2)


def _packed(padded, trees):
    return padded[torch.arange(padded.shape[1])[None, :] < torch.tensor(trees)[:, None]]


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "accept":
        trees, _ = _sizes({**case, "min_len": 1, "max_len": 1})
        up = _parents(trees, gen)
        picks = torch.randint(0, VOCAB, up.shape, generator=gen)
        # two of three drafts are what the target picks after their parent
        right = torch.rand(up.shape, generator=gen) < 0.67
        drafts = torch.where(right, picks.gather(1, up.clamp(min=0)), torch.randint(0, VOCAB, up.shape, generator=gen))
        indptr = torch.cat((torch.zeros(1, dtype=torch.int64), torch.tensor(trees).cumsum(0))).int()
        return {"kind": "accept", "width": up.shape[1], "qo_indptr": indptr.cuda(), "parents": _packed(up, trees).int().cuda(),
                "tokens": _packed(drafts, trees).cuda(), "picks": _packed(picks, trees).cuda()}
    hq, hkv = HEADS[case["heads"]]
    dtype, page = DTYPES[case["dtype"]], case["page"]
    if case["kind"] == "copy":
        n = case["pages"]
        ids = torch.randperm(2 * n + 1, generator=gen).tolist()
        cache = torch.randn((case["layers"], 2 * n + 1, 2, page, hkv, HEAD_DIM), dtype=dtype, device="cuda", generator=dev)
        return {"kind": "copy", "cache": cache, "src": ids[:n], "dst": ids[n: 2 * n]}
    trees, lens = _sizes(case)
    tables, pool = _tables(trees, lens, page, gen, extra=3)
    if case["kind"] == "commit":
        # accepted paths whose tokens lie behind every slot they go to
        width = case["max_path"]
        counts = _counts(case)
        path = torch.full((len(trees), width), -1)
        for b, (t, c) in enumerate(zip(trees, counts)):
            path[b, 0] = 0
            path[b, 1:c] = c + torch.randperm(t - c, generator=gen)[: c - 1].sort().values
        cache = torch.randn((case["layers"], pool, 2, page, hkv, HEAD_DIM), dtype=dtype, device="cuda", generator=dev)
        return {"kind": "commit", "cache": cache, "path": path.int().cuda(), "count": torch.tensor(counts).int().cuda(),
                "tables": {k: v.cuda() for k, v in tables.items()}}
    up = _parents(trees, gen)
    q = torch.randn((sum(trees), hq, HEAD_DIM), dtype=dtype, device="cuda", generator=dev)
    cache = torch.randn((pool, 2, page, hkv, HEAD_DIM), dtype=dtype, device="cuda", generator=dev)
    state = {"kind": "attn", "q": q, "cache": cache, "heads": (hq, hkv), "tables": {k: v.cuda() for k, v in tables.items()},
             "sees": _ancestors(up).cuda(), "width": up.shape[1], "most": max(a + b for a, b in zip(trees, lens))}
    if own:
        # the step's plan, which all layers of a decoder share
        from pagelora_amd.attention_backend import PagedDecodeAttention

        state["backend"] = PagedDecodeAttention(device="cuda", workspace_mb=1, num_qo_heads=hq, num_kv_heads=hkv,
                                                head_dim=HEAD_DIM, page_size=page)
        state["backend"].plan_tree(**tables, tree_parents=_packed(up, trees).int())
    return state


def _counts(case):
    trees, _ = _sizes(case)
    return [min(c, (t + 1) // 2) for t, c in zip(trees, _spread(len(trees), 1, case["max_path"]))]


def _ancestors(up):
    """sees[r, i, j]: node j is node i or one of its ancestors."""
    n, width = up.shape
    sees = torch.zeros((n, width, width), dtype=torch.bool)
    sees[:, 0, 0] = True
    for i in range(1, width):
        live = up[:, i] >= 0
        sees[live, i] = sees[live, up[live, i]]
        sees[live, i, i] = True
    return sees


# --------------------------------------------------------------------- runs
def run(state):
    return _RUNS[state["kind"]](state)


def _run_attn(state):
    if own:
        return state["backend"].run_tree(state["q"], state["cache"])
    q, cache, t = state["q"], state["cache"], state["tables"]
    hq, hkv = state["heads"]
    dim, page, width = q.shape[2], cache.shape[2], state["width"]
    # every request's tokens side by side: [requests, positions, kv heads, dim]
    starts, pages = t["paged_kv_indptr"][:-1].long(), t["paged_kv_indptr"].diff().long()
    at = torch.arange(-(-state["most"] // page), device=q.device)
    ids = t["paged_kv_indices"].long()[starts[:, None] + at.clamp(max=pages[:, None] - 1)]
    k, v = (cache[ids, i].flatten(1, 2).transpose(1, 2).float() for i in (0, 1))
    # the trees' queries padded to the widest: [requests, kv heads, tokens x group, dim]
    first, trees = t["qo_indptr"][:-1].long(), t["qo_indptr"].diff().long()
    node = torch.arange(width, device=q.device)
    inside = node < trees[:, None]
    rows = (first[:, None] + node).clamp(max=q.shape[0] - 1)
    g = hq // hkv
    qs = q[rows].float().unflatten(2, (hkv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = torch.matmul(qs, k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    total = (pages - 1) * page + t["paged_kv_last_page_len"]
    pos = torch.arange(k.shape[2], device=q.device)
    j = pos - (total - trees)[:, None]  # the tree's nodes by position
    sees = torch.where((j < 0)[:, None], True, state["sees"].gather(2, j.clamp(0, width - 1)[:, None].expand(-1, width, -1)))
    sees &= (pos < total[:, None])[:, None]
    scores = scores.unflatten(2, (width, g)).masked_fill_(~sees[:, None, :, None], -math.inf).flatten(2, 3)
    p = torch.exp(scores - scores.amax(3, keepdim=True).clamp(min=-3e38))
    out = torch.matmul(p, v) / p.sum(3, keepdim=True).clamp(min=1e-38)
    return out.unflatten(2, (width, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)[inside].to(q.dtype)


def _run_accept(state):
    if own:
        from pagelora_amd.speculative import accept_tree

        got = accept_tree(state["tokens"], state["parents"], state["picks"], state["qo_indptr"], max_path=state["width"])
        return {"path": got.path, "count": got.count, "tokens": got.tokens}
    first, trees, width = state["qo_indptr"][:-1].long(), state["qo_indptr"].diff().long(), state["width"]
    node = torch.arange(width, device=first.device)
    rows = (first[:, None] + node).clamp(max=state["tokens"].numel() - 1)
    up = torch.where(node < trees[:, None], state["parents"][rows].long(), -2)
    tokens, picks = state["tokens"][rows], state["picks"][rows]
    # step[r, i]: the first child of node i that the target picks after it; past the tree where there is none
    good = (up[:, None, :] == node[:, None]) & (tokens[:, None, :] == picks[:, :, None]) & (node[None, None, :] > node[:, None])
    step = torch.where(good, node, width).amin(2)
    step = torch.cat((step, torch.full_like(step[:, :1], width)), 1)
    path = torch.zeros_like(first)[:, None]
    while path.shape[1] < width:  # twice as far with every turn
        path = torch.cat((path, step.gather(1, path)), 1)
        step = step.gather(1, step)
    path = path[:, :width]
    kept = path < width
    out = torch.where(kept, picks.gather(1, path.clamp(max=width - 1)), -1)
    return {"path": torch.where(kept, path, -1).int(), "count": kept.sum(1).int(), "tokens": out}


def _run_commit(state):
    t, cache, path = state["tables"], state["cache"], state["path"]
    if own:
        from pagelora_amd.speculative import commit_tree

        commit_tree(cache, path, state["count"], **t)
        return cache
    page = cache.shape[3]
    starts, pages = t["paged_kv_indptr"][:-1].long(), t["paged_kv_indptr"].diff().long()
    base = (pages - 1) * page + t["paged_kv_last_page_len"] - t["qo_indptr"].diff()
    k = torch.arange(path.shape[1], device=path.device)
    live = k < state["count"][:, None]
    # an entry past the path moves the root onto itself
    src, dst = (base[:, None] + torch.where(live, x, 0) for x in (path.long(), k[None, :].expand_as(path)))
    slots = [(t["paged_kv_indices"].long()[starts[:, None] + x // page].flatten(), (x % page).flatten()) for x in (src, dst)]
    moved = cache[:, slots[0][0], :, slots[0][1]]
    cache[:, slots[1][0], :, slots[1][1]] = moved
    return cache


def _run_copy(state):
    if own:
        from pagelora_amd.kv_pool import kv_copy_pages

        kv_copy_pages(state["cache"], state["src"], state["dst"])
        return state["cache"]
    cache = state["cache"]
    src, dst = (torch.tensor(x, device=cache.device) for x in (state["src"], state["dst"]))
    cache.index_copy_(1, dst, cache.index_select(1, src))
    return cache


_RUNS = {"attn": _run_attn, "accept": _run_accept, "commit": _run_commit, "copy": _run_copy}


# --------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "accept":
        trees, _ = _sizes({**case, "min_len": 1, "max_len": 1})
        # a node's parent, token and pick; a row's path, count and tokens
        return {"bytes": sum(trees) * 20 + len(trees) * (4 + 12 * max(trees) + 4), "flops": 0}
    hq, hkv = HEADS[case["heads"]]
    token = 2 * hkv * HEAD_DIM * 2
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * case["page"] * token, "flops": 0}
    trees, lens = _sizes(case)
    if case["kind"] == "commit":
        return {"bytes": 2 * sum(c - 1 for c in _counts(case)) * case["layers"] * token + 4 * len(trees) * case["max_path"],
                "flops": 0}
    # every token's K and V once, q and the output once; products over the committed tokens and the node itself
    pairs = sum(t * (n + 1) for t, n in zip(trees, lens))
    return {"bytes": sum(t + n for t, n in zip(trees, lens)) * token + 4 * sum(trees) * hq * HEAD_DIM,
            "flops": 4 * pairs * hq * HEAD_DIM}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "accept":
        return _exact_accept(s)
    if case["kind"] in ("commit", "copy"):
        return None  # values are moved, none is computed
    t = {k: v.tolist() for k, v in s["tables"].items()}
    (hq, hkv), page, outs = s["heads"], s["cache"].shape[2], []
    for r, last in enumerate(t["paged_kv_last_page_len"]):
        ids = t["paged_kv_indices"][t["paged_kv_indptr"][r]: t["paged_kv_indptr"][r + 1]]
        total = (len(ids) - 1) * page + last
        kv = s["cache"][torch.tensor(ids, device="cuda")].double()
        k, v = (kv[:, i].reshape(-1, hkv, HEAD_DIM)[:total] for i in (0, 1))
        q = s["q"][t["qo_indptr"][r]: t["qo_indptr"][r + 1]].double()
        n = q.shape[0]
        seen = torch.ones((n, total), dtype=torch.bool, device="cuda")
        seen[:, total - n:] = s["sees"][r, :n, :n]
        heads = []
        for h in range(hq):
            x = q[:, h] @ k[:, h // (hq // hkv)].T.contiguous() * HEAD_DIM ** -0.5
            heads.append(torch.softmax(torch.where(seen, x, -math.inf), 1) @ v[:, h // (hq // hkv)])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)


def _exact_accept(s):
    ptr, up, tokens, picks = (s[k].tolist() for k in ("qo_indptr", "parents", "tokens", "picks"))
    paths = []
    for a, e in zip(ptr, ptr[1:]):
        path = [0]
        while True:
            here = path[-1]
            found = [i for i in range(here + 1, e - a) if up[a + i] == here and tokens[a + i] == picks[a + here]]
            if not found:
                break
            path.append(found[0])
        paths.append(path)
    pad = lambda x: x + [-1] * (s["width"] - len(x))  # noqa: E731
    return {"path": torch.tensor([pad(p) for p in paths], dtype=torch.int32), "count": torch.tensor([len(p) for p in paths], dtype=torch.int32),
            "tokens": torch.tensor([pad([picks[a + i] for i in p]) for a, p in zip(ptr, paths)])}
