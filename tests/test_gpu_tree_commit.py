"""Acceptance of drafted trees and the commit of the accepted paths, bit for bit against the oracle; and a whole step."""

import numpy as np
import pytest
import torch

from oracle import tree as otree
from pagelora_amd import fused_ops
from pagelora_amd.attention_backend import PagedDecodeAttention, kv_append
from pagelora_amd.kv_pool import PagedKVPool, Request
from pagelora_amd.speculative import accept_tree, commit_tree
from tests.test_gpu_tree_attention import random_parents

pytestmark = pytest.mark.gpu


def draft(trees, rng, hit=0.7, vocab=50):
    """Random trees whose drafts the picks often follow: (parents, tokens, picks, qo_indptr), equal siblings among them."""
    parents = sum((random_parents(n, rng) for n in trees if n), [])
    ptr = [0] + [int(x) for x in np.cumsum(trees)]
    picks = rng.integers(0, vocab, ptr[-1])
    tokens = rng.integers(0, vocab, ptr[-1])
    for a, e in zip(ptr, ptr[1:]):
        for i in range(a, e):
            if parents[i] >= 0 and rng.random() < hit:
                tokens[i] = picks[a + parents[i]]
    return parents, tokens.tolist(), picks.tolist(), ptr


def on(device, parents, tokens, picks, ptr):
    t = lambda x, d: torch.tensor(x, dtype=d, device=device)  # noqa: E731
    return t(tokens, torch.int64), t(parents, torch.int32), t(picks, torch.int64), t(ptr, torch.int32)


def check_accept(got, parents, tokens, picks, ptr, max_path):
    path, count, kept = otree.accept(tokens, parents, picks, ptr, max_path)
    assert got.path.cpu().tolist() == path
    assert got.count.cpu().tolist() == count
    assert got.tokens.cpu().tolist() == kept


@pytest.mark.parametrize("trees", [[1], [8], [64], [65], [300], [0, 5, 0, 64, 130, 1], [3] * 200])
@pytest.mark.parametrize("max_path", [1, 4, 64, 70])
def test_accept(gpu_device, trees, max_path):
    d = draft(trees, np.random.default_rng(sum(trees) + max_path))
    check_accept(accept_tree(*on(gpu_device, *d), max_path=max_path), *d, max_path)


@pytest.mark.parametrize("n", [64, 65, 200])
def test_accept_a_whole_chain(gpu_device, n):
    rng = np.random.default_rng(n)
    picks = rng.integers(0, 2**60, n).tolist()  # ids past 32 bits
    d = (list(range(-1, n - 1)), [7] + picks[:-1], picks, [0, n])
    check_accept(accept_tree(*on(gpu_device, *d), max_path=n), *d, n)


def test_accept_takes_the_first_of_equal_children_and_ignores_other_parents(gpu_device):
    # children of the root: 2, 3 (equal tokens), 4; node 1 is a second root, node 5 names itself, node 6 a later node
    parents, tokens = [-1, -1, 0, 0, 0, 5, 9, 2], [1, 9, 9, 9, 9, 9, 9, 4]
    picks = [9, 9, 4, 5, 6, 9, 9, 8]
    got = accept_tree(*on(gpu_device, parents, tokens, picks, [0, 8]), max_path=8)
    assert got.path.tolist() == [[0, 2, 7] + [-1] * 5] and got.tokens.tolist() == [[9, 4, 8] + [-1] * 5]


def test_accept_into_given_tensors_in_a_graph(gpu_device):
    rng = np.random.default_rng(0)
    d = draft([20, 70], rng)
    args = on(gpu_device, *d)
    out = accept_tree(*args, max_path=9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accept_tree(*args, max_path=9, out=out)
    for _ in range(3):
        d = draft([20, 70], rng)
        for t, x in zip(args, on(gpu_device, *d)):
            t.copy_(x)
        out.path.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_accept(out, *d, 9)


def commit_case(trees, lens, page, layers, hkv, dim, dtype, seed, max_path):
    rng = np.random.default_rng(seed)
    totals = [a + b for a, b in zip(trees, lens)]
    pages = [-(-n // page) for n in totals]
    ids = rng.permutation(sum(pages) + 4)
    kv = [0] + [int(x) for x in np.cumsum(pages)]
    last = [n - (p - 1) * page if p else 0 for n, p in zip(totals, pages)]
    qo = [0] + [int(x) for x in np.cumsum(trees)]
    gen = torch.Generator().manual_seed(seed)
    cache = torch.randn((layers, len(ids), 2, page, hkv, dim), generator=gen).to(dtype)
    count, path = [], []
    for n in trees:
        c = int(rng.integers(0, min(n, max_path) + 1))
        p = sorted(rng.choice(n, size=c, replace=False).tolist()) if c else []
        count.append(c)
        path.append(p + [-1] * (max_path - c))
    return cache, qo, kv, ids[: kv[-1]].tolist(), last, path, count


def commit_args(device, qo, kv, ids, last, path, count):
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return (t(path), t(count)), dict(qo_indptr=t(qo), paged_kv_indptr=t(kv), paged_kv_indices=t(ids),
                                     paged_kv_last_page_len=t(last))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("heads", [(2, 64), (8, 128), (5, 8)])
def test_commit(gpu_device, dtype, page, heads):
    """Ascending paths whose slots are sources of earlier tokens, empty ones, requests without a prefix."""
    hkv, dim = heads
    cache, *rest = commit_case([1, 8, 0, 64, 30], [5, 0, 17, 3, 40], page, 3, hkv, dim, dtype, seed=page, max_path=30)
    want = otree.commit(cache.float().numpy(), *rest)
    got = cache.to(gpu_device)
    args, kw = commit_args(gpu_device, *rest)
    commit_tree(got, *args, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(got.float().cpu().numpy(), want)


@pytest.mark.parametrize("n", [64, 65, 150])
def test_commit_long_paths(gpu_device, n):
    """More tokens than one window, each slot the source of the token before."""
    cache, qo, kv, ids, last, _, _ = commit_case([n + 1], [10], 16, 2, 2, 64, torch.bfloat16, n, max_path=n)
    rest = (qo, kv, ids, last, [[0] + list(range(2, n + 1))], [n])
    want = otree.commit(cache.float().numpy(), *rest)
    got = cache.to(gpu_device)
    args, kw = commit_args(gpu_device, *rest)
    commit_tree(got, *args, **kw)
    assert np.array_equal(got.float().cpu().numpy(), want)


def test_commit_bad_paths_and_tables_move_nothing_astray(gpu_device):
    cache, qo, kv, ids, last, _, _ = commit_case([8, 8, 8, 8], [20] * 4, 16, 2, 2, 64, torch.bfloat16, 1, max_path=4)
    path = [[0, 3, 1, 5], [0, 8, 3, 4], [-1, 2, 3, 4], [0, 2, 7, 1]]  # below k, past the tree, negative, below k
    rest = (qo, kv, ids, last, path, [4, 4, 9, 4])
    want = otree.commit(cache.float().numpy(), *rest)
    got = cache.to(gpu_device)
    args, kw = commit_args(gpu_device, *rest)
    commit_tree(got, *args, **kw)
    assert np.array_equal(got.float().cpu().numpy(), want)
    # tables: pages outside the pool, more pages than listed, a tree longer than its sequence
    for name, value in (("paged_kv_indices", [10**6, -4] * (len(ids) // 2) + [10**6] * (len(ids) % 2)),
                        ("paged_kv_indptr", [-3, 10**8, 10**8, 5, 2]), ("qo_indptr", [0, 4000, 8000, 8000, -1])):
        got = cache.to(gpu_device)
        args, kw = commit_args(gpu_device, qo, kv, ids, last, [[0, 2, 5, 7]] * 4, [4] * 4)
        kw[name] = torch.tensor(value, dtype=torch.int32, device=gpu_device)
        commit_tree(got, *args, **kw)
        torch.cuda.synchronize()
        if name != "paged_kv_indptr":
            assert torch.equal(got.cpu(), cache), name


def test_commit_one_layer_and_in_a_graph(gpu_device):
    cache, *rest = commit_case([16, 5], [9, 40], 16, 2, 2, 64, torch.bfloat16, 5, max_path=5)
    want = otree.commit(cache.float().numpy(), *rest)
    args, kw = commit_args(gpu_device, *rest)
    got = cache.to(gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        commit_tree(got[1], *args, **kw)
    for _ in range(3):
        got.copy_(cache)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(got[1].float().cpu().numpy(), want[1]) and torch.equal(got[0].cpu(), cache[0])


def test_refusals(gpu_device):
    d = on(gpu_device, [-1, 0], [1, 2], [2, 3], [0, 2])
    with pytest.raises(ValueError, match="max_path"):
        accept_tree(*d, max_path=0)
    with pytest.raises(ValueError, match="tokens"):
        accept_tree(d[0].int(), *d[1:], max_path=2)
    with pytest.raises(ValueError, match="picks"):
        accept_tree(d[0], d[1], d[2][:1], d[3], max_path=2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        accept_tree(d[0].cpu(), *d[1:], max_path=2)
    with pytest.raises(RuntimeError, match="same ROCm device"):
        accept_tree(d[0], d[1], d[2].cpu(), d[3], max_path=2)
    out = accept_tree(*d, max_path=2)
    with pytest.raises(ValueError, match="out.path"):
        accept_tree(*d, max_path=3, out=out)
    cache, *rest = commit_case([4], [9], 16, 2, 2, 64, torch.bfloat16, 5, max_path=5)
    args, kw = commit_args(gpu_device, *rest)
    with pytest.raises(RuntimeError, match="ROCm device"):
        commit_tree(cache, *args, **kw)
    cache = cache.to(gpu_device)
    with pytest.raises(ValueError, match="cache must be"):
        commit_tree(cache[0, 0], *args, **kw)
    with pytest.raises(ValueError, match="path"):
        commit_tree(cache, args[0].long(), args[1], **kw)
    with pytest.raises(ValueError, match="entries"):
        commit_tree(cache, args[0], torch.cat((args[1], args[1])), **kw)
    with pytest.raises(NotImplementedError):
        commit_tree(cache.double(), *args, **kw)


@pytest.mark.parametrize("layers", [2])
def test_a_speculative_step_decodes_what_single_steps_do(gpu_device, layers):
    """Prefix, tree, verification, commit, truncate and fork, with attention as the whole model.

    A toy target: the K, V and query of a token are a table's rows at its id and
    position, a layer's output feeds a random head, the pick is its argmax.  The
    tokens that steps over trees decode are those of decoding one token at a
    time, up to a pick whose two best logits lie within what the attention's
    bf16 roundings can move them (2^-9 of the output in each of 1024 dims, by
    chance: 0.003 of the logits' spread and hardly ever 0.02).
    """
    hq, hkv, d, ps, vocab = 8, 2, 64, 16, 96
    gen = torch.Generator().manual_seed(0)
    emb = (torch.randn((layers, 3, vocab, hq, d), generator=gen)).to(torch.bfloat16).to(gpu_device)
    rot = (torch.randn((layers, 1024, hq, d), generator=gen) * 0.3).to(torch.bfloat16).to(gpu_device)
    head = torch.randn((hq * d, vocab), generator=gen).to(gpu_device)

    def rows(layer, which, tokens, pos):
        return (emb[layer, which, tokens] + rot[layer, pos])[:, : hkv if which else hq].contiguous()

    def new_pool():
        return PagedKVPool(num_layers=layers, capacity_pages=64, page_size=ps, num_kv_heads=hkv, head_dim=d,
                           dtype=torch.bfloat16, device=gpu_device)

    def forward(pool, be, reqs, tokens, pos, slots, attend):
        page = torch.tensor([s[0] for s in slots], device=gpu_device)
        off = torch.tensor([s[1] for s in slots], device=gpu_device)
        x = torch.zeros((len(tokens), hq * d), device=gpu_device)
        for layer in range(layers):
            kv_append(pool.layer_cache(layer), rows(layer, 1, tokens, pos), rows(layer, 2, tokens, pos), page, off,
                      num_kv_heads=hkv, head_dim=d, page_size=ps)
            x += attend(rows(layer, 0, tokens, pos), pool.layer_cache(layer)).reshape(len(tokens), -1).float()
        logits = x @ head
        return fused_ops.greedy_argmax(logits), logits

    def table(pool, reqs):
        return dict(zip(("paged_kv_indptr", "paged_kv_indices", "paged_kv_last_page_len"),
                        (torch.from_numpy(x) for x in pool.tables(reqs))))

    def single(pool, reqs, tokens, steps):
        be = PagedDecodeAttention(device=gpu_device, workspace_mb=4, num_qo_heads=hq, num_kv_heads=hkv, head_dim=d,
                                  page_size=ps)
        out, gaps = [[] for _ in reqs], [[] for _ in reqs]
        for _ in range(steps):
            pos = torch.tensor([r.length for r in reqs], device=gpu_device)
            for r in reqs:
                pool.reserve(r, 1)
            be.plan_decode(**table(pool, reqs))
            picks, logits = forward(pool, be, reqs, torch.tensor(tokens, device=gpu_device), pos,
                                    [r.slot(r.length - 1, ps) for r in reqs],
                                    lambda q, c: be.run_decode(q, c))
            tokens = picks.tolist()
            top = logits.topk(2, dim=1).values
            gap = ((top[:, 0] - top[:, 1]) / logits.std(dim=1)).tolist()
            for b, t in enumerate(tokens):
                out[b].append(t)
                gaps[b].append(gap[b])
        return out, gaps

    def prompt(pool, lens):
        be = PagedDecodeAttention(device=gpu_device, workspace_mb=4, num_qo_heads=hq, num_kv_heads=hkv, head_dim=d,
                                  page_size=ps)
        reqs = [Request() for _ in lens]
        for r, n in zip(reqs, lens):
            pool.reserve(r, n)
            toks, pos = (torch.arange(n, device=gpu_device) * 31) % vocab, torch.arange(n, device=gpu_device)
            be.plan_prefill(qo_indptr=torch.tensor([0, n], dtype=torch.int32), **table(pool, [r]))
            forward(pool, be, [r], toks, pos, [r.slot(i, ps) for i in range(n)], be.run_prefill)
        return reqs

    lens, first, steps = [30, 47], [5, 11], 24
    pool = new_pool()
    want, gaps = single(pool, prompt(pool, lens), first, steps)

    pool = new_pool()
    reqs = prompt(pool, lens)
    reqs = pool.fork(reqs) + reqs  # the forks decode; their origins stay
    origins = reqs[2:]
    before = [pool.cache[:, r.own_pages].clone() for r in origins]
    reqs = reqs[:2]
    be = PagedDecodeAttention(device=gpu_device, workspace_mb=4, num_qo_heads=hq, num_kv_heads=hkv, head_dim=d,
                              page_size=ps)
    got, tokens = [[], []], list(first)
    rng = np.random.default_rng(1)
    turns, most = 0, 0
    while min(len(g) for g in got) < steps:
        # drafts: the right continuation on one branch here and there, wrong ones beside it
        trees, parents, drafts, depth = [], [], [], []
        for b in range(2):
            n = int(rng.integers(1, 12))
            p = random_parents(n, rng)
            dep = [0] * n
            for i in range(1, n):
                dep[i] = dep[p[i]] + 1
            right = [tokens[b]] + want[b][len(got[b]):] + [0] * 40
            trees.append(n)
            parents += p
            depth += dep
            drafts += [tokens[b]] + [right[dep[i]] if rng.random() < 0.6 else int(rng.integers(0, vocab))
                                     for i in range(1, n)]
        qo = torch.tensor([0, trees[0], sum(trees)], dtype=torch.int32)
        base = [r.length for r in reqs]
        pos = torch.tensor([base[0 if i < trees[0] else 1] + x for i, x in enumerate(depth)], device=gpu_device)
        for r, n in zip(reqs, trees):
            pool.reserve(r, n)
        t = table(pool, reqs)
        par = torch.tensor(parents, dtype=torch.int32)
        be.plan_tree(qo_indptr=qo, **t, tree_parents=par)
        slots = [reqs[b].slot(base[b] + i, ps) for b in range(2) for i in range(trees[b])]
        drafts = torch.tensor(drafts, device=gpu_device)
        picks, _ = forward(pool, be, reqs, drafts, pos, slots, be.run_tree)
        acc = accept_tree(drafts, par.to(gpu_device), picks, qo.to(gpu_device), max_path=12)
        commit_tree(pool.cache, acc.path, acc.count, qo_indptr=qo.to(gpu_device),
                    **{k: v.to(gpu_device) for k, v in t.items()})
        for b, (r, c) in enumerate(zip(reqs, acc.count.tolist())):
            pool.truncate(r, base[b] + c)
            new = acc.tokens[b, :c].tolist()
            got[b] += new
            tokens[b] = new[-1]
            most = max(most, c)
        turns += 1
    assert most > 2 and turns < steps
    for b in range(2):
        first_off = next((i for i in range(steps) if got[b][i] != want[b][i]), None)
        assert first_off is None or (first_off > 4 and gaps[b][first_off] < 0.02), (b, first_off)
    for r, x in zip(origins, before):
        assert torch.equal(pool.cache[:, r.own_pages], x)
