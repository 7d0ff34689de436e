"""Plans of trees: captured runs as their sequences grow, fewer nodes than a tree has, runs on other streams."""

import pytest
import torch

from pagelora_amd import _lib
from tests.test_gpu_tree_attention import BF16, F16, backend, check, oracle, tables, tree_case

pytestmark = pytest.mark.gpu


def grown(lens, trees=(6, 9), seed=3):
    """The same trees behind sequences of other lengths, in pools of one size."""
    cases = [tree_case(list(trees), [n + trees[0], n // 2 + trees[1]], 8, 2, 128, 16, BF16, "cpu", seed=seed + n)
             for n in lens]
    pool = max(c["cache_host"].shape[0] for c in cases)
    for c in cases:
        cache = torch.full((pool, *c["cache_host"].shape[1:]), float("nan"), dtype=BF16)
        cache[: c["cache_host"].shape[0]] = c["cache_host"]
        c["cache_host"] = cache
    return cases


def test_a_captured_run_follows_its_sequences_past_any_number_of_pages(gpu_device):
    """The tables list 14 pages when the run is captured, then 17, 40, 300 and 14 again: plans of the same sizes."""
    cases = grown([100, 130, 400, 3000, 100, 2000])
    be = backend(8, 2, 128, 16, gpu_device)
    q, cache = cases[0]["q"].to(gpu_device), cases[0]["cache_host"].to(gpu_device)
    out = torch.empty_like(q)
    be.plan_tree(**tables(cases[0]), tree_parents=cases[0]["parents"])
    be.run_tree_into(q, cache, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.run_tree_into(q, cache, out)
    signature = be.tree_graph_signature()
    for n, c in enumerate(cases):
        q.copy_(c["q_host"])
        cache.copy_(c["cache_host"])
        t = tables(c) if n % 2 == 0 else tables(c, gpu_device)
        be.plan_tree(**t, tree_parents=c["parents"] if n % 2 == 0 else c["parents"].to(gpu_device), max_tree=9)
        assert be.tree_graph_signature() == signature
        for _ in range(2):
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            check(c, out)
        check(c, be.run_tree(q, cache))


def test_a_captured_plan_beside_plans_of_more_pages(gpu_device):
    """A graph of plan and run, replayed after eager plans of the same sizes and more pages: each reads its own page ids."""
    small, large = grown([40, 3000])
    be = backend(8, 2, 128, 16, gpu_device)
    dev = tables(small, gpu_device)
    parents = small["parents"].to(gpu_device)
    q, cache = small["q"].to(gpu_device), small["cache_host"].to(gpu_device)
    out = torch.empty_like(q)

    def step():
        be.plan_tree(**dev, tree_parents=parents, max_tree=9)
        be.run_tree_into(q, cache, out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        be.plan_tree(**tables(large), tree_parents=large["parents"], max_tree=9)
        check(large, be.run_tree(large["q"].to(gpu_device), large["cache_host"].to(gpu_device)))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(small, out)


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("most", [1, 5, 64, 70])
def test_fewer_nodes_planned_than_a_tree_has(gpu_device, most, mask):
    """Device tables and max_tree below a tree's nodes: its first ones are right, the rows behind them stay untouched."""
    case = tree_case([100, 3], [150, 40], 4, 2, 64, 16, F16, gpu_device, seed=most)
    be = backend(4, 2, 64, 16, gpu_device)
    if mask:
        sees = torch.zeros((103, 100), dtype=torch.bool)
        sees[:100] = torch.from_numpy(case["sees"][0])
        sees[100:, :3] = torch.from_numpy(case["sees"][1])
        tree = {"tree_mask": sees.to(gpu_device)}
    else:
        tree = {"tree_parents": case["parents"].to(gpu_device)}
    be.plan_tree(**tables(case, gpu_device), **tree, max_tree=most)
    out = torch.full_like(case["q"], 7.0)
    be.run_tree_into(case["q"], case["cache"], out)
    torch.cuda.synchronize()
    want = torch.from_numpy(oracle(case)[0])
    kept = [(0, min(100, most)), (100, 100 + min(3, most))]
    for a, e in kept:
        err = (out[a:e].double().cpu() - want[a:e]).abs()
        assert (err <= 2.0**-11 * want[a:e].abs() + 1e-4).all()  # weights off by less than 2^-16, values up to 5
    assert (out[kept[0][1]:100] == 7).all() and (out[kept[1][1]:] == 7).all()


@pytest.mark.parametrize("kept", [False, True])
def test_a_plan_made_while_a_run_waits_on_another_stream(gpu_device, kept):
    """The run reads the plan before it, though the next plan of the same sizes is made first; `kept`: in a buffer that
    a captured run reads."""
    a, b = (tree_case([9, 30], [lens, 2000], 8, 2, 128, 16, BF16, gpu_device, seed=lens) for lens in (1990, 300))
    be = backend(8, 2, 128, 16, gpu_device)
    busy = torch.randn((4096, 4096), device=gpu_device)
    if kept:
        be.plan_tree(**tables(a), tree_parents=a["parents"])
        out = be.run_tree(a["q"], a["cache"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            be.run_tree_into(a["q"], a["cache"], out)
    side = torch.cuda.Stream()
    for first, second in ((a, b), (b, a)):
        torch.cuda.synchronize()
        be.plan_tree(**tables(first), tree_parents=first["parents"])
        with torch.cuda.stream(side):
            for _ in range(8):
                torch.mm(busy, busy)  # a millisecond and more each
            waits = [be.run_tree(first["q"], first["cache"]) for _ in range(2)]
        be.plan_tree(**tables(second), tree_parents=second["parents"])
        now = be.run_tree(second["q"], second["cache"])
        with torch.cuda.stream(side):
            be.plan_tree(**tables(first), tree_parents=first["parents"])
            last = be.run_tree(first["q"], first["cache"])
        torch.cuda.synchronize()
        for out in (*waits, last):
            check(first, out)
        check(second, now)


@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_deep_trees_by_parents_and_by_mask(gpu_device, kind):
    """Masks of many words, packed on one walk to the root: the same bits as from the mask that says the same."""
    n = 5000 if kind == "chain" else 3001
    parents = torch.arange(-1, n - 1) if kind == "chain" else (torch.rand(n, generator=torch.Generator().manual_seed(1))
                                                               * torch.arange(n)).long()
    parents[0] = -1
    sees = torch.zeros((n, n), dtype=torch.bool)
    for i, up in enumerate(parents.tolist()):
        if up >= 0:
            sees[i] = sees[up]
        sees[i, i] = True
    length = n + 40
    pages = -(-length // 16)
    t = {"qo_indptr": [0, n], "paged_kv_indptr": [0, pages], "paged_kv_indices": list(range(pages))[::-1],
         "paged_kv_last_page_len": [length - (pages - 1) * 16]}
    t = {k: torch.tensor(v, dtype=torch.int32) for k, v in t.items()}
    gen = torch.Generator(device=gpu_device).manual_seed(2)
    q = torch.randn((n, 2, 64), device=gpu_device, generator=gen).to(F16)
    cache = torch.randn((pages, 2, 16, 1, 64), device=gpu_device, generator=gen).to(F16)
    be = backend(2, 1, 64, 16, gpu_device)
    be.plan_tree(**t, tree_mask=sees)
    want = be.run_tree(q, cache)
    be.plan_tree(**t, tree_parents=parents.int())
    assert torch.equal(be.run_tree(q, cache), want)
    if kind == "chain":
        be.plan_prefill(**t)
        causal = be.run_prefill(q, cache).float()
        # two roundings to fp16, and weights off by less than 2^-13 for values of up to 5
        assert ((want.float() - causal).abs() <= 2.0**-10 * causal.abs() + 1e-3).all()


def test_a_c_plan_of_no_nodes(gpu_device):
    """max_tree 0 with tokens, through the C entries: nothing is worked on, by parents and by mask."""
    lib = _lib.load()
    case = tree_case([4, 3], [40, 30], 4, 2, 64, 16, F16, gpu_device, seed=1)
    t = tables(case, gpu_device)
    dev = {k: v.data_ptr() for k, v in t.items()}
    parents, mask = case["parents"].to(gpu_device), torch.ones((7, 4), dtype=torch.uint8, device=gpu_device)
    n, out = t["paged_kv_indices"].numel(), torch.full_like(case["q"], 7.0)
    size = lib.pl_tree_plan_size(2, 7, 0, n, 4, 2, 64)
    plan = torch.zeros(size + 64, dtype=torch.uint8, device=gpu_device)
    plan[size:] = 5
    stream = _lib.stream_handle(gpu_device)
    for by in ((parents.data_ptr(), None, 0), (None, mask.data_ptr(), 4)):
        assert lib.pl_tree_plan(dev["qo_indptr"], dev["paged_kv_indptr"], dev["paged_kv_indices"], n,
                                dev["paged_kv_last_page_len"], 2, 7, 0, *by, 4, 2, 64, 16, 0, n, plan.data_ptr(), size,
                                stream) == 0
        ws = torch.empty(lib.pl_tree_workspace_size(2, 7, 0, 4, 2, 64), dtype=torch.uint8, device=gpu_device)
        c = case["cache"]
        assert lib.pl_tree_run(case["q"].data_ptr(), 256, 64, c.data_ptr(), c[:, 1].data_ptr(), c.stride(0), c.stride(2),
                               c.stride(3), c.shape[0], out.data_ptr(), 256, 64, None, 2, 7, 0, 4, 2, 64, 16, 0.125,
                               _lib.PL_DTYPE_F16, plan.data_ptr(), size, n, ws.data_ptr(), ws.numel(), stream) == 0
        torch.cuda.synchronize()
        assert (out == 7).all() and (plan[size:] == 5).all()
