"""Plans of trees: of fewer nodes than a tree has, and beside runs on other streams."""

import pytest
import torch

from tests.test_gpu_tree_attention import BF16, F16, backend, check, oracle, tables, tree_case

pytestmark = pytest.mark.gpu


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
