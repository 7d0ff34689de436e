"""How long windowed attention keeps the plans that captured graphs read."""

import gc

import pytest
import torch

from tests.window_cases import BF16, F16, attention, case, check, set_cache, tables

pytestmark = pytest.mark.gpu

ROOM = 1 << 20  # page ids of a table: a plan of 4 MiB


def roomy(c, device):
    """The case's tables on the device, with room for more pages."""
    t = tables(c, device)
    t["paged_kv_indices"] = torch.cat([t["paged_kv_indices"], torch.zeros(ROOM, dtype=torch.int32, device=device)])
    return t


def decode_case(device, seed):
    return case([300, 40], 8, 2, 128, 16, BF16, device, window=64, sinks=3, seed=seed)


def captured(*steps):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for step in steps:
            out = step()
    return graph, out


def held():
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return torch.cuda.memory_allocated()


def test_a_graph_with_its_plan_leaves_nothing_behind(gpu_device):
    c = decode_case(gpu_device, 1)
    attn, t = attention(c), roomy(c, gpu_device)
    before = None
    for _ in range(5):
        graph, out = captured(lambda: attn.plan_decode(**t), lambda: attn.run_decode(c["q"], c["cache"]))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out)
        del graph, out
        before = before or held()  # (the last plan stays)
    assert held() - before < 4 * ROOM, "plans of graphs that are gone are kept"


def test_graphs_hold_their_plans(gpu_device):
    """Two graphs of one object, each with its plan; allocations and eager steps between the replays."""
    cases = [decode_case(gpu_device, s) for s in (2, 3)]
    attn = attention(cases[0])
    graphs = []
    for c in cases:
        t = roomy(c, gpu_device)
        graphs.append((c, t, *captured(lambda: attn.plan_decode(**t), lambda: attn.run_decode(c["q"], c["cache"]))))
    attn.plan_decode(**tables(cases[0]))  # (the last captured plan is the object's no more)
    for _ in range(3):
        for c, _, graph, out in graphs:
            held()
            junk = torch.full((32 << 20,), -1, dtype=torch.int32, device=gpu_device)
            graph.replay()
            check(cases[0], attn.run_decode(cases[0]["q"], cases[0]["cache"]))
            torch.cuda.synchronize()
            check(c, out)
            del junk


def test_a_side_stream_of_the_capture(gpu_device):
    """The plan on one stream, a run on another that joins again, then a second plan and run."""
    a, b = (decode_case(gpu_device, s) for s in (4, 5))
    attn, ta, tb = attention(a), roomy(a, gpu_device), roomy(b, gpu_device)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.plan_decode(**ta)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            first = attn.run_decode(a["q"], a["cache"])
        attn.plan_decode(**tb)
        second = attn.run_decode(b["q"], b["cache"])
        here.wait_stream(side)
    assert not attn._captured  # (the side stream is of the same capture)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(a, first)
        check(b, second)


def test_a_plan_in_one_graph_and_its_runs_in_another(gpu_device):
    """The plan is kept for the second graph."""
    c = decode_case(gpu_device, 6)
    attn, t = attention(c), roomy(c, gpu_device)
    plan, _ = captured(lambda: attn.plan_decode(**t))
    run, out = captured(lambda: attn.run_decode(c["q"], c["cache"]))
    assert len(attn._captured) == 1
    plan.replay()
    other = decode_case(gpu_device, 7)
    attn.plan_decode(**tables(other))
    del plan
    held()
    junk = torch.full((32 << 20,), -1, dtype=torch.int32, device=gpu_device)
    for _ in range(2):
        out.zero_()
        run.replay()
        torch.cuda.synchronize()
        check(c, out)
    del junk


@pytest.mark.parametrize("how", ["decode", "prefill"])
def test_captured_runs_of_eager_plans_are_released(gpu_device, how):
    c = decode_case(gpu_device, 8)
    if how == "prefill":
        c = case([300, 40], 8, 2, 128, 16, BF16, gpu_device, new=[20, 3], window=64, sinks=3, seed=8)
    attn, t = attention(c), roomy(c, gpu_device)
    extra = {"qo_indptr": c["qo_indptr"]} if how == "prefill" else {}
    before = None
    for _ in range(4):
        getattr(attn, "plan_" + how)(**t, **extra)
        graph, out = captured(lambda: getattr(attn, "run_" + how)(c["q"], c["cache"]))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out)
        del graph, out
        attn.release_captured()
        before = before or held()
    assert held() - before < 4 * ROOM
    check(c, getattr(attn, "run_" + how)(c["q"], c["cache"]))  # (the plan at hand stays)


@pytest.mark.parametrize("fits", [True, False])
def test_captured_prompts_of_fp16_over_4_bits(gpu_device, fits):
    """Both ways of an item, by what fp16 holds, replayed with eager prompts in between."""
    c = case([300, 1500], 4, 2, 128, 16, F16, gpu_device, bits=4, new=[130, 40], window=200, sinks=5, seed=9)
    if not fits:
        cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1))
        cache[:, 1, :, 1, 32:64] *= 2.0**-30
        set_cache(c, cache)
    attn = attention(c)
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c))
    want = attn.run_prefill(c["q"], c["cache"])
    torch.cuda.synchronize()
    check(c, want)
    graph, out = captured(lambda: attn.run_prefill(c["q"], c["cache"]))
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(attn.run_prefill(c["q"], c["cache"]), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
