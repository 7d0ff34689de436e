"""Attention of drafted trees (plan_tree / run_tree) against the float64 oracle.

Tolerance of an output element, from the kernel's arithmetic: half a step of
the storage type for the store; for the weights the rounding of p to two planes
(2^-17 and less), twice the error of a score (fp32 sums
of D products, and an exponent below 2^5) and of the sums over the tokens, all
times the largest |v| that the row attends.
"""

import math

import numpy as np
import pytest
import torch

from oracle import paged_decode as opd
from oracle import tree as otree
from pagelora_amd.attention_backend import PagedDecodeAttention
from tests.gpu_cases import ragged_case

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def random_parents(n, rng, kind="tree"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":
        return [-1] * n
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)]


def tree_case(trees, kv_lens, hq, hkv, head_dim, page_size, dtype, device, seed, kind="tree", q_scale=1.0):
    rng = np.random.default_rng(seed)
    case = ragged_case(lens=kv_lens, hq=hq, hkv=hkv, head_dim=head_dim, page_size=page_size, dtype=dtype,
                       device=device, seed=seed, pool_extra=3)
    gen = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((sum(trees), hq, head_dim), generator=gen) * q_scale).to(dtype)
    parents = [random_parents(n, rng, kind) if n else [] for n in trees]
    case.update(q=q.to(device), q_host=q, trees=trees,
                qo_indptr=torch.tensor([0] + list(np.cumsum(trees)), dtype=torch.int32),
                parents=torch.tensor(sum(parents, []), dtype=torch.int32),
                sees=[otree.ancestors(p) for p in parents])
    return case


def tables(case, device=None):
    t = {"qo_indptr": case["qo_indptr"], "paged_kv_indptr": case["indptr"], "paged_kv_indices": case["indices"],
         "paged_kv_last_page_len": case["last"]}
    return {k: v.to(device) for k, v in t.items()} if device is not None else t


def backend(hq, hkv, head_dim, page_size, device):
    return PagedDecodeAttention(device=device, workspace_mb=1, num_qo_heads=hq, num_kv_heads=hkv, head_dim=head_dim,
                                page_size=page_size)


def oracle(case, sm_scale=None):
    return otree.paged_tree(case["q_host"].double().numpy(), case["cache_host"].double().numpy(),
                            case["qo_indptr"].numpy(), case["indptr"].numpy(), case["indices"].numpy(),
                            case["last"].numpy(), case["sees"], sm_scale)


def check(case, out, lse=None, dtype=BF16):
    ref, ref_lse = oracle(case)
    cache, q = case["cache_host"].double().numpy(), case["q_host"].double().numpy()
    d = q.shape[2]
    got = out.double().cpu().numpy()
    half, p_err = 2.0**-8 if dtype == BF16 else 2.0**-11, 2.0**-17
    for r, n in enumerate(case["trees"]):
        if n == 0:
            continue
        a = int(case["qo_indptr"][r])
        k, v = opd.gather_row_kv(cache, case["indptr"].numpy(), case["indices"].numpy(), case["last"].numpy(), r)
        k, v = np.nan_to_num(k, posinf=0, neginf=0), np.nan_to_num(v, posinf=0, neginf=0)
        g = q.shape[1] // k.shape[1]
        qk = max(float((np.abs(k[:, h // g]) @ np.abs(q[a:a + n, h]).T).max()) for h in range(q.shape[1]))
        score = d * 2.0**-24 * qk / math.sqrt(d) + 2.0**-19
        weights = p_err + 2 * score + 2 * len(k) * 2.0**-24
        tol = half * np.abs(ref[a:a + n]) + weights * np.abs(v).max() + 1e-30
        err = np.abs(got[a:a + n] - ref[a:a + n])
        assert np.isfinite(got[a:a + n]).all(), f"request {r}: not finite"
        assert (err <= tol).all(), f"request {r}: error {err.max()} at tolerance {tol[err > tol][0]}"
        if lse is not None:
            x, y = lse.double().cpu().numpy()[a:a + n], ref_lse[a:a + n]
            live = np.isfinite(y)
            assert (live == np.isfinite(x)).all() and (x[~live] == y[~live]).all()
            assert (np.abs(x - y)[live] <= 2 * score + 2 * len(k) * 2.0**-24 + np.abs(y[live]) * 2.0**-22).all()


def run(case, hq, hkv, head_dim, page_size, device, **kw):
    be = backend(hq, hkv, head_dim, page_size, device)
    be.plan_tree(**tables(case), tree_parents=case["parents"], **kw)
    out = torch.full_like(case["q"], float("nan"))
    lse = torch.full(case["q"].shape[:2], float("nan"), device=device)
    be.run_tree_into(case["q"], case["cache"], out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (14, 2), (32, 8)])
def test_ragged_trees(gpu_device, dtype, head_dim, heads):
    hq, hkv = heads
    trees, lens = [1, 0, 7, 16, 33], [1, 20, 130, 16, 700]
    case = tree_case(trees, lens, hq, hkv, head_dim, 16, dtype, gpu_device, seed=hq + head_dim)
    out, lse = run(case, hq, hkv, head_dim, 16, gpu_device)
    check(case, out, lse, dtype)


@pytest.mark.parametrize("page_size", [1, 5, 8, 16, 32, 48])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_page_sizes(gpu_device, page_size, dtype):
    case = tree_case([5, 12, 3], [5, 301, 96], 8, 2, 128, page_size, dtype, gpu_device, seed=page_size)
    out, lse = run(case, 8, 2, 128, page_size, gpu_device)
    check(case, out, lse, dtype)


@pytest.mark.parametrize("min_share", [0, 2, 3, 1000])
@pytest.mark.parametrize("kv_len", [31, 127, 128, 129, 1000, 5000])
def test_split_ranges(gpu_device, min_share, kv_len):
    """The kv range cut into shares of several sizes, at the edges of blocks and tiles."""
    case = tree_case([9, 2], [kv_len, 50], 8, 2, 128, 16, BF16, gpu_device, seed=kv_len)
    out, lse = run(case, 8, 2, 128, 16, gpu_device, min_share=min_share)
    check(case, out, lse)


@pytest.mark.parametrize("kind", ["chain", "star", "forest", "tree"])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 200])
def test_tree_shapes(gpu_device, kind, n):
    """Masks of one word and of several, one row block and several."""
    case = tree_case([n, 3], [n + 77, 40], 4, 1, 128, 16, F16, gpu_device, seed=n, kind=kind)
    out, lse = run(case, 4, 1, 128, 16, gpu_device)
    check(case, out, lse, F16)


@pytest.mark.parametrize("prefix", [0, 1, 15, 31, 32, 33, 100])
def test_general_mask_with_empty_rows(gpu_device, prefix):
    """tree_mask: any pattern, rows that see no node, and without a prefix nothing at all."""
    n = 70
    case = tree_case([n, 5], [prefix + n, 5], 4, 2, 128, 16, BF16, gpu_device, seed=prefix)
    rng = np.random.default_rng(prefix)
    mask = np.zeros((n + 5, 72), dtype=bool)
    mask[:n, :n] = rng.random((n, n)) < 0.2
    mask[3] = mask[n + 2] = False
    mask[n:, :5] = rng.random((5, 5)) < 0.5
    mask[n + 2] = False
    mask[n:, 5:] = True  # past the tree: not read as nodes
    case["sees"] = [mask[:n, :n], mask[n:, :5]]
    be = backend(4, 2, 128, 16, gpu_device)
    for m in (torch.from_numpy(mask), torch.from_numpy(mask.astype(np.uint8) * 3)):
        be.plan_tree(**tables(case), tree_mask=m)
        out, lse = torch.full_like(case["q"], float("nan")), torch.zeros(case["q"].shape[:2], device=gpu_device)
        be.run_tree_into(case["q"], case["cache"], out, lse)
        torch.cuda.synchronize()
        check(case, out, lse)
        assert (out[n + 2] == 0).all() and (lse[n + 2] == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_values_may_be_anything(gpu_device, dtype, bad):
    """K and V of nodes hold infinities or NaN: rows that do not see them are exact, rows that do are not finite."""
    n, prefix = 40, 71
    case = tree_case([n], [prefix + n], 8, 2, 128, 16, dtype, gpu_device, seed=3, kind="tree")
    ip, ind = case["indptr"].tolist(), case["indices"].tolist()
    poisoned = [5, 17, 39]
    for j in poisoned:
        pos = prefix + j
        case["cache_host"][ind[ip[0] + pos // 16], :, pos % 16, :, ::3] = bad
    case["cache"] = case["cache_host"].to(gpu_device)
    out, _ = run(case, 8, 2, 128, 16, gpu_device)
    touched = case["sees"][0][:, poisoned].any(axis=1)
    got = out.double().cpu().numpy()
    assert touched.any() and not touched.all()
    ref, _ = oracle(case)
    assert np.isfinite(got[~touched]).all()
    tol = 2.0**-7 * np.abs(ref[~touched]) + 0.01
    assert (np.abs(got[~touched] - ref[~touched]) <= tol).all()
    assert not np.isfinite(got[touched]).all(axis=(1, 2)).any()


def test_infinite_v_alone(gpu_device):
    """An infinity in V only: the dims of the rows that see it are not finite, every other value is exact."""
    n, prefix = 20, 44
    case = tree_case([n], [prefix + n], 4, 1, 128, 16, BF16, gpu_device, seed=8)
    ip, ind = case["indptr"].tolist(), case["indices"].tolist()
    pos = prefix + 4
    case["cache_host"][ind[ip[0] + pos // 16], 1, pos % 16, 0, 50] = float("inf")
    case["cache"] = case["cache_host"].to(gpu_device)
    out, _ = run(case, 4, 1, 128, 16, gpu_device)
    got, ref = out.double().cpu().numpy(), oracle(case)[0]
    assert (np.isfinite(got) == np.isfinite(ref)).all() and not np.isfinite(ref).all()
    live = np.isfinite(ref)
    assert (np.abs(got - ref)[live] <= 2.0**-7 * np.abs(ref[live]) + 0.01).all()


@pytest.mark.parametrize("scale", [0.0, 30.0, -1.0])
def test_scores_of_any_size(gpu_device, scale):
    """Scores far apart (one weight is all), all equal, and a negative softmax scale."""
    case = tree_case([11], [400], 8, 2, 128, 16, F16, gpu_device, seed=5, q_scale=abs(scale))
    be = backend(8, 2, 128, 16, gpu_device)
    if scale < 0:
        be.sm_scale = -be.sm_scale
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    out = be.run_tree(case["q"], case["cache"])
    ref, _ = oracle(case, be.sm_scale)
    # scores of up to 30 * 128 * 16 / 11 in fp32: 2^-8 of error and less in an exponent
    np.testing.assert_allclose(out.double().cpu().numpy(), ref, rtol=2.0**-10, atol=2.0**-5 if scale > 1 else 2.0**-8)


def test_fp16_far_tokens_keep_their_weight(gpu_device):
    """20000 tokens 2^-26 as heavy each as one: three ten-thousandths of the row, which fp16 would round to nothing."""
    L = 20001
    case = tree_case([1], [L], 1, 1, 64, 16, F16, gpu_device, seed=1)
    ip, ind = case["indptr"].tolist(), case["indices"].tolist()
    cache = torch.zeros_like(case["cache_host"])
    cache[:, 1] = 4096.0
    cache[ind[0], 0, 0, 0, 0] = 8.0
    cache[ind[0], 1, 0] = 0.0
    q = torch.zeros((1, 1, 64), dtype=F16)
    q[0, 0, 0] = 18.0  # 18 * 8 / 8 = 18 above the others' 0: e^-18 = 2^-26
    be = backend(1, 1, 64, 16, gpu_device)
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    out = be.run_tree(q.to(gpu_device), cache.to(gpu_device)).double().cpu()
    w = (L - 1) * math.exp(-18.0)
    want = 4096.0 * w / (1 + w)
    # p of 2^-26 times 2^14 has 10 bits of fp16
    assert abs(float(out[0, 0, 0]) - want) <= want * (2.0**-10 + 2.0**-11)


def test_strided_tensors(gpu_device):
    """q and out as slices of wider rows, K/V as a pair of HND-ordered caches, rows behind the last request untouched."""
    hq, hkv, d, ps = 8, 2, 128, 16
    case = tree_case([6, 9], [100, 33], hq, hkv, d, ps, BF16, gpu_device, seed=4)
    n = 15
    wide = torch.randn((n, 2 * hq, d + 8), device=gpu_device).to(BF16)
    q = wide[:, ::2, :d]
    q.copy_(case["q"])
    room = torch.full((n, 3 * hq, d + 4), 7.0, dtype=BF16, device=gpu_device)
    out = room[:, hq:2 * hq, :d]
    pool = case["cache"].transpose(2, 3).contiguous()  # [P, 2, Hkv, page, D]
    k, v = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    be = backend(hq, hkv, d, ps, gpu_device)
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    be.run_tree_into(q, (k, v), out)
    torch.cuda.synchronize()
    check(case, out)
    assert (room[:, :hq] == 7).all() and (room[:, 2 * hq:] == 7).all() and (room[:, hq:2 * hq, d:] == 7).all()
    # in place
    be.run_tree_into(q, (k, v), q)
    torch.cuda.synchronize()
    check(case, q)


def test_device_tables_and_rows_behind(gpu_device):
    """Device tables whose qo_indptr ends before the last row: rows behind stay as they were."""
    case = tree_case([6, 9], [100, 33], 8, 2, 128, 16, BF16, gpu_device, seed=4)
    q = torch.cat((case["q"], torch.ones((5, 8, 128), dtype=BF16, device=gpu_device)))
    parents = torch.cat((case["parents"], torch.zeros(5, dtype=torch.int32))).to(gpu_device)
    be = backend(8, 2, 128, 16, gpu_device)
    be.plan_tree(**tables(case, gpu_device), tree_parents=parents, max_tree=9)
    out = torch.full_like(q, 3.0)
    be.run_tree_into(q, case["cache"], out)
    torch.cuda.synchronize()
    check(case, out[:15])
    assert (out[15:] == 3).all()


def test_malformed_device_tables_stay_in_bounds(gpu_device):
    """Clamped, not read astray: the results mean nothing, the neighbours stay untouched."""
    case = tree_case([6, 9, 4], [100, 33, 20], 8, 2, 128, 16, BF16, gpu_device, seed=4)
    good = tables(case)
    be = backend(8, 2, 128, 16, gpu_device)
    bad = {
        "qo_indptr": [0, 19, 3, 19], "paged_kv_indptr": [-5, 7, 2, 10**9], "paged_kv_last_page_len": [0, 900, -3],
        "paged_kv_indices": [10**6, -1] + [5] * (case["indices"].numel() - 2), "tree_parents": [18] * 10 + [-7] * 9,
    }
    for name, values in bad.items():
        t = {**good, "tree_parents": case["parents"]}
        t[name] = torch.tensor(values, dtype=torch.int32)
        room = torch.full((21, 8, 128), 3.0, dtype=BF16, device=gpu_device)
        be.plan_tree(**{k: v.to(gpu_device) for k, v in t.items()}, max_tree=9)
        be.run_tree_into(case["q"], torch.nan_to_num(case["cache"]), room[1:20])
        torch.cuda.synchronize()
        assert (room[0] == 3).all() and (room[20] == 3).all(), name


def test_matches_causal_prefill_on_a_chain(gpu_device):
    """A chain is a causal segment: the same result as run_prefill within two roundings."""
    case = tree_case([37], [300], 8, 2, 128, 16, BF16, gpu_device, seed=6, kind="chain")
    be = backend(8, 2, 128, 16, gpu_device)
    be.plan_prefill(**tables(case))
    a = be.run_prefill(case["q"], case["cache"]).float()
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    b = be.run_tree(case["q"], case["cache"]).float()
    assert ((a - b).abs() <= 2.0**-7 * a.abs() + 1e-4).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("n", [2, 9, 17, 60, 130, 300])
def test_row_blocks_of_every_size(gpu_device, head_dim, n, dtype):
    """16 to 256 rows of a row block, several per request, shares that begin and end inside them."""
    case = tree_case([n, 3, n // 2], [n + 1500, 3, 900], 2, 1, head_dim, 16, dtype, gpu_device, seed=n)
    out, lse = run(case, 2, 1, head_dim, 16, gpu_device)
    check(case, out, lse, dtype)
    out, lse = run(case, 2, 1, head_dim, 16, gpu_device, min_share=5)
    check(case, out, lse, dtype)


@pytest.mark.parametrize("n", [20, 50, 120, 250])
def test_row_blocks_of_every_size_masked_values(gpu_device, n):
    """Infinities and NaN in nodes, for each number of waves per block."""
    for bad in (float("nan"), float("inf")):
        case = tree_case([n], [n + 45], 1, 1, 128, 16, BF16, gpu_device, seed=n)
        ip, ind = case["indptr"].tolist(), case["indices"].tolist()
        for j in (3, n // 2, n - 1):
            case["cache_host"][ind[ip[0] + (45 + j) // 16], :, (45 + j) % 16] = bad
        case["cache"] = case["cache_host"].to(gpu_device)
        out, _ = run(case, 1, 1, 128, 16, gpu_device)
        touched = case["sees"][0][:, [3, n // 2, n - 1]].any(axis=1)
        got, ref = out.double().cpu().numpy(), oracle(case)[0]
        assert np.isfinite(got[~touched]).all() and not np.isfinite(got[touched]).any()
        assert (np.abs(got - ref)[~touched] <= 2.0**-7 * np.abs(ref[~touched]) + 0.01).all()


@pytest.mark.parametrize("kv_len,tree", [(40000, 3), (70000, 2), (70000, 40)])
def test_one_long_sequence_in_very_many_parts(gpu_device, kv_len, tree):
    """One kv head: its rows come together from more than 64 and more than 256 parts."""
    case = tree_case([tree], [kv_len], 1, 1, 64, 16, BF16, gpu_device, seed=tree)
    out, lse = run(case, 1, 1, 64, 16, gpu_device)
    check(case, out, lse)


@pytest.mark.parametrize("long,small", [(30000, 250), (3000, 250), (9000, 40), (2000, 300)])
def test_long_wide_trees_among_many_small_ones(gpu_device, long, small):
    """Shares that hold several requests, chunks of row blocks that slots share."""
    trees, lens = [40] + [1] * small + [33], [long] + [3 + i % 120 for i in range(small)] + [long // 2]
    case = tree_case(trees, lens, 4, 1, 64, 16, F16, gpu_device, seed=small)
    out, lse = run(case, 4, 1, 64, 16, gpu_device)
    check(case, out, lse, F16)


def test_many_requests(gpu_device):
    """More requests than slots, empty ones among them."""
    rng = np.random.default_rng(2)
    trees = [int(x) for x in rng.integers(0, 6, 300)]
    lens = [t + int(x) for t, x in zip(trees, rng.integers(0, 90, 300))]
    case = tree_case(trees, lens, 4, 2, 64, 16, BF16, gpu_device, seed=12)
    out, lse = run(case, 4, 2, 64, 16, gpu_device)
    check(case, out, lse)


def test_long_cache_offsets(gpu_device):
    """A pool whose byte offsets pass 2^32: the pages of a request at its end."""
    hkv, d, ps = 8, 128, 16
    pages = 2**32 // (2 * ps * hkv * d * 2) + 40
    cache = torch.zeros((pages, 2, ps, hkv, d), dtype=BF16, device=gpu_device)
    case = tree_case([5], [150], 8, 8, d, ps, BF16, gpu_device, seed=9)
    n = case["cache_host"].shape[0]
    cache[pages - n:] = case["cache"]
    be = backend(8, hkv, d, ps, gpu_device)
    t = tables(case)
    t["paged_kv_indices"] = t["paged_kv_indices"] + (pages - n)
    be.plan_tree(**t, tree_parents=case["parents"])
    out = be.run_tree(case["q"], cache)
    torch.cuda.synchronize()
    check(case, out)


def test_other_stream(gpu_device):
    """Planned on one stream and run on another."""
    case = tree_case([9, 30], [1000, 2000], 8, 2, 128, 16, BF16, gpu_device, seed=7)
    be = backend(8, 2, 128, 16, gpu_device)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    with torch.cuda.stream(side):
        out = be.run_tree(case["q"], case["cache"])
    torch.cuda.synchronize()
    check(case, out)


def test_captured_plan_and_run_follow_the_tables(gpu_device):
    """One graph of plan + run over device tables replays as a tree and its sequence change."""
    hq, hkv, d, ps, n = 8, 2, 128, 16, 12
    cases = [tree_case([n, n], [L, L + 5], hq, hkv, d, ps, BF16, gpu_device, seed=L) for L in (40, 300, 41)]
    room = max(c["indices"].numel() for c in cases)
    be = backend(hq, hkv, d, ps, gpu_device)
    pool = max(c["cache"].shape[0] for c in cases)
    static = {"qo": torch.zeros(3, dtype=torch.int32), "kv": torch.zeros(3, dtype=torch.int32),
              "ind": torch.zeros(room, dtype=torch.int32), "last": torch.ones(2, dtype=torch.int32),
              "parents": torch.zeros(2 * n, dtype=torch.int32)}
    static = {k: v.to(gpu_device) for k, v in static.items()}
    q = torch.zeros_like(cases[0]["q"])
    cache = torch.zeros((pool, 2, ps, hkv, d), dtype=BF16, device=gpu_device)
    out = torch.zeros_like(q)

    def load(c):
        static["qo"].copy_(c["qo_indptr"])
        static["kv"].copy_(c["indptr"])
        static["ind"][: c["indices"].numel()].copy_(c["indices"])
        static["last"].copy_(c["last"])
        static["parents"].copy_(c["parents"])
        q.copy_(c["q"])
        cache[: c["cache"].shape[0]].copy_(c["cache"])

    def step():
        be.plan_tree(qo_indptr=static["qo"], paged_kv_indptr=static["kv"], paged_kv_indices=static["ind"],
                     paged_kv_last_page_len=static["last"], tree_parents=static["parents"], max_tree=n)
        be.run_tree_into(q, cache, out)

    load(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c in (cases[1], cases[2], cases[0], cases[1]):
        load(c)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out)


def test_two_captured_runs_of_other_sizes(gpu_device):
    """Graphs of two batch sizes keep their plans apart; each replays on the plan made last for its size."""
    a = tree_case([4], [70], 8, 2, 128, 16, BF16, gpu_device, seed=1)
    b = tree_case([60] * 20, [100] * 20, 8, 2, 128, 16, BF16, gpu_device, seed=2)
    be = backend(8, 2, 128, 16, gpu_device)
    graphs = []
    for c in (a, b):
        be.plan_tree(**tables(c), tree_parents=c["parents"])
        out = be.run_tree(c["q"], c["cache"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            be.run_tree_into(c["q"], c["cache"], out)
        graphs.append((c, g, out))
    for _ in range(3):
        for c, g, out in graphs:
            be.plan_tree(**tables(c), tree_parents=c["parents"])
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            check(c, out)


def test_captured_run_keeps_its_plan(gpu_device):
    """Plans of other sizes that need as many bytes, made after the capture, leave the graph's plan alone."""
    a, b = (tree_case([n], [70], 8, 2, 128, 16, BF16, gpu_device, seed=n) for n in (4, 5))
    be = backend(8, 2, 128, 16, gpu_device)
    be.plan_tree(**tables(a), tree_parents=a["parents"])
    signature = be.tree_graph_signature()
    out = be.run_tree(a["q"], a["cache"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.run_tree_into(a["q"], a["cache"], out)
    for _ in range(3):
        be.plan_tree(**tables(b), tree_parents=b["parents"])
        check(b, be.run_tree(b["q"], b["cache"]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(a, out)
    be.plan_tree(**tables(a), tree_parents=a["parents"])
    assert be.tree_graph_signature() == signature


def test_batches_without_nodes(gpu_device):
    """No request, or requests without nodes: nothing runs, nothing is written."""
    be = backend(8, 2, 128, 16, gpu_device)
    cache = torch.zeros((3, 2, 16, 2, 128), dtype=BF16, device=gpu_device)
    none = torch.zeros(0, dtype=torch.int32)
    for qo, kv, ind, last in (([0], [0], none, none), ([0, 0, 0], [0, 1, 1], torch.tensor([2], dtype=torch.int32),
                                                     torch.tensor([7, 0], dtype=torch.int32))):
        for dev in ("cpu", gpu_device):
            t = {"qo_indptr": torch.tensor(qo, dtype=torch.int32), "paged_kv_indptr": torch.tensor(kv, dtype=torch.int32),
                 "paged_kv_indices": ind, "paged_kv_last_page_len": last, "tree_parents": none}
            be.plan_tree(**{k: v.to(dev) for k, v in t.items()})
            q = torch.zeros((0, 8, 128), dtype=BF16, device=gpu_device)
            assert be.run_tree(q, cache).shape == q.shape
    torch.cuda.synchronize()


def test_masks_in_any_order(gpu_device):
    """A mask whose rows are not rows of memory, on the host and on the device."""
    for n in (1, 9):
        case = tree_case([n], [n + 40], 4, 2, 64, 16, F16, gpu_device, seed=n)
        mask = torch.from_numpy(case["sees"][0].copy())
        be = backend(4, 2, 64, 16, gpu_device)
        for dev in ("cpu", gpu_device):
            room = torch.ones((mask.shape[1] + 3, n), dtype=torch.bool, device=dev)
            view = room.t()
            view[:, :n] = mask.to(dev)
            be.plan_tree(**tables(case, dev), tree_mask=view)
            out = be.run_tree(case["q"], case["cache"])
            torch.cuda.synchronize()
            check(case, out, None, F16)


def test_same_bits_twice(gpu_device):
    case = tree_case([33, 8], [3000, 777], 8, 2, 128, 16, BF16, gpu_device, seed=13)
    a, la = run(case, 8, 2, 128, 16, gpu_device)
    b, lb = run(case, 8, 2, 128, 16, gpu_device)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_refusals(gpu_device):
    case = tree_case([4], [40], 8, 2, 128, 16, BF16, gpu_device, seed=1)
    be = backend(8, 2, 128, 16, gpu_device)
    with pytest.raises(RuntimeError, match="plan_tree must be called"):
        be.run_tree(case["q"], case["cache"])
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    with pytest.raises(ValueError, match="tokens but the plan"):
        be.run_tree(case["q"][:3], case["cache"])
    with pytest.raises(ValueError, match="dtype"):
        be.run_tree(case["q"].half(), case["cache"])
    with pytest.raises(ValueError, match="outside the"):
        be.run_tree(case["q"], case["cache"][:1])
    with pytest.raises(ValueError, match="lse"):
        be.run_tree_into(case["q"], case["cache"], torch.empty_like(case["q"]),
                         torch.empty((8, 4), device=gpu_device))
    with pytest.raises(RuntimeError, match="device"):
        be.run_tree(case["q"].cpu(), case["cache"])
    with pytest.raises(NotImplementedError):
        be.run_tree(case["q"].float(), case["cache"].float())
    with pytest.raises(ValueError, match="multiples of 8"):
        q = torch.zeros((4, 8, 132), dtype=BF16, device=gpu_device)[:, :, :128]
        be.run_tree(q, case["cache"])
    with pytest.raises(ValueError, match="all on the host or all on the device"):
        be.plan_tree(**tables(case), tree_parents=case["parents"].to(gpu_device))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            be.plan_tree(**tables(case), tree_parents=case["parents"])
