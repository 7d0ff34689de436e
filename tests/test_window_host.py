"""What the windowed attention and the 4-bit cache refuse before any launch (host checks; pointers are never read), the
prefill plan, and the oracle's format against a search over all its values."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import window as ow
from pagelora_amd import _lib
from pagelora_amd.kv4 import kv4_append, kv4_page_shape, kv4_read
from pagelora_amd.kv_pool import PagedKVPool, kv_copy_pages
from pagelora_amd.window_attention import WindowAttention

PTR = 4096  # aligned, never dereferenced
BF16 = torch.bfloat16


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def attention(**kw):
    return WindowAttention(**{**dict(device="cpu", num_qo_heads=4, num_kv_heads=2, head_dim=64, page_size=16), **kw})


@pytest.mark.parametrize("kw,error", [
    (dict(num_qo_heads=5), ValueError), (dict(num_kv_heads=0), ValueError), (dict(num_qo_heads=0), ValueError),
    (dict(head_dim=96), NotImplementedError), (dict(head_dim=256), NotImplementedError), (dict(page_size=0), ValueError),
    (dict(window=-1), ValueError), (dict(sinks=-1), ValueError), (dict(window=2**31), ValueError),
])
def test_constructor_refuses(kw, error):
    with pytest.raises(error):
        attention(**kw)


def good():
    return dict(paged_kv_indptr=i32(0, 1, 3), paged_kv_indices=i32(4, 2, 7), paged_kv_last_page_len=i32(5, 1))


@pytest.mark.parametrize("name,value,what", [
    ("paged_kv_indptr", i32(0, 1), "batch \\+ 1"), ("paged_kv_indptr", i32(1, 2, 3), "start at 0"),
    ("paged_kv_indptr", i32(0, 2, 1), "non-decreasing"), ("paged_kv_indptr", i32(0, 1, 4), "exceeds"),
    ("paged_kv_indptr", i32(0, 1, 3).long(), "int32"), ("paged_kv_indices", i32(4, -2, 7), "negative"),
    ("paged_kv_indices", i32(4, 2, 7)[None], "1-D"), ("paged_kv_last_page_len", i32(5, 17), "outside"),
    ("paged_kv_last_page_len", i32(0, 1), "outside"),
])
def test_plans_refuse(name, value, what):
    with pytest.raises(ValueError, match=what):
        attention().plan_decode(**{**good(), name: value})
    with pytest.raises(ValueError, match=what):
        attention().plan_prefill(**{**good(), "qo_indptr": i32(0, 1, 2), name: value})


def test_plans_need_a_device():
    with pytest.raises(RuntimeError, match="ROCm device"):
        attention().plan_decode(**good())
    with pytest.raises(RuntimeError, match="ROCm device"):
        attention().plan_prefill(**good(), qo_indptr=i32(0, 1, 2))
    with pytest.raises(RuntimeError, match="plan_decode"):
        attention().run_decode(torch.zeros(2, 4, 64, dtype=BF16), torch.zeros(8, 2, 16, 2, 64, dtype=BF16))
    with pytest.raises(ValueError, match="batch \\+ 1"):
        attention().plan_prefill(**good(), qo_indptr=i32(0, 1))


# ------------------------------------------------------------ prefill plan
def plan(qo, kv_pages, last, hq=4, hkv=2, head_dim=128, page=16, window=0, sinks=0, max_records=None):
    """(status, work items, merges, workspace bytes)"""
    lib = _lib.load()
    qo_t, last_t = i32(*np.cumsum([0, *qo])), i32(*last)
    kv_t = i32(*np.cumsum([0, *kv_pages]))
    n, m, b = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_size_t(0)
    out = (ctypes.byref(n), ctypes.byref(m), ctypes.byref(b))
    args = (qo_t.data_ptr(), kv_t.data_ptr(), last_t.data_ptr(), len(qo), hq, hkv, head_dim, page, window, sinks)
    status = lib.pl_window_prefill_plan(*args, None, 0, *out)
    if status:
        return status, None, None, None
    records = torch.zeros((n.value + m.value, 16), dtype=torch.int32)
    status = lib.pl_window_prefill_plan(*args, records.data_ptr() if records.numel() else PTR,
                                        records.shape[0] if max_records is None else max_records, *out)
    return status, records[: n.value].tolist(), records[n.value:].tolist(), b.value


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5), (64, 0), (1, 200), (1000, 64), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (14, 2), (33, 1)])
def test_prefill_plan_covers_what_is_seen(window, sinks, hq, hkv):
    """Every row's seen tokens lie in its item's tiles, counted once, no tile outside what its rows see; parts are whole."""
    lens, new, page = [1, 300, 64, 5000, 700], [1, 290, 0, 3, 130], 16
    pages = [-(-n // page) for n in lens]
    status, items, merges, nbytes = plan(new, pages, [n - (p - 1) * page for n, p in zip(lens, pages)], hq, hkv, window=window,
                                         sinks=sinks)
    assert status == 0
    g = hq // hkv
    blocks = {}
    starts = np.cumsum([0, *new]), np.cumsum([0, *pages])
    for r, row0, rows, qo_begin, kv_len, page_begin, begin, end, slot, part, parts, *_ in items:
        assert (rows, kv_len) == (new[r] * g, lens[r]) and (qo_begin, page_begin) == (starts[0][r], starts[1][r])
        assert begin < end and (slot >= 0) == (parts > 1)
        blocks.setdefault((r, row0), []).append((begin, end, slot, part, parts))
    assert sorted(blocks) == [(r, r0) for r in range(5) for r0 in range(0, new[r] * g, 128)]
    slots = set()
    for (r, row0), cut in blocks.items():
        cut.sort()
        assert cut[0][0] == 0 and all(a[1] == b[0] for a, b in zip(cut, cut[1:]))
        assert [c[3] for c in cut] == list(range(len(cut))) and all(c[4] == len(cut) for c in cut)
        first = lens[r] - new[r] + row0 // g
        final = lens[r] - new[r] + min(row0 + 127, new[r] * g - 1) // g
        lo = max(0, first - window + 1) if window else 0
        head = min((min(sinks, lo) + 63) // 64, lo // 64)
        tiles = [i if i < head else i - head + lo // 64 for i in range(cut[-1][1])]
        assert tiles[-1] == final // 64 and len(set(tiles)) == len(tiles)
        for p in (first, final):
            assert {t // 64 for t in ow.sees(p, lens[r], window, sinks)} <= set(tiles)
        if cut[0][2] >= 0:
            slots.update(range(cut[0][2], cut[0][2] + len(cut)))
            assert [r, row0, cut[0][2], len(cut)] in [[m[0], m[1], m[8], m[10]] for m in merges]
    assert len(merges) == sum(len(c) > 1 for c in blocks.values())
    assert slots == set(range(len(slots))) and nbytes == len(slots) * hkv * 128 * 130 * 4


def test_prefill_plan_refuses():
    for kw in (dict(qo=[5], kv_pages=[0], last=[0]), dict(qo=[20], kv_pages=[1], last=[16]), dict(qo=[1], kv_pages=[1], last=[17]),
               dict(qo=[1], kv_pages=[1], last=[0]), dict(qo=[-1], kv_pages=[1], last=[1]), dict(qo=[1], kv_pages=[-1], last=[1]),
               dict(qo=[1], kv_pages=[1], last=[1], window=-1), dict(qo=[1], kv_pages=[1], last=[1], sinks=-1),
               dict(qo=[1], kv_pages=[1], last=[1], hq=3), dict(qo=[1], kv_pages=[1], last=[1], page=0),
               dict(qo=[1], kv_pages=[2**27], last=[16])):
        assert plan(**kw)[0] == _lib.PL_ERR_INVALID, kw
    assert plan([1], [1], [1], head_dim=256)[0] == _lib.PL_ERR_UNSUPPORTED
    assert plan([1], [1], [1], max_records=0)[0] == _lib.PL_ERR_WORKSPACE
    assert plan([0, 0], [0, 3], [0, 1]) == (0, [], [], 0)


# ------------------------------------------------------------- C entries
def decode_run(**kw):
    a = dict(q=PTR, q_sb=512, q_sh=128, k=PTR, v=PTR, page=4096, token=256, head=128, pages=8, bits=16, o=PTR, o_sb=512, o_sh=128,
             lse=None, batch=2, hq=4, hkv=2, d=128, ps=16, window=0, sinks=0, scale=0.1, dtype=2, plan=PTR, plan_bytes=1 << 20,
             indices=4, ws=PTR, ws_bytes=1 << 30, stream=None)
    return _lib.load().pl_window_decode_run(*{**a, **kw}.values())


def prefill_run(**kw):
    a = dict(q=PTR, q_sb=512, q_sh=128, k=PTR, v=PTR, page=4096, token=256, head=128, pages=8, bits=16, ind=PTR,
             items=PTR, n=1, m=1, o=PTR, o_sb=512, o_sh=128, hq=4, hkv=2, d=128, ps=16, window=0, sinks=0,
             scale=0.1, dtype=2, ws=PTR, ws_bytes=64, need=64, stream=None)
    return _lib.load().pl_window_prefill_run(*{**a, **kw}.values())


COMMON = [
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(o=None), 1), (dict(q=PTR + 2), 1), (dict(v=PTR + 8), 1),
    (dict(q_sb=514), 1), (dict(o_sh=4), 1), (dict(token=132), 1), (dict(head=4), 1), (dict(page=12), 1), (dict(pages=0), 1),
    (dict(hq=5), 1), (dict(hkv=0), 1), (dict(ps=0), 1), (dict(window=-1), 1), (dict(sinks=-2), 1),
    (dict(bits=4, ps=12), 1), (dict(bits=4, ps=1 << 21), 1), (dict(bits=4, head=8), 1), (dict(bits=8), 2), (dict(d=256), 2),
    (dict(dtype=0), 2),
]


@pytest.mark.parametrize("kw,status", COMMON + [(dict(batch=-1), 1), (dict(plan=None), 1), (dict(plan=PTR + 16), 1), (dict(plan_bytes=64), 3),
                                                (dict(ws_bytes=64), 3), (dict(ws=None), 1), (dict(indices=-1), 1)])
def test_decode_run_refuses(kw, status):
    assert decode_run(**kw) == status and _lib.last_error()


def test_launches_of_too_many_workgroups_are_refused():
    assert decode_run(batch=1 << 21) == 1 and decode_run(batch=2**31 - 1, hq=1, hkv=1) == 1
    assert prefill_run(n=1 << 22) == 1 and prefill_run(m=1 << 22) == 1


@pytest.mark.parametrize("kw,status", COMMON + [(dict(items=None), 1), (dict(n=-1), 1), (dict(ws=None), 3), (dict(ws_bytes=60), 3),
                                                (dict(ind=None), 1), (dict(items=PTR + 16), 1), (dict(m=-1), 1),
                                                (dict(n=1 << 30, hkv=4), 1)])
def test_prefill_run_refuses(kw, status):
    assert prefill_run(**kw) == status and _lib.last_error()


def test_nothing_to_do_launches_nothing():
    assert decode_run(batch=0) == 0 and prefill_run(n=0, m=0) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 1), (dict(indices=None), 1), (dict(indptr=None), 1), (dict(last=None), 1), (dict(plan=None), 1),
    (dict(plan=PTR + 32), 1), (dict(nbytes=64), 3), (dict(count=-1), 1), (dict(ps=0), 1), (dict(window=-1), 1), (dict(hq=3), 1),
])
def test_decode_plan_refuses(kw, status):
    a = dict(indptr=PTR, indices=PTR, count=4, last=PTR, batch=2, hq=4, hkv=2, ps=16, window=0, sinks=0, plan=PTR, nbytes=1 << 20,
             stream=None)
    assert _lib.load().pl_window_decode_plan(*{**a, **kw}.values()) == status


def test_decode_sizes():
    lib = _lib.load()
    good = dict(batch=64, indices=1000, hq=32, hkv=8, ps=16, window=0, sinks=0)
    for kw in (dict(batch=-1), dict(indices=-1), dict(hq=5), dict(ps=0), dict(window=-1), dict(sinks=-1)):
        a = {**good, **kw}
        assert lib.pl_window_decode_plan_size(*a.values()) == 0
        assert lib.pl_window_decode_workspace_size(*list(a.values())[:4], 128, *list(a.values())[4:]) == 0
    assert lib.pl_window_decode_plan_size(*good.values()) >= 64 + 4000 + 64 * 40
    assert lib.pl_window_decode_workspace_size(64, 1000, 32, 8, 128, 16, 0, 0) >= 64 * 8 * 16 * 130 * 4


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=-1), 1), (dict(hkv=0), 1), (dict(d=32), 2), (dict(d=256), 2), (dict(dtype=0), 2), (dict(ps=4), 1), (dict(ps=12), 1),
    (dict(pages=0), 1), (dict(k=None), 1), (dict(kc=None), 1), (dict(ids=None), 1), (dict(k=PTR + 8), 1), (dict(vc=PTR + 4), 1),
    (dict(kt=260), 1), (dict(head=8), 1), (dict(page=100), 1), (dict(tokens=2**31 - 1, hkv=2**16), 1),
    (dict(tokens=1 << 26), 1),
])
def test_kv4_entries_refuse(kw, status):
    a = dict(k=PTR, v=PTR, kt=256, kh=128, vt=256, vh=128, kc=PTR, vc=PTR, page=4096, head=1088, pages=4, ps=16, ids=PTR, offs=PTR,
             tokens=2, hkv=2, d=128, dtype=2, stream=None)
    a.update(kw)
    lib = _lib.load()
    assert lib.pl_kv4_append(*a.values()) == status
    names = ("kc", "vc", "page", "head", "pages", "ps", "ids", "offs", "tokens", "hkv", "d", "k", "v", "kt", "kh", "vt", "vh", "dtype",
             "stream")
    assert lib.pl_kv4_read(*(a[n] for n in names)) == status


# ---------------------------------------------------------- 4-bit wrappers
def test_kv4_wrappers_refuse():
    size = dict(num_kv_heads=2, head_dim=64, page_size=16)
    assert kv4_page_shape(**size) == (2, 2, 16 * 34)
    for kw, error in ((dict(head_dim=96), NotImplementedError), (dict(page_size=12), ValueError), (dict(page_size=0), ValueError)):
        with pytest.raises(error):
            kv4_page_shape(**{**size, **kw})
    layer, x, at = torch.zeros((3, 2, 2, 544), dtype=torch.uint8), torch.zeros((2, 2, 64), dtype=BF16), torch.zeros(2, dtype=torch.int64)
    for bad in (layer[:, :1], layer[..., :500], layer.view(torch.int8), layer[None]):
        with pytest.raises(ValueError, match="4-bit KV cache"):
            kv4_append(bad, x, x, at, at, **size)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kv4_append(layer, x, x, at, at, **size)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kv4_read(layer, at, at, **size)


def test_4_bit_pools():
    kw = dict(num_layers=2, capacity_pages=4, page_size=16, num_kv_heads=2, head_dim=64, dtype=BF16, device="cpu")
    pool = PagedKVPool(**kw, kv_bits=4)
    assert pool.cache.shape == (2, 4, 2, 2, 544) and pool.cache.dtype == torch.uint8
    pool.cache.random_(0, 256)
    old = pool.cache.clone()
    pool._grow(9)
    assert torch.equal(pool.cache[:, :4], old) and pool.cache.shape[1] == 16
    assert PagedKVPool(**kw).cache.shape == (2, 4, 2, 16, 2, 64)
    with pytest.raises(ValueError, match="kv_bits"):
        PagedKVPool(**kw, kv_bits=8)
    with pytest.raises(ValueError, match="multiple of 8"):
        PagedKVPool(**{**kw, "page_size": 4}, kv_bits=4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kv_copy_pages(pool.cache, [1], [2])
    with pytest.raises(ValueError, match="cache must be"):
        kv_copy_pages(pool.cache[0, 0], [1], [2])


# ------------------------------------------------------------------ oracle
def test_oracle_quantizes_to_the_nearest_level():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 64)) * np.exp(rng.uniform(-20, 20, (40, 1)))
    codes, scales = ow.quantize(x)
    got = ow.values(codes, scales)
    for i in range(40):
        for g in range(2):
            v = x[i, 32 * g: 32 * g + 32]
            e = -125
            while 6 * 2.0**e < np.abs(v).max():
                e += 1
            assert scales[i, g] == e + 127
            grid = np.concatenate([ow.LEVELS, -ow.LEVELS]) * 2.0**e
            assert (np.abs(got[i, 32 * g: 32 * g + 32] - v) == np.abs(grid[None] - v[:, None]).min(1)).all()


def test_oracle_packs_pages():
    """A nibble of its own for every (page, K or V, head, token, dim)."""
    rng = np.random.default_rng(2)
    kc, vc = (rng.integers(0, 16, (2, 8, 3, 64)).astype(np.uint8) for _ in range(2))
    ks, vs = (rng.integers(0, 256, (2, 8, 3, 2)).astype(np.uint8) for _ in range(2))
    layer = ow.pack_pages(kc, ks, vc, vs)
    assert layer.shape == (2, 2, 3, 8 * 34)
    for p, t, h, d in ((0, 0, 0, 0), (1, 7, 2, 63), (0, 5, 1, 34), (1, 2, 0, 9)):
        nibble = lambda byte: byte >> 4 if d % 2 else byte & 15  # noqa: E731
        assert nibble(layer[p, 0, h, t * 32 + d // 2]) == kc[p, t, h, d]
        assert layer[p, 0, h, 256 + t * 2 + d // 32] == ks[p, t, h, d // 32]
        assert nibble(layer[p, 1, h, t // 4 * 128 + d // 8 * 16 + t % 4 * 4 + d % 8 // 2]) == vc[p, t, h, d]
        assert layer[p, 1, h, 256 + t // 4 * 8 + d // 32 * 4 + t % 4] == vs[p, t, h, d // 32]


def test_oracle_window():
    assert ow.sees(10, 20, 0, 0).tolist() == list(range(11))
    assert ow.sees(10, 20, 3, 2).tolist() == [0, 1, 8, 9, 10]
    assert ow.sees(1, 20, 3, 5).tolist() == [0, 1]
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((2, 2, 4)), rng.standard_normal((9, 1, 4)), rng.standard_normal((9, 1, 4))
    o, lse, _, _ = ow.attend(q, k, v, 2, 1, 0.5)
    for i, at in enumerate(([0, 6, 7], [0, 7, 8])):
        w = np.exp(k[at, 0] @ q[i, 1] * 0.5)
        assert np.allclose(o[i, 1], w @ v[at, 0] / w.sum()) and np.isclose(lse[i, 1], np.log(w.sum()))
