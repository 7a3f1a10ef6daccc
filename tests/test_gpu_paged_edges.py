"""Calls of the 8-bit paged cache at the edges of what its documentation allows:
batches that need the large shared-memory grant, tables without the pages that
nobody sees, values at the top of their type, offsets that answer nothing, ids
and sizes past 32 bits."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import paged_plain as P
from test_gpu_paged import DEV, _Case, _data, _i32, _pool

from kvdlra_b200 import PagedKVCache
from kvdlra_b200.paged import PagedPool, build_page_tables, paged_append, paged_attention, paged_peek

pytestmark = pytest.mark.gpu
REPO = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("new", [300, 5000])  # one launch, two launches
def test_tables_between_the_default_and_the_large_shared_memory(new) -> None:
    """6100 requests' prefix sums are just under 48 KB, the kernel's static memory
    goes on top.  A process of its own: a larger call before would have raised the limit."""
    code = f"""
import sys; sys.path[:0] = [{str(REPO)!r}, {str(REPO / 'tests')!r}]
import torch, paged_plain as P
from kvdlra_b200.paged import build_page_tables
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
cached, new = [i % 3 for i in range(6100)], [int(i < {new}) for i in range(6100)]
table, free = [[i if c else -1, -1] for i, c in enumerate(cached)], list(range(7000, 13200))
ok, *want = P.tables(cached, new, table, free, 16, {new} + 5)
t = i32(table)
p = build_page_tables(i32(cached), i32(new), t, i32(free), i32([len(free)]), page_size=16, capacity={new} + 5)
assert ok and want == [t.tolist(), p.lens.tolist(), p.cu_new.tolist(), p.slots.tolist(), p.positions.tolist(), p.free_count.item()]
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("n", [1, 40])  # the few-row kernel, the tensor-memory kernel
@pytest.mark.parametrize("page", [16, 64])
def test_pages_that_nobody_sees_need_no_id(n, page) -> None:
    """A server gives the pages behind the window back; padding needs none."""
    case = _Case("e4m3", 64, 2, page, [300, 301], seed=31)
    q = torch.randn(2, 8, n, 64, device=DEV).to(torch.bfloat16)
    want = paged_attention(case.pool, case.table, case.lens, q, window=20)
    t = case.table.clone()
    t[:, : (300 - n + 1 - 20) // page] = -1
    assert torch.equal(paged_attention(case.pool, t, case.lens, q, window=20), want)
    case.pool.check_status()
    starts = _i32([0, 200])
    want = paged_attention(case.pool, case.table, case.lens, q, starts=starts)
    t = case.table.clone()
    t[1, : 200 // page] = 1 << 30
    assert torch.equal(paged_attention(case.pool, t, case.lens, q, starts=starts), want)
    case.pool.check_status()


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 128])
def test_the_largest_values_come_back_finite(store, dtype, dim) -> None:
    """A code may round up past the type's largest value; the value read back is held to that."""
    top = torch.finfo(dtype).max
    pool = _pool(store, 2, 1, 16, dim)
    x = torch.zeros(16, 1, dim, dtype=dtype, device=DEV)
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2] = top, -top, top * 0.97
    paged_append(pool, _i32(list(range(16))), x, x)
    k, v = paged_peek(pool, _i32([[0]]), _i32([16]), 16, dtype=dtype)
    want = _exact_peek(pool, store).clip(-top, top)
    for y in (k, v):
        assert np.array_equal(y[0, 0].double().cpu().numpy(), torch.tensor(want).to(dtype).double().numpy())
    assert k[0, 0, 0, 0].item() == top and k[0, 0, 1, 1].item() == -top
    pool.check_status()


def _exact_peek(pool, store):
    return pool.k[0, 0].float().double().cpu().numpy() * pool.k_scale[0, 0].double().item()


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_over_the_largest_f16_values_is_finite(store, dim, n) -> None:
    """65504 is stored as 65536 (code 256 or 64): an average of such values is above
    65520 less 2^-11 of it at the most, so every output rounds to 65504 or would to infinity."""
    pool = _pool(store, 4, 1, 16, dim)
    k = torch.randn(40, 1, dim, device=DEV).half()
    v = torch.full((40, 1, dim), 65504.0, device=DEV).half()
    v[:, :, 1::2] *= -1
    paged_append(pool, _i32(list(range(40))), k, v)
    q = torch.randn(1, 4, n, dim, device=DEV).half()
    out = paged_attention(pool, _i32([[0, 1, 2]]), _i32([40]), q)
    assert bool((out[..., ::2] == 65504).all()) and bool((out[..., 1::2] == -65504).all())


@pytest.mark.parametrize("dim, dtype", [(64, torch.bfloat16), (128, torch.float32)])
@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("tokens", [70, 5000])
def test_values_up_to_2_to_the_90(dim, dtype, n, tokens) -> None:
    rng = np.random.default_rng(4)
    pool = _pool("e4m3", tokens // 64 + 1, 1, 64, dim)
    k, v = (torch.tensor(rng.standard_normal((tokens, 1, dim)), dtype=torch.float32, device=DEV) for _ in "kv")
    v = (v * 2.0**90 / v.abs().max()).contiguous()
    paged_append(pool, torch.arange(tokens, dtype=torch.int32, device=DEV), k, v)
    table, lens = torch.arange(tokens // 64 + 1, dtype=torch.int32, device=DEV)[None], _i32([tokens])
    dk, dv = (x[0].double().cpu().numpy() for x in paged_peek(pool, table, lens, tokens, dtype=torch.float32))
    q = torch.tensor(rng.standard_normal((1, 2, n, dim)), dtype=dtype, device=DEV)
    out = paged_attention(pool, table, lens, q)
    vs = np.repeat(pool.v_scale[:, 0].double().cpu().numpy(), 64)[None, :tokens]
    ref, le, *parts = P.attention(q[0].transpose(0, 1).double().cpu().numpy(), dk, dv, dim**-0.5, vs=vs)
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= P.bounds(ref, le, *parts, dim, tokens, dtype)[0]).all()


def _stale(shape, dtype):
    """Memory of a freed tensor full of sevens, which the allocator hands out next."""
    for _ in range(4):
        x = torch.full(shape, 7.0, dtype=dtype, device=DEV)
        del x


@pytest.mark.parametrize("dtype, scale", [(torch.float32, 1), (torch.bfloat16, 1), (torch.bfloat16, 12)])
@pytest.mark.parametrize("cu, live", [([2, 5, 5], [2, 3, 4]), ([0, 9, 5], []), ([-3, 2, 5], [2, 3, 4]), ([5, 2, 900], []), ([0, 3, 900], [0, 1, 2]),
                                      ([1, 3, 6], [1, 2, 3, 4, 5]), ([7, 7, 7], [])])
def test_rows_that_no_request_answers_are_zero(dtype, scale, cu, live) -> None:
    """Rows before the first offset, behind the last, and of offsets that make no
    sense: zeros in an output that the call makes, left alone in the caller's."""
    case = _Case("int8", 64, 1, 16, [90, 80], seed=6)
    rows = 7 * scale
    cu = [c * scale for c in cu]
    live = sorted(r for x in live for r in range(x * scale, (x + 1) * scale))
    q = torch.randn(rows, 2, 64, device=DEV).to(dtype)
    mine = torch.full_like(q, 5.0)
    paged_attention(case.pool, case.table, case.lens, q, cu_q=_i32(cu), out=mine)
    _stale(q.shape, dtype)
    _stale(q.shape[:2], torch.float32)
    out, lse = paged_attention(case.pool, case.table, case.lens, q, cu_q=_i32(cu), return_lse=True)
    dead = [r for r in range(rows) if r not in live]
    assert not out[dead].any() and bool((lse[dead] == -torch.inf).all())
    assert bool((mine[dead] == 5.0).all())
    assert torch.equal(mine[live], out[live]) and bool(out[live].any(-1).all()) and bool(lse[live].isfinite().all())


def test_queries_over_a_table_without_columns_are_zero_in_the_callers_output() -> None:
    pool = PagedPool.allocate(4, 16, 2, 64, device=DEV)
    q = torch.randn(6, 4, 64, device=DEV)
    mine = torch.full_like(q, 5.0)
    table = torch.empty((2, 0), dtype=torch.int32, device=DEV)
    out, lse = paged_attention(pool, table, _i32([0, 3]), q, cu_q=_i32([1, 2, 4]), out=mine, return_lse=True)
    assert not out[1:4].any() and bool((out[[0, 4, 5]] == 5.0).all()) and bool((lse == -torch.inf).all())


@pytest.mark.parametrize("rows", [2, 9000])  # one launch, two launches
@pytest.mark.parametrize("bad", [-1, -(1 << 20), 1 << 28])
def test_ids_that_name_no_page_are_reported_by_the_tables(rows, bad) -> None:
    """The page that a new token continues has no id, or one whose slots pass 32
    bits: the token goes nowhere, and the status says so."""
    pages = -(-rows // 16) + 1
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    table = torch.full((2, pages + 1), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[1, 0] = 3, bad
    p = build_page_tables(_i32([5, 3]), _i32([1, rows]), table, torch.arange(9, 9 + pages, dtype=torch.int32, device=DEV), _i32([pages]),
                          page_size=16, capacity=rows + 1, status=status)
    slots = p.slots.tolist()
    assert slots[0] == 3 * 16 + 5
    n = min(rows, 13)
    assert slots[1 : 1 + n] == [-1] * n
    assert all(s >= 9 * 16 for s in slots[1 + n :])
    assert status[1].item() != 0
    assert p.positions.tolist()[:3] == [5, 3, 4]


def test_sizes_past_32_bits_are_not_cut() -> None:
    case = _Case("int8", 64, 1, 16, [60, 50], seed=8)
    q = torch.randn(2, 2, 1, 64, device=DEV)
    want = paged_attention(case.pool, case.table, case.lens, q)
    assert torch.equal(paged_attention(case.pool, case.table, case.lens, q, window=2**32 + 5), want)
    assert torch.equal(paged_attention(case.pool, case.table, case.lens, q[:, :, 0], cu_q=_i32([0, 1, 2]), max_q=2**32 + 1), want[:, 0])


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 30])
def test_queries_near_the_top_of_their_type(dim, dtype, n) -> None:
    """Queries of 2^120 over keys of 2^-100: scores of ordinary size."""
    pool = _pool("e4m3", 6, 1, 16, dim)
    g = torch.Generator(device=DEV).manual_seed(5)
    k = torch.randn(70, 1, dim, device=DEV, generator=g) * 2.0**-97
    v = torch.randn(70, 1, dim, device=DEV, generator=g)
    paged_append(pool, _i32(list(range(70))), k, v)
    table, lens = _i32([[0, 1, 2, 3, 4]]), _i32([70])
    dk, dv = (x[0].double().cpu().numpy() for x in paged_peek(pool, table, lens, 70, dtype=torch.float32))
    q = (torch.randn(1, 2, n, dim, device=DEV, generator=g) * 2.0**120).to(dtype)
    assert bool(q.isfinite().all())
    scaling = 2.0**-23 * dim**-0.5
    out, lse = paged_attention(pool, table, lens, q, scaling=scaling, return_lse=True)
    vs = np.repeat(pool.v_scale[:5, 0].double().cpu().numpy(), 16)[None, :70]
    ref, le, *parts = P.attention(q[0].transpose(0, 1).double().cpu().numpy(), dk, dv, scaling, vs=vs)
    tol, tol_e = P.bounds(ref, le, *parts, dim, 70, dtype)
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= tol).all()
    assert (np.abs(lse[0].double().cpu().numpy() - le) <= tol_e).all()


def test_small_weights_of_pages_without_values_count() -> None:
    """One token ahead of 65535 others by 26.15 powers of two, whose values are all
    zero (scale 2^-100): their weights are 8.8e-4 of the sum.  152 requests over the
    same pages, so that a request is one CTA's.  The sum of 65536 terms, 16 at a time
    into one of fp32, is off by 4112 half steps of 2^-24 at most, 2.5e-4."""
    n, page = 65536, 128
    pool = PagedPool.allocate(n // page, page, 1, 64, storage="int8", device=DEV)
    k, v = torch.zeros(2, n, 1, 64, device=DEV).to(torch.bfloat16)
    k[0, 0, 0], v[0] = 1.0, 30000.0
    paged_append(pool, torch.arange(n, dtype=torch.int32, device=DEV), k, v)
    assert pool.v_scale[1, 0].item() == 2.0**-100
    q = torch.zeros(152, 40, 1, 64, device=DEV).to(torch.bfloat16)
    q[..., 0] = 145.0
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).repeat(152, 1)
    _, lse = paged_attention(pool, table, torch.full((152,), n, dtype=torch.int32, device=DEV), q, return_lse=True)
    ks = pool.k_scale[0, 0].item()
    s0 = 145.0 * 0.125 * float(pool.k[0, 0, 0, 0].item()) * ks
    want = s0 + np.log1p((n - 1) * np.exp(-s0))
    assert float((lse.double() - want).abs().max()) <= 2.6e-4


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("page, dim", [(16, 32), (128, 128)])
@pytest.mark.parametrize("slots, kept", [
    ([5, 5], [5, -1]), ([3, 5], [3, -1]), ([6, 4], [6, -1]), ([0, 0, 1, 2], [0, -1, -1, -1]), ([4, 5, 7, 8, 20], [4, 5, -1, -1, -1]),
    ([3, 4, 3, 5], [3, 4, -1, -1]), ([7, 8, 8, 9], [7, 8, -1, -1]),
])
def test_rows_of_a_page_out_of_order_are_skipped_and_reported(store, page, dim, slots, kept) -> None:
    """A second run into the page that the row before went to (the same slot twice,
    a gap, a step back) would race with the first; the rows that follow another
    page's are stored, whatever the order of the pages."""
    rng = np.random.default_rng(7)
    slots, kept = [page + s for s in slots], [s if s < 0 else page + s for s in kept]
    if page == 16 and slots[-1] == 16 + 20:
        kept[-1] = slots[-1]  # the next page: continues there
    slots, kept = slots + [2, 3], kept + [2, 3]
    pool = _pool(store, 6, 3, page, dim)
    x = _data(rng, (len(slots), 3, dim), torch.bfloat16)
    before = pool.k.float().double().cpu().numpy(), pool.k_scale.double().cpu().numpy()
    paged_append(pool, _i32(slots), x, x)
    want = P.append(*before, kept, x.double().cpu().numpy(), store)
    for name in "kv":
        assert np.array_equal(getattr(pool, name).float().double().cpu().numpy(), want[0], equal_nan=True)
        assert np.array_equal(getattr(pool, name + "_scale").double().cpu().numpy(), want[1])
    with pytest.raises(RuntimeError, match="bad indices"):
        pool.check_status()


@pytest.mark.parametrize("page, dim, heads", [(16, 64, 8), (128, 128, 3), (32, 256, 1)])
@pytest.mark.parametrize("batch, new", [(300, 1), (70, 5), (3, 200)])
def test_append_of_many_requests_whatever_the_launch(page, dim, heads, batch, new) -> None:
    """Many runs a CTA or one, with and without the length of the longest run, and
    with a wrong one: the same codes and scales."""
    rng = np.random.default_rng(batch + page)
    lens = [page * int(rng.integers(0, 3)) + int(rng.integers(0, page)) for _ in range(batch)]
    held = [-(-(n + new) // page) for n in lens]
    ids = rng.permutation(sum(held)).tolist()
    slots, at = [], 0
    for n, h in zip(lens, held):
        mine, at = ids[at : at + h], at + h
        slots += [mine[t // page] * page + t % page for t in range(n, n + new)]
    x = [_data(rng, (batch * new, heads, dim), torch.bfloat16) for _ in "kv"]
    pools = []
    for kw in ({}, {"max_new": new}, {"max_new": 1}, {"max_new": 2**40}, None):
        pool = _pool("e4m3", sum(held), heads, page, dim)
        if kw is None:
            paged_append(pool, _i32(slots), *(t.view(batch, new, heads, dim).transpose(1, 2) for t in x))
        else:
            paged_append(pool, _i32(slots), *x, **kw)
        pool.check_status()
        pools.append(pool)
    n = min(batch * new, 400)  # the plain form of the first rows, whole runs
    n -= n % new
    before = _pool("e4m3", sum(held), heads, page, dim)
    want = P.append(before.k.float().double().cpu().numpy(), before.k_scale.double().cpu().numpy(), slots[:n], x[0][:n].double().cpu().numpy(), "e4m3")
    rows = sorted({s // page for s in slots[:n]})
    assert np.array_equal(pools[0].k[rows].float().double().cpu().numpy(), want[0][rows], equal_nan=True)
    assert np.array_equal(pools[0].k_scale[rows].double().cpu().numpy(), want[1][rows])
    for p in pools[1:]:
        assert torch.equal(p.k.view(torch.uint8), pools[0].k.view(torch.uint8)) and torch.equal(p.v.view(torch.uint8), pools[0].v.view(torch.uint8))
        assert torch.equal(p.k_scale, pools[0].k_scale) and torch.equal(p.v_scale, pools[0].v_scale)


def test_a_cache_after_a_capture_that_never_ran() -> None:
    """Nothing that a captured step made is used by an eager one."""
    cache = PagedKVCache(None, 64, page_size=16, num_layers=1)
    k = torch.randn(2, 2, 5, 64, device=DEV).to(torch.bfloat16)
    cache.update(k, k, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.update(k[:, :, :1], k[:, :, :1], 0)
    del graph
    cache.reset()
    cache.update(k, k, 0)
    got = cache.update(k[:, :, :1], k[:, :, :1], 0)[0]
    assert cache.tables.lens.tolist() == [6, 6]
    assert torch.equal(got[:, :, 5], got[:, :, 0])
    cache.check_status()
