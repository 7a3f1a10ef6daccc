"""The 8-bit paged cache's operators on the GPU against their plain 64-bit
forms (``paged_plain``), at the sizes and masks where they can go wrong.

Tables, codes and scales are exact (power-of-two scales make every code one
rounding of the value); attention is held to ``paged_plain.bounds``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_plain as P

from kvdlra_b200.paged import PagedPool, PageTables, build_page_tables, paged_append, paged_attention, paged_peek

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _i32(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ tables


def _state(rng, batch, page, cached, width, spare):
    held = [-(-c // page) for c in cached]
    ids = rng.permutation(sum(held) + spare).tolist()
    table = [[-1] * width for _ in range(batch)]
    for b, n in enumerate(held):
        table[b][:n] = ids[:n]
        ids = ids[n:]
    return table, ids


@pytest.mark.parametrize("batch, page, cached_hi, new_hi, pad", [
    (1, 16, 0, 1, 0), (1, 128, 300, 700, 3), (7, 16, 40, 1, 2), (33, 32, 100, 5, 0), (300, 16, 50, 90, 11), (1025, 64, 200, 3, 1),
    (2500, 16, 20, 40, 5), (12288, 16, 3, 1, 0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(batch, page, cached_hi, new_hi, pad, in_place) -> None:
    rng = np.random.default_rng(batch + page)
    cached = rng.integers(0, cached_hi + 1, batch).tolist()
    new = rng.integers(0, new_hi + 1, batch).tolist()
    width = max(-(-(c + t) // page) for c, t in zip(cached, new)) + 2
    need = sum(-(-(c + t) // page) + (-c // page) for c, t in zip(cached, new))
    table, free = _state(rng, batch, page, cached, width, need + 1)
    cap = sum(new) + pad
    ok, *want = P.tables(cached, new, table, free, page, cap)
    assert ok
    # the table as a strided view, the stack with room behind its top
    store = torch.full((batch, width + 3), -7, dtype=torch.int32, device=DEV)
    t = store[:, :width]
    t.copy_(_i32(table))
    lens, count, stack = _i32(cached), _i32([len(free)]), _i32(free + [99999])
    p = build_page_tables(lens, _i32(new), t, stack, count, page_size=page, capacity=cap, in_place=in_place)
    got = [t.tolist(), p.lens.tolist(), p.cu_new.tolist(), p.slots.tolist(), p.positions.tolist(), p.free_count.item()]
    assert got == want
    assert bool((store[:, width:] == -7).all())
    assert (lens.tolist(), count.item()) == ((want[1], want[5]) if in_place else (cached, len(free)))


@pytest.mark.parametrize("case", ["pages", "columns", "rows", "negative", "negative new", "count"])
def test_tables_that_do_not_fit_change_nothing(case) -> None:
    t = PageTables(3, 4, 6, 16, DEV)
    assert t.advance(_i32([20, 5, 0]), 25).slots.tolist() == [*range(0, 20), *range(32, 37)]
    new, cap = [1, 1, 1], 3
    if case == "pages":
        new, cap = [40, 20, 1], 61
    elif case == "columns":
        new, cap = [45, 0, 0], 45
    elif case == "rows":
        cap = 2
    elif case == "negative":
        t.lens[1] = -3
    elif case == "negative new":
        new = [1, -1, 1]
    else:
        t.free_count[0] = 7
    before = (t.table.clone(), t.lens.clone(), t.free_count.clone(), t.free_pages.clone())
    p = t.advance(_i32(new), cap)
    assert p.slots.tolist() == [-1] * cap and p.cu_new.tolist() == [0] * 4 and p.positions.tolist() == [0] * cap
    assert all(torch.equal(a, b) for a, b in zip(before, (t.table, t.lens, t.free_count, t.free_pages)))
    with pytest.raises(RuntimeError, match="could not be built"):
        t.check_status()
    t.check_status()  # cleared


def test_release_gives_pages_back_in_order() -> None:
    t = PageTables(5, 4, 12, 16, DEV)
    t.advance(_i32([17, 0, 32, 1, 16]), 66)
    assert t.table[:, :2].tolist() == [[0, 1], [-1, -1], [2, 3], [4, -1], [5, -1]]
    t.release(torch.tensor([True, True, False, True, False], device=DEV))
    assert t.lens.tolist() == [0, 0, 32, 0, 16]
    n = t.free_count.item()
    assert n == 6 + 3 and t.free_pages[:n].tolist() == [11, 10, 9, 8, 7, 6, 0, 1, 4]
    p = t.advance(_i32([1, 40, 1, 0, 0]), 42)
    assert t.table[0, 0] == 4 and t.table[1, :3].tolist() == [1, 0, 6] and t.table[2, 2] == 7
    assert p.free_count.item() == 4
    t.check_status()
    t.free_count[0] = 10  # more than can be: refused whole
    t.release(torch.tensor([False, True, False, False, False], device=DEV))
    assert t.lens.tolist() == [1, 40, 33, 0, 16] and t.free_count.item() == 10
    with pytest.raises(RuntimeError):
        t.check_status()


# ---------------------------------------------------------- append and peek


def _pool(store, pages, heads, page, dim, order="phsd"):
    """A pool in page-head-slot or page-slot-head order, its slack full of NaN codes."""
    shape = (pages, heads, page, dim) if order == "phsd" else (pages, page, heads, dim)
    kv = [torch.full(shape, 0x7F if store == "e4m3" else 0x55, dtype=torch.uint8, device=DEV).view(P.CODE[store]) for _ in "kv"]
    if order != "phsd":
        kv = [x.transpose(1, 2) for x in kv]
    s = [torch.full((pages, heads), 3.0, device=DEV) for _ in "kv"]
    return PagedPool(*kv, *s)


def _values(pool, name):
    return getattr(pool, name).float().double().cpu().numpy()


def _data(rng, shape, dtype):
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)))
    return torch.tensor(x, dtype=dtype, device=DEV)


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, page, heads, order", [(32, 16, 3, "phsd"), (64, 16, 8, "pshd"), (64, 64, 5, "phsd"), (128, 32, 2, "phsd"),
                                                     (128, 128, 1, "pshd"), (256, 16, 3, "phsd"), (256, 128, 2, "phsd")])
def test_append_in_steps_and_peek(store, dtype, dim, page, heads, order) -> None:
    """Prompts, chunks and single tokens of three requests, growing scales."""
    rng = np.random.default_rng(dim + page)
    t = PageTables(3, 6, 20, page, DEV)
    pool = _pool(store, 20, heads, page, dim, order)
    codes, scales = {}, {}
    steps = [[page + 3, 0, 1], [1, 2, 1], [5, 1, page - 2], [1, 1, 1], [2 * page, 0, 3]]
    for i, new in enumerate(steps):
        plan = t.advance(_i32(new), sum(new) + 1)
        x = {n: _data(rng, (sum(new) + 1, heads, dim), dtype) * (2.0**i) for n in "kv"}
        before = {n: (_values(pool, n), getattr(pool, n + "_scale").double().cpu().numpy()) for n in "kv"}
        paged_append(pool, plan.slots, x["k"], x["v"])
        for n in "kv":
            codes[n], scales[n] = P.append(*before[n], plan.slots.tolist(), x[n].double().cpu().numpy(), store)
            assert np.array_equal(_values(pool, n), codes[n], equal_nan=True), (i, n)
            assert np.array_equal(getattr(pool, n + "_scale").double().cpu().numpy(), scales[n]), (i, n)
    lens = t.lens.tolist()
    most = max(lens) + 3
    got = paged_peek(pool, t.table, t.lens, most, dtype=dtype)
    for n, g in zip("kv", got):
        for b in range(3):
            want = P.dense(codes[n], scales[n], t.table[b].tolist(), lens[b])
            ref = torch.tensor(want).to(dtype).double().numpy()
            assert np.array_equal(g[b, :, : lens[b]].double().cpu().numpy(), ref)
            assert not g[b, :, lens[b]:].any()
    pool.check_status()
    t.check_status()


@pytest.mark.parametrize("store", ["e4m3", "int8"])
def test_append_hf_layout_strides_and_skips(store) -> None:
    """(B, H, T, D) views with other strides; slots that skip, end and jump."""
    rng = np.random.default_rng(1)
    pool = _pool(store, 6, 2, 16, 64)
    base = _data(rng, (2, 5, 3, 64), torch.bfloat16)           # (B, T, H + 1, D): a projection's layout
    k, v = base.transpose(1, 2)[:, :2], base.transpose(1, 2)[:, 1:]
    slots = [-1, 16, 17, -5, 46, 47, 48, 49, -1, 0]            # row-major over (B, T)
    before = {n: (_values(pool, n), getattr(pool, n + "_scale").double().cpu().numpy()) for n in "kv"}
    paged_append(pool, _i32(slots), k, v)
    for n, x in (("k", k), ("v", v)):
        want = P.append(*before[n], slots, x.transpose(1, 2).reshape(10, 2, 64).double().cpu().numpy(), store)
        assert np.array_equal(_values(pool, n), want[0], equal_nan=True)
        assert np.array_equal(getattr(pool, n + "_scale").double().cpu().numpy(), want[1])
    paged_append(pool, _i32([]), k[:, :, :0], v[:, :, :0])  # nothing
    pool.check_status()


def test_append_slots_out_of_range_are_skipped_and_reported() -> None:
    pool = _pool("int8", 2, 1, 16, 32)
    x = torch.ones(3, 1, 32, device=DEV)
    paged_append(pool, _i32([31, 32, 1 << 30]), x, x)
    # slot 31 continues a page whose scale is 3: its code is round(1 / 3)
    got = _values(pool, "k")
    assert (got[1, 0, 15] == 0).all() and (got[1, 0, :15] == 0x55).all() and (got[0] == 0x55).all()
    assert pool.k_scale.tolist() == [[3.0], [3.0]]
    with pytest.raises(RuntimeError, match="bad indices"):
        pool.check_status()
    pool.check_status()


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dim, page", [(32, 16), (128, 32), (256, 128)])
def test_append_values_that_are_not_finite(store, dim, page) -> None:
    rng = np.random.default_rng(3)
    pool = _pool(store, 3, 3, page, dim)
    x = _data(rng, (page, 3, dim), torch.bfloat16)
    x[0, 0, 3], x[2, 0, 5], x[3, 2, 7] = float("nan"), float("inf"), float("-inf")
    x[:, 1] = 0
    before = _values(pool, "k"), pool.k_scale.double().cpu().numpy()
    slots = list(range(page, 2 * page))
    paged_append(pool, _i32(slots), x, x)
    want = P.append(*before, slots, x.double().cpu().numpy(), store)
    assert np.array_equal(_values(pool, "k"), want[0], equal_nan=True)
    assert np.array_equal(pool.k_scale.double().cpu().numpy(), want[1])
    assert pool.k_scale[1, 1] == 2.0**-100
    with pytest.raises(RuntimeError, match="not finite"):
        pool.check_status()


def test_extreme_magnitudes() -> None:
    """Scales at both ends of their range, subnormal and huge values."""
    pool = _pool("e4m3", 2, 1, 16, 32)
    x = torch.zeros(16, 1, 32, device=DEV)
    x[0, 0, 0], x[1, 0, 0] = 3.0e38, 1e-45
    before = _values(pool, "k"), pool.k_scale.double().cpu().numpy()
    paged_append(pool, _i32(list(range(16))), x, x)
    want = P.append(*before, list(range(16)), x.double().cpu().numpy(), "e4m3")
    assert np.array_equal(_values(pool, "k"), want[0], equal_nan=True) and pool.k_scale[0, 0].item() == want[1][0, 0]
    pool.check_status()


# --------------------------------------------------------------- attention


class _Case:
    """Requests of given lengths in a shuffled pool, and their plain forms."""

    def __init__(self, store, dim, heads, page, lens, seed=0, order="phsd", extra_width=1):
        rng = np.random.default_rng(seed)
        held = [-(-n // page) for n in lens]
        pages = sum(held) + 2
        ids = rng.permutation(pages).tolist()
        self.table_list = []
        width = max(held, default=0) + extra_width
        for n in held:
            self.table_list.append(ids[:n] + [-1] * (width - n))
            ids = ids[n:]
        self.pool = _pool(store, pages, heads, page, dim, order)
        self.table, self.lens_list, self.lens = _i32(self.table_list).view(len(lens), width), list(lens), _i32(lens)
        for b, n in enumerate(lens):
            slots = [self.table_list[b][t // page] * page + t % page for t in range(n)]
            x = [_data(rng, (n, heads, dim), torch.float32) for _ in "kv"]
            paged_append(self.pool, _i32(slots), *x)
        c = {n: _values(self.pool, n) for n in "kv"}
        s = {n: getattr(self.pool, n + "_scale").double().cpu().numpy() for n in "kv"}
        self.dense = [tuple(P.dense(c[n], s[n], self.table_list[b], m) for n in "kv") for b, m in enumerate(lens)]
        vs = s["v"]
        self.vs = [np.repeat(vs[self.table_list[b][: -(-m // page)]], page, axis=0)[:m].T for b, m in enumerate(lens)]  # (H, len)
        self.rng = rng


def _check(case, q_rows, out, lse, scaling, dtype, window=0, starts=None):
    """q_rows, out, lse: one (n, Hq, D), (n, Hq, D), (n, Hq) per request."""
    worst = 0.0
    for b, (q, o, e) in enumerate(zip(q_rows, out, lse)):
        k, v = case.dense[b]
        ref, le, *parts = P.attention(q.double().cpu().numpy(), k, v, scaling, window, 0 if starts is None else starts[b], case.vs[b])
        tol, tol_e = P.bounds(ref, le, *parts, q.shape[-1], max(1, case.lens_list[b]), dtype)
        d = np.abs(o.double().cpu().numpy() - ref)
        assert (d <= tol).all(), (b, float((d / tol).max()))
        g = e.double().cpu().numpy()
        assert np.array_equal(np.isfinite(g), np.isfinite(le)) and (g[~np.isfinite(g)] == -np.inf).all()
        f = np.isfinite(le)
        assert (np.abs(g[f] - le[f]) <= tol_e[f]).all(), b
        worst = max(worst, float((d / tol).max()) if d.size else 0.0)
    return worst


def _run(case, q_lens, group, dtype, window=0, starts=None, scaling=None, max_q=0, **kw):
    heads, dim = case.pool.num_heads, case.pool.head_dim
    scaling = dim**-0.5 if scaling is None else scaling
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(int)
    q = torch.tensor(case.rng.standard_normal((int(cu[-1]), heads * group, dim)), dtype=dtype, device=DEV)
    out, lse = paged_attention(case.pool, case.table, case.lens, q, cu_q=_i32(cu.tolist()), max_q=max_q, scaling=scaling, window=window,
                               starts=None if starts is None else _i32(starts), return_lse=True, **kw)
    cut = [slice(a, b) for a, b in zip(cu[:-1], cu[1:])]
    return _check(case, [q[c] for c in cut], [out[c] for c in cut], [lse[c] for c in cut], scaling, dtype, window, starts)


LENS = [0, 1, 15, 16, 17, 33, 127, 128, 129, 260]


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, heads, group, page", [(32, 2, 3, 16), (64, 2, 4, 16), (64, 1, 8, 64), (128, 2, 4, 32), (128, 1, 12, 128),
                                                     (256, 1, 2, 16), (256, 2, 1, 128)])
def test_decode_lengths(store, dtype, dim, heads, group, page) -> None:
    case = _Case(store, dim, heads, page, LENS)
    _run(case, [1] * len(LENS), group, dtype, max_q=1)
    case.pool.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim, group, page, window", [(64, 4, 16, 0), (64, 1, 32, 7), (128, 4, 64, 0), (128, 7, 16, 100), (256, 2, 32, 0),
                                                      (32, 5, 16, 20)])
def test_ragged_queries(dtype, dim, group, page, window) -> None:
    """Requests with none, one, a few and all of their tokens as queries, and
    with more queries than tokens (rows that see nothing)."""
    lens = [0, 5, 40, 129, 1, 200, 64]
    case = _Case("e4m3", dim, 2, page, lens, seed=5)
    _run(case, [3, 0, 40, 9, 4, 1, 70], group, dtype, window=window)
    case.pool.check_status()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("starts", [[0, 3, 60, 64, 200], [64, 17, 0, 1, 129]])
@pytest.mark.parametrize("n", [1, 20])
def test_left_padding(dim, starts, n) -> None:
    case = _Case("int8", dim, 1, 16, [64, 64, 64, 64, 130], seed=9)
    _run(case, [n] * 5, 4, torch.bfloat16, starts=starts)
    _run(case, [n] * 5, 4, torch.bfloat16, starts=starts, window=11)


@pytest.mark.parametrize("dim, page, n", [(64, 16, 4200), (64, 16, 8193), (128, 128, 4097)])
@pytest.mark.parametrize("q", [1, 3, 40])
def test_long_contexts(dim, page, n, q) -> None:
    """More pages than are staged at a time, split over CTAs, beside short ones."""
    case = _Case("e4m3", dim, 2, page, [n, 2, 700], seed=2)
    _run(case, [q, 1, q], 2, torch.bfloat16)


@pytest.mark.parametrize("order", ["phsd", "pshd"])
def test_uniform_queries_and_strides(order) -> None:
    """(B, Hq, T, D) queries as a projection leaves them, page-slot-head pools,
    a range of KV heads, an output given by the caller."""
    case = _Case("e4m3", 64, 3, 16, [30, 77], seed=4, order=order)
    base = torch.tensor(case.rng.standard_normal((2, 5, 8, 64)), dtype=torch.bfloat16, device=DEV)  # (B, T, heads, D)
    q = base.transpose(1, 2)[:, 1:7]
    out, lse = paged_attention(case.pool, case.table, case.lens, q, return_lse=True)
    rows = [q[b].transpose(0, 1) for b in range(2)]
    _check(case, rows, out, lse, 64**-0.5, torch.bfloat16)
    part = case.pool.heads(1, 2)
    got = paged_attention(part, case.table, case.lens, q[:, 2:])
    assert torch.equal(got, out[:, :, 2:])
    mine = torch.empty_like(out)
    assert paged_attention(case.pool, case.table, case.lens, q, out=mine) is mine and torch.equal(mine, out)
    odd = torch.empty(2 * 6 * 5 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 6, 5, 64).copy_(q)  # 2 bytes off
    assert torch.equal(paged_attention(case.pool, case.table, case.lens, odd), out)


def test_rows_behind_the_last_request() -> None:
    case = _Case("int8", 64, 1, 16, [20, 9], seed=6)
    q = torch.randn(7, 2, 64, device=DEV)
    cu = _i32([0, 2, 5])
    out, lse = paged_attention(case.pool, case.table, case.lens, q, cu_q=cu, return_lse=True)
    assert not out[5:].any() and bool((lse[5:] == -torch.inf).all()) and bool(out[:5].any(-1).all())
    mine = torch.full_like(q, 5.0)
    paged_attention(case.pool, case.table, case.lens, q, cu_q=cu, out=mine)
    assert bool((mine[5:] == 5.0).all()) and torch.equal(mine[:5], out[:5])
    # offsets that make no sense answer nothing, in bounds
    for bad in ([0, 9, 5], [-3, 2, 5], [5, 2, 900]):
        mine.fill_(5.0)
        paged_attention(case.pool, case.table, case.lens, q, cu_q=_i32(bad), out=mine)
    torch.cuda.synchronize()


def test_bad_pages_and_lengths_are_skipped_and_reported() -> None:
    case = _Case("int8", 64, 1, 16, [40, 40], seed=8)
    q = torch.randn(2, 2, 1, 64, device=DEV)
    good = paged_attention(case.pool, case.table, case.lens, q)
    case.pool.check_status()
    t = case.table.clone()
    t[0, 1] = 1 << 20
    out = paged_attention(case.pool, t, case.lens, q)
    assert torch.equal(out[1], good[1]) and bool(out.isfinite().all())
    keep = torch.cat([torch.arange(16), torch.arange(32, 40)]).numpy()
    k, v = (x[:, keep] for x in case.dense[0])
    ref, le, *parts = P.attention(q[0].transpose(0, 1).double().cpu().numpy(), k, v, 0.125, vs=case.vs[0][:, keep])
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= P.bounds(ref, le, *parts, 64, 40, torch.float32)[0]).all()
    with pytest.raises(RuntimeError, match="bad indices"):
        case.pool.check_status()
    paged_peek(case.pool, t, case.lens, 40)
    with pytest.raises(RuntimeError, match="bad indices"):
        case.pool.check_status()
    # lengths beyond the table's columns end with them; negative ones are empty
    wide = _i32([10**9, -4])
    out, lse = paged_attention(case.pool, case.table[:, :3], wide, q, return_lse=True)
    assert not out[1].any() and bool((lse[1] == -torch.inf).all())
    case.pool.check_status()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_nan_and_infinite_queries_stay_in_their_rows(dim, n) -> None:
    case = _Case("e4m3", dim, 1, 16, [70, 70], seed=3)
    q = torch.randn(2, 4, n, dim, device=DEV).to(torch.bfloat16)
    good = paged_attention(case.pool, case.table, case.lens, q)
    q[0, 1, n // 2, 5] = float("nan")
    q[1, 2, 0, 0] = float("inf")
    out = paged_attention(case.pool, case.table, case.lens, q)
    same = torch.ones(2, n, 4, dtype=torch.bool, device=DEV)
    same[0, n // 2, 1] = same[1, 0, 2] = False
    assert torch.equal(out[same], good[same])
    assert bool(out[0, n // 2, 1].isnan().all())


def test_later_tokens_do_not_reach_earlier_queries() -> None:
    """What lies behind a query changes nothing in its row."""
    a = _Case("e4m3", 64, 2, 16, [50], seed=1)
    q = torch.randn(1, 4, 20, 64, device=DEV).to(torch.bfloat16)
    whole = paged_attention(a.pool, a.table, a.lens, q)
    fewer = paged_attention(a.pool, a.table, _i32([40]), q[:, :, :10])
    assert float((whole[:, :10].double() - fewer.double()).abs().max()) <= 2.0**-8 * float(whole.double().abs().max())


def test_other_streams_and_two_calls_at_once() -> None:
    case = _Case("e4m3", 128, 2, 32, [5000, 33, 900], seed=7)
    qs = [torch.randn(3, 8, 1, 128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    want = [paged_attention(case.pool, case.table, case.lens, q) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(case.pool, case.table, case.lens, qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)


def test_repeated_calls_give_the_same_bits() -> None:
    case = _Case("int8", 64, 2, 16, [3000, 17], seed=11)
    q = torch.randn(2, 8, 4, 64, device=DEV).to(torch.float16)
    first = paged_attention(case.pool, case.table, case.lens, q)
    for _ in range(5):
        assert torch.equal(paged_attention(case.pool, case.table, case.lens, q), first)


def _step(t, pool, new, cap, k, v, q):
    plan = t.advance(new, cap)
    paged_append(pool, plan.slots, k, v)
    return paged_attention(pool, t.table, t.lens, q, cu_q=plan.cu_new, max_q=2), plan


def test_serving_steps_and_their_captured_graph() -> None:
    """Advance, append and attend as a serving loop runs them: eager, and as
    one captured graph replayed with new inputs, give the same bits."""
    runs = []
    for captured in (False, True):
        g = torch.Generator(device=DEV).manual_seed(0)
        t = PageTables(4, 8, 24, 16, DEV)
        pool = PagedPool.allocate(24, 16, 2, 64, device=DEV)
        k0, v0 = (torch.randn(60, 2, 64, device=DEV, generator=g).to(torch.bfloat16) for _ in "kv")
        plan = t.advance(_i32([31, 0, 20, 9]), 60)
        paged_append(pool, plan.slots, k0, v0)
        new = _i32([0, 0, 0, 0])
        k, v = (torch.zeros(6, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in "kv")
        q = torch.zeros(6, 8, 64, device=DEV, dtype=torch.bfloat16)
        outs = []
        if captured:
            saved = [x.clone() for x in (t.table, t.lens, t.free_count, pool.k.view(torch.uint8), pool.k_scale, pool.v.view(torch.uint8), pool.v_scale)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out, _ = _step(t, pool, new, 6, k, v, q)
            for x, y in zip((t.table, t.lens, t.free_count, pool.k.view(torch.uint8), pool.k_scale, pool.v.view(torch.uint8), pool.v_scale), saved):
                assert torch.equal(x, y)  # capture ran nothing
        for step in ([1, 2, 1, 1], [1, 0, 2, 1], [0, 1, 1, 2], [2, 2, 0, 2], [1, 1, 1, 1]):
            new.copy_(_i32(step))
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, device=DEV, generator=g).to(x.dtype) * len(outs))
            if captured:
                graph.replay()
                outs.append(out.clone())
            else:
                outs.append(_step(t, pool, new, 6, k, v, q)[0].clone())
        t.release(torch.tensor([True, False, False, False], device=DEV))
        t.check_status()
        pool.check_status()
        runs.append(outs + [t.table.clone(), t.lens.clone(), t.free_count.clone(), pool.k.view(torch.uint8).clone(), pool.v_scale.clone()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    # and against the plain form, for the last step
    assert bool(runs[0][4][:4].float().abs().sum(-1).gt(0).all())


def test_offsets_past_32_bits() -> None:
    """A pool whose codes lie over more than 4 GiB: its last pages are read and written there."""
    pages, heads, page, dim = 70_000, 4, 128, 128  # 4.6 GB of codes each
    pool = PagedPool.allocate(pages, page, heads, dim, device=DEV)
    ids = [pages - 1, 3, pages - 2]
    table, lens = _i32([ids]), _i32([300])
    slots = torch.cat([torch.arange(128) + i * 128 for i in ids])[:300].to(torch.int32).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(300, heads, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in "kv")
    paged_append(pool, slots, k, v)
    dk, dv = paged_peek(pool, table, lens, 300)
    assert float((dk[0].transpose(0, 1).float() - k.float()).abs().max()) <= 2.0**-4 * float(k.float().abs().max())
    q = torch.randn(1, 8, 1, dim, device=DEV, generator=g).to(torch.bfloat16)
    out, lse = paged_attention(pool, table, lens, q, return_lse=True)
    kd, vd = dk[0].double().cpu().numpy(), dv[0].double().cpu().numpy()
    ref, le, *parts = P.attention(q[0].transpose(0, 1).double().cpu().numpy(), kd, vd, dim**-0.5)
    tol, _ = P.bounds(ref, le, *parts, dim, 300, torch.bfloat16)
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= tol).all()


def test_refusals_of_calls() -> None:
    case = _Case("int8", 64, 2, 16, [20], seed=0)
    q = torch.randn(1, 4, 1, 64, device=DEV)
    with pytest.raises(ValueError, match="query heads"):
        paged_attention(case.pool, case.table, case.lens, q[:, :3])
    with pytest.raises(NotImplementedError, match="float32, bfloat16 or float16"):
        paged_attention(case.pool, case.table, case.lens, q.double())
    with pytest.raises(ValueError, match="lens must be"):
        paged_attention(case.pool, case.table, case.lens.long(), q)
    with pytest.raises(ValueError, match="requests' queries"):
        paged_attention(case.pool, case.table, case.lens, q.expand(2, -1, -1, -1))
    with pytest.raises(ValueError, match="out must be"):
        paged_attention(case.pool, case.table, case.lens, q, out=torch.empty(1, 1, 4, 64, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError, match="window"):
        paged_attention(case.pool, case.table, case.lens, q, window=-1)
    with pytest.raises(ValueError, match="is on cpu"):
        paged_attention(case.pool, case.table, case.lens.cpu(), q)
    with pytest.raises(NotImplementedError, match="inference only"):
        paged_attention(case.pool, case.table, case.lens, q.requires_grad_())
    with pytest.raises(NotImplementedError, match="inference only"):
        paged_append(case.pool, _i32([0]), torch.ones(1, 2, 64, device=DEV, requires_grad=True), torch.ones(1, 2, 64, device=DEV))
    with pytest.raises(ValueError, match="slots must be"):
        paged_append(case.pool, _i32([0, 1]), torch.ones(1, 2, 64, device=DEV), torch.ones(1, 2, 64, device=DEV))
    with pytest.raises(ValueError, match="pool holds"):
        paged_append(case.pool, _i32([0]), torch.ones(1, 3, 64, device=DEV), torch.ones(1, 3, 64, device=DEV))
    with pytest.raises(NotImplementedError, match="dtype must be"):
        paged_peek(case.pool, case.table, case.lens, 4, dtype=torch.float64)
    with pytest.raises(ValueError, match="done must be"):
        PageTables(2, 2, 4, 16, DEV).release(torch.ones(2, device=DEV))


@pytest.mark.parametrize("dim", [64, 128])
def test_many_short_requests_of_a_few_rows(dim) -> None:
    """Hundreds of units that fill half a pair of row tiles, several to a CTA,
    beside one that fills both: the row tiles run at their own pace."""
    lens = [40 + (37 * i) % 300 for i in range(150)]
    case = _Case("e4m3", dim, 4, 32, lens, seed=12)
    q_lens = [5] * 150
    q_lens[75] = 40
    out = _run(case, q_lens, 4, torch.bfloat16)
    assert out <= 1.0
    case.pool.check_status()


@pytest.mark.parametrize("dim, order, dtype", [(64, "pshd", torch.bfloat16), (128, "pshd", torch.float16), (128, "phsd", torch.bfloat16)])
def test_chunks_of_strided_pools_and_queries(dim, order, dtype) -> None:
    """Many rows over page-slot-head pools, a range of KV heads, (B, Hq, T, D)
    queries as a projection leaves them, lengths at the tiles' borders."""
    case = _Case("int8", dim, 3, 32, [127, 300, 128, 64], seed=14, order=order)
    base = torch.tensor(case.rng.standard_normal((4, 61, 8, dim)), dtype=dtype, device=DEV)  # (B, T, heads, D)
    q = base.transpose(1, 2)[:, 1:7]
    out, lse = paged_attention(case.pool, case.table, case.lens, q, return_lse=True)
    _check(case, [q[b].transpose(0, 1) for b in range(4)], out, lse, dim**-0.5, dtype)
    part = paged_attention(case.pool.heads(1, 2), case.table, case.lens, q[:, 2:])
    assert float((part.double() - out[:, :, 2:].double()).abs().max()) <= 2.0**-7 * float(out.double().abs().max())  # other units, other splits
    case.pool.check_status()


@pytest.mark.parametrize("n", [1, 30])
def test_a_window_beyond_every_length_hides_nothing(n) -> None:
    case = _Case("e4m3", 64, 1, 16, [40, 3], seed=15)
    q = torch.randn(2, 2, n, 64, device=DEV).to(torch.bfloat16)
    plain = paged_attention(case.pool, case.table, case.lens, q)
    for window in (40, 2**31 - 1):
        assert torch.equal(paged_attention(case.pool, case.table, case.lens, q, window=window), plain)


def test_scales_of_another_size_and_zero() -> None:
    """Attention and peek take any scales: values' scales 2^60 apart, one of 0."""
    for n in (1, 24):
        case = _Case("int8", 64, 1, 16, [64, 50], seed=16)
        ids = case.table_list[0]
        case.pool.v_scale[ids[0]] *= 2.0**30
        case.pool.v_scale[ids[2]] *= 2.0**-30
        case.pool.v_scale[ids[1]] = 0
        case.pool.k_scale[ids[3]] = 0
        s = {x: getattr(case.pool, x + "_scale").double().cpu().numpy() for x in "kv"}
        case.dense = [tuple(P.dense(_values(case.pool, x), s[x], case.table_list[b], m) for x in "kv") for b, m in enumerate(case.lens_list)]
        vs = np.repeat(s["v"][ids[:4]], 16, axis=0).T
        case.vs[0] = np.where(vs == 0, 2.0**-20, vs)  # a scale of 0: values of 0, whatever it counts as
        _run(case, [n, n], 4, torch.bfloat16)


def test_nothing_to_do() -> None:
    pool = PagedPool.allocate(4, 16, 2, 64, device=DEV)
    none = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    q = torch.randn(5, 4, 64, device=DEV)
    out, lse = paged_attention(pool, none, _i32([]), q, cu_q=_i32([0]), return_lse=True)
    assert not out.any() and bool((lse == -torch.inf).all())
    empty = torch.empty((2, 0), dtype=torch.int32, device=DEV)
    out = paged_attention(pool, empty, _i32([0, 0]), q[:2, :, None])
    assert out.shape == (2, 1, 4, 64) and not out.any()
    assert not paged_peek(pool, empty, _i32([0, 0]), 3)[0].any()
    assert paged_peek(pool, empty, _i32([0, 0]), 0)[1].shape == (2, 2, 0, 64)
    assert paged_attention(pool, _i32([[0]]), _i32([1]), q[:0], cu_q=_i32([0, 0])).shape == (0, 4, 64)
    p = build_page_tables(_i32([0, 3]), _i32([0, 0]), _i32([[-1], [2]]), _i32([]), _i32([0]), page_size=16, capacity=0)
    assert p.cu_new.tolist() == [0, 0, 0] and p.lens.tolist() == [0, 3] and p.free_count.item() == 0


def test_more_refusals() -> None:
    case = _Case("int8", 64, 2, 16, [20], seed=0)
    q = torch.randn(1, 4, 1, 64, device=DEV)
    for scaling in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scaling"):
            paged_attention(case.pool, case.table, case.lens, q, scaling=scaling)
    with pytest.raises(ValueError, match="memory of its own"):
        paged_attention(case.pool, case.table, case.lens, q, out=q.view(1, 1, 4, 64))


def test_a_captured_call_and_an_eager_one_side_by_side() -> None:
    """Two graphs and an eager call of one pool, on three streams at once."""
    case = _Case("e4m3", 64, 2, 16, [2000, 900], seed=17)
    qs = [torch.randn(2, 8, n, 64, device=DEV).to(torch.bfloat16) for n in (1, 40, 1)]
    want = [paged_attention(case.pool, case.table, case.lens, q) for q in qs]
    graphs, outs = [], []
    for q in qs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(case.pool, case.table, case.lens, q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = paged_attention(case.pool, case.table, case.lens, qs[2])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs + [eager], want))
