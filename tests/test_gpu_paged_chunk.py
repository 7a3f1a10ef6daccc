"""Requests of more query rows than the few-row kernel takes (33 and up: bf16 and
f16, head_dim 64 and 128), where the tensor-memory kernel's own order of work
counts: the same bits from every call, alone and beside another, and pages that
lie beyond 4 GiB."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_plain as P
from test_gpu_paged import DEV, _Case, _i32, _run

from kvdlra_b200 import _native as N
from kvdlra_b200.paged import PagedPool, paged_append, paged_attention, paged_peek

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, dtype, store", [(64, torch.bfloat16, "e4m3"), (128, torch.float16, "int8"), (128, torch.bfloat16, "e4m3")])
@pytest.mark.parametrize("tokens", [12, 40, 300])  # rows 48 (one row tile), 160 and 1200 (two, and units of one behind them)
def test_repeated_chunks_give_the_same_bits(dim, dtype, store, tokens) -> None:
    """The next scores go where the weights lay that the product before reads: a
    product that ran late would show as other bits, or as a wrong row."""
    case = _Case(store, dim, 2, 64, [4000, 321, 1500], seed=21)
    q = torch.randn(3, 8, tokens, dim, device=DEV).to(dtype)
    first, lse = paged_attention(case.pool, case.table, case.lens, q, return_lse=True)
    rows = [q[b].transpose(0, 1) for b in range(3)]
    some = slice(0, tokens, max(1, tokens // 5))
    n = torch.arange(tokens)[some].tolist()
    for i in n:  # rows of the plain form, each as the last query of a shorter request
        cut = [m - (tokens - 1 - i) for m in case.lens_list]
        for b, m in enumerate(cut):
            k, v = (x[:, :m] for x in case.dense[b])
            ref, le, *parts = P.attention(rows[b][i : i + 1].double().cpu().numpy(), k, v, dim**-0.5, vs=case.vs[b][:, :m])
            tol, tol_e = P.bounds(ref, le, *parts, dim, m, dtype)
            assert (np.abs(first[b, i : i + 1].double().cpu().numpy() - ref) <= tol).all()
            assert (np.abs(lse[b, i : i + 1].double().cpu().numpy() - le) <= tol_e).all()
    for _ in range(60):
        out, e = paged_attention(case.pool, case.table, case.lens, q, return_lse=True)
        assert torch.equal(out, first) and torch.equal(e, lse)
    case.pool.check_status()


@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_on_two_streams_at_once(dim) -> None:
    case = _Case("e4m3", dim, 2, 32, [3000, 777], seed=22)
    qs = [torch.randn(2, 8, n, dim, device=DEV).to(torch.bfloat16) for n in (40, 200)]
    want = [paged_attention(case.pool, case.table, case.lens, q) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(case.pool, case.table, case.lens, qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)
    case.pool.check_status()


def test_chunks_of_pages_past_32_bits() -> None:
    """The loaders' page offsets beyond 4 GiB."""
    pages, heads, page, dim = 70_000, 4, 128, 128  # 4.6 GB of codes each
    pool = PagedPool.allocate(pages, page, heads, dim, device=DEV)
    ids = [pages - 1, 3, pages - 2]
    table, lens = _i32([ids]), _i32([300])
    slots = torch.cat([torch.arange(128) + i * 128 for i in ids])[:300].to(torch.int32).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(300, heads, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in "kv")
    paged_append(pool, slots, k, v)
    dk, dv = (x[0].double().cpu().numpy() for x in paged_peek(pool, table, lens, 300, dtype=torch.float32))
    q = torch.randn(1, 8, 40, dim, device=DEV, generator=g).to(torch.bfloat16)
    out, lse = paged_attention(pool, table, lens, q, return_lse=True)
    vs = pool.v_scale[torch.tensor(ids, device=DEV)].double().cpu().numpy()
    ref, le, *parts = P.attention(q[0].transpose(0, 1).double().cpu().numpy(), dk, dv, dim**-0.5, vs=np.repeat(vs, page, axis=0)[:300].T)
    tol, tol_e = P.bounds(ref, le, *parts, dim, 300, torch.bfloat16)
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= tol).all()
    assert (np.abs(lse[0].double().cpu().numpy() - le) <= tol_e).all()
    pool.check_status()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_wait_that_runs_out_sets_the_status(dim) -> None:
    """With no patience at all, some wait gives up (the planner, eight units
    ahead, waits for one of 512 tiles): the call ends, the status says so, and the next call is right."""
    n, page = 65536, 128
    pool = PagedPool.allocate(n // page, page, 1, dim, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(n, 1, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in "kv")
    paged_append(pool, torch.arange(n, dtype=torch.int32, device=DEV), k, v)
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).repeat(1480, 1)
    lens = torch.full((1480,), n, dtype=torch.int32, device=DEV)
    q = torch.randn(1480, 40, 1, dim, device=DEV, generator=g).to(torch.bfloat16)
    want = paged_attention(pool, table, lens, q)
    pool.check_status()
    L = N.lib()
    try:
        assert L.kvd_paged_wait_limit(-1) == 0
        paged_attention(pool, table, lens, q)
        with pytest.raises(RuntimeError, match="timed out"):
            pool.check_status()
    finally:
        L.kvd_paged_wait_limit(0)
    assert torch.equal(paged_attention(pool, table, lens, q), want)
    pool.check_status()


@pytest.mark.parametrize("dim", [64, 128])
def test_many_short_requests_of_one_row_tile(dim) -> None:
    """Hundreds of units that fill half a pair of row tiles, several to a CTA, beside
    one that fills both and a few of the other kernel's."""
    lens = [40 + (37 * i) % 300 for i in range(150)]
    case = _Case("e4m3", dim, 4, 32, lens, seed=12)
    q_lens = [12 if i % 10 else 1 + i % 8 for i in range(150)]
    q_lens[75] = 40
    assert _run(case, q_lens, 4, torch.bfloat16) <= 1.0
    case.pool.check_status()


@pytest.mark.parametrize("dim, dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("group, tokens", [(16, 1), (17, 1), (32, 1), (33, 1), (8, 4), (11, 3), (64, 1), (1, 32), (1, 33), (43, 3)])
def test_rows_at_the_border_of_the_two_kernels(dim, dtype, group, tokens) -> None:
    case = _Case("int8", dim, 1, 16, [200, 33, 1], seed=13)
    _run(case, [tokens] * 3, group, dtype)
    _run(case, [tokens, 0, 1], group, dtype, window=20)
    case.pool.check_status()
