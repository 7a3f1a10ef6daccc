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
from test_gpu_paged import DEV, _Case, _i32, _pool

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
