"""Calls of the 8-bit paged cache at the edges of what its documentation allows,
as far as the host sees them."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from kvdlra_b200 import _native as N
from kvdlra_b200 import paged
from kvdlra_b200.paged import build_page_tables


@pytest.mark.parametrize("capacity", [2**31, 2**32 + 5])
def test_capacities_past_32_bits_are_refused(capacity) -> None:
    z = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="capacity"):
        build_page_tables(z, z, torch.zeros(3, 4, dtype=torch.int32), torch.arange(9, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                          page_size=16, capacity=capacity)


def test_tangents_are_refused() -> None:
    """Forward-mode differentiation would end at the codes without a word."""
    import torch.autograd.forward_ad as fwd

    x = torch.ones(2, 3)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones(2, 3))
        for args in ((d,), (x, d), (d, x)):
            with pytest.raises(NotImplementedError, match="inference only"):
                paged._no_grad(*args)
        paged._no_grad(x, x)
    paged._no_grad(x)
    with pytest.raises(NotImplementedError, match="inference only"):
        paged._no_grad(x, torch.ones(2, requires_grad=True))


def test_new_lengths_of_their_own() -> None:
    """In place, the lengths are overwritten while the new ones are still read."""
    z, table = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    free, count = torch.arange(9, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="new_lens must have memory of their own"):
        build_page_tables(z, z, table, free, count, page_size=16, capacity=4, in_place=True)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        build_page_tables(z, z, table, free, count, page_size=16, capacity=4)


def test_calls_with_hints_refuse_what_the_plain_ones_do() -> None:
    """The addresses are never read: every refusal comes before a launch."""
    L, a = N.lib(), 1 << 20
    p = N.PagedPool(a, 2 * a, 3 * a, 4 * a, 2048, 1024, 64, 2, 4, 16, 2, 64, 0, None)
    ref, v, w = C.byref(p), N.HFView(a, 0, 64, 128, 4), N.HFView(a, 0, 64, 128, 5)
    assert L.kvd_paged_append_runs(ref, a, 1, 1, v, v, -1, None) != 0
    assert L.kvd_paged_append_runs(ref, a, 1, 1, v, w, 1, None) != 0 and "tokens" in L.kvd_last_error().decode()
    assert L.kvd_paged_append_runs(ref, a, 1, 9, v, v, 1, None) != 0 and "dtype" in L.kvd_last_error().decode()
    assert L.kvd_paged_append_runs(ref, None, 0, 1, v, v, 1, None) == 0
    assert L.kvd_paged_attention(ref, 2, None, 4, 4, a, None, None, 1, a, 512, 64, 512, 1, 0, 8, 1.0, 0, a, None, 0, a, 1 << 40, None) != 0
    assert "null" in L.kvd_last_error().decode()
    for clocks in (-5, 1, 1 << 62, 0):
        assert L.kvd_paged_wait_limit(clocks) == 0
