"""Host-side checks of the 8-bit paged cache that need no GPU: the Python
layer's refusals, the C entry points' own (they return before any launch),
and the plain forms that the GPU tests compare with."""

from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import paged_plain as P

from kvdlra_b200 import _native as N
from kvdlra_b200 import paged
from kvdlra_b200.paged import PagedPool, PageTables, build_page_tables

REPO = Path(__file__).resolve().parent.parent


def _pool_tensors(pages=4, heads=2, page=16, dim=64, dtype=torch.int8):
    k = torch.zeros(pages, heads, page, dim, dtype=torch.uint8).view(dtype)
    return [k, k.clone(), torch.zeros(pages, heads), torch.zeros(pages, heads)]


def test_pool_refusals() -> None:
    def make(**kw):
        return PagedPool(*_pool_tensors(**kw))

    with pytest.raises(NotImplementedError, match="float8_e4m3fn or int8"):
        make(dtype=torch.uint8)
    with pytest.raises(ValueError, match="page_size must be one of"):
        make(page=24)
    with pytest.raises(ValueError, match="head_dim must be one of"):
        make(dim=80)
    t = _pool_tensors()
    t[1] = t[1][:3]
    with pytest.raises(ValueError, match="alike"):
        PagedPool(*t)
    t = _pool_tensors()
    t[2] = t[2].double()
    with pytest.raises(ValueError, match="k_scale must be float32"):
        PagedPool(*t)
    t = _pool_tensors()
    t[0] = t[0].transpose(2, 3).contiguous().transpose(2, 3)
    with pytest.raises(ValueError, match="contiguous D"):
        PagedPool(*t)
    t = _pool_tensors()
    t[0] = t[0][:1].expand(4, -1, -1, -1)
    with pytest.raises(ValueError, match="strides"):
        PagedPool(*t)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        make()
    with pytest.raises(ValueError, match="storage must be"):
        PagedPool.allocate(4, 16, 2, 64, storage="int4", device="cpu")


def test_table_refusals() -> None:
    z = torch.zeros(3, dtype=torch.int32)
    table, free, count = torch.zeros(3, 4, dtype=torch.int32), torch.arange(9, dtype=torch.int32), torch.ones(1, dtype=torch.int32)

    def call(cached=z, new=z, table=table, free=free, count=count, page_size=16, capacity=8):
        return build_page_tables(cached, new, table, free, count, page_size=page_size, capacity=capacity)

    with pytest.raises(ValueError, match="cached_lens must be a contiguous int32"):
        call(cached=z.long())
    with pytest.raises(ValueError, match="new_lens must be a contiguous int32"):
        call(new=z[:2])
    with pytest.raises(ValueError, match="table must be int32"):
        call(table=table[:2])
    with pytest.raises(ValueError, match="page_size"):
        call(page_size=20)
    with pytest.raises(ValueError, match="capacity"):
        call(capacity=-1)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        call()
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        PageTables(2, 4, 8, 16, device="cpu")


def _c_pool(**kw) -> N.PagedPool:
    d = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, page_stride=2048, head_stride=1024, slot_stride=64, scale_stride=2,
             num_pages=4, page_size=16, num_heads=2, head_dim=64, store=0, status=None)
    return N.PagedPool(*{**d, **kw}.values())


@pytest.mark.parametrize("kw, what", [
    (dict(k=None), "null"), (dict(store=3), "unknown store"), (dict(page_size=48), "page_size"), (dict(head_dim=96), "head_dim"),
    (dict(num_pages=0), "pages"), (dict(num_pages=1 << 28), "pages"), (dict(slot_stride=72), "16 bytes"), (dict(k=(1 << 20) + 8), "16 bytes"),
    (dict(scale_stride=1), "scale_stride"),
])
def test_c_pool_refusals(kw, what) -> None:
    """The addresses are never read: every refusal comes before a launch."""
    L = N.lib()
    p = _c_pool(**kw)
    v = N.HFView(1 << 20, 0, 64, 128, 4)
    assert L.kvd_paged_append(C.byref(p), 1 << 20, 1, 1, v, v, None) != 0
    assert what in L.kvd_last_error().decode()
    assert L.kvd_paged_attention_workspace_bytes(C.byref(p), 1, 8) == 0


def test_c_call_refusals() -> None:
    L, p, a = N.lib(), _c_pool(), 1 << 20
    ref = C.byref(p)

    def attention(dtype=1, batch=2, stride=4, pages=4, sb=512, sh=64, st=512, tokens=1, hq=8, window=0, q=a, ws=a, ws_bytes=1 << 40):
        return L.kvd_paged_attention(ref, batch, a, stride, pages, a, None, None, dtype, q, sb, sh, st, tokens, 0, hq, 1.0, window, a, None, 0,
                                     ws, ws_bytes, None)

    for kw, what in ((dict(dtype=7), "dtype"), (dict(hq=3), "query heads"), (dict(batch=-1), "negative"), (dict(stride=3), "stride"),
                     (dict(window=-1), "negative"), (dict(q=a + 2), "16 bytes"), (dict(sh=60), "16 bytes"), (dict(ws=None), "workspace"),
                     (dict(ws_bytes=64), "workspace"), (dict(q=None), "null"), (dict(tokens=1 << 30), "too many")):
        assert attention(**kw) != 0, kw
        assert what in L.kvd_last_error().decode(), (kw, L.kvd_last_error())
    assert attention(batch=0) == 0 and attention(tokens=0) == 0  # nothing to do
    v, w = N.HFView(a, 0, 64, 128, 4), N.HFView(a, 0, 64, 128, 5)
    assert L.kvd_paged_append(ref, a, 1, 1, v, w, None) != 0 and "tokens" in L.kvd_last_error().decode()
    assert L.kvd_paged_append(ref, a, 1, 9, v, v, None) != 0 and "dtype" in L.kvd_last_error().decode()
    assert L.kvd_paged_append(ref, a, 1, 1, N.HFView(a, 0, 60, 128, 4), v, None) != 0 and "16 bytes" in L.kvd_last_error().decode()
    assert L.kvd_paged_append(ref, None, 0, 1, v, v, None) == 0
    assert L.kvd_paged_peek(ref, 40000, a, 4, 4, a, 1, v, v, None) != 0 and "batch" in L.kvd_last_error().decode()
    assert L.kvd_paged_peek(ref, 2, None, 4, 4, a, 1, v, v, None) != 0

    def tables(batch=2, pages=4, page=16, stride=4, num_free=8, capacity=16, lens=a):
        return L.kvd_page_tables(batch, pages, page, a, a, a, stride, a, num_free, a, capacity, lens, a, a, a, a, None, None, 0, None)

    for kw, what in ((dict(batch=0), "batch"), (dict(batch=20000), "batch"), (dict(page=8), "page_size"), (dict(stride=2), "stride"),
                     (dict(num_free=-1), "free"), (dict(capacity=-1), "capacity"), (dict(lens=None), "null")):
        assert tables(**kw) != 0, kw
        assert what in L.kvd_last_error().decode(), (kw, L.kvd_last_error())
    assert L.kvd_page_release(2, 4, 16, None, a, a, 4, a, 8, a, None, None) != 0
    assert L.kvd_paged_check_status(None, None) != 0


def test_pool_struct_matches_the_header() -> None:
    text = (REPO / "include" / "kvdlra_b200.h").read_text()
    body = re.search(r"typedef struct kvd_paged_pool \{(.*?)\} kvd_paged_pool;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).replace("*", " ")
    names = re.findall(r"([a-z_]+)\s*(?=[;,])", body)
    assert [f for f, _ in N.PagedPool._fields_] == names


def test_plain_rounding_is_the_types_own() -> None:
    """The plain forms' code grids against torch's casts."""
    x = torch.linspace(-500, 500, 40001, dtype=torch.float64)
    x = torch.cat([x, x / 1000, torch.tensor([448.0, 464.0, -1e9, 2.0**-9, 2.0**-10, 3 * 2.0**-10])])
    want = x.clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn).double().numpy()
    y = x.clamp(-448, 448).to(torch.float32).double().numpy()
    assert np.array_equal(P.round_code(y, "e4m3"), want)
    assert np.array_equal(P.round_code(np.array([0.5, 1.5, -2.5, 200.0]), "int8"), [0, 2, -2, 127])
    for store, top in P.TOP.items():
        for a in (top, np.nextafter(top, 1e9), 1.0, 3e38, 0.0, 1e-45):
            s = P.scale_of(a, store)
            assert a <= top * s and (s == 2.0**-100 or a > top * s / 2)


def test_plain_tables_hand_worked() -> None:
    ok, table, lens, cu, slots, pos, left = P.tables([3, 16, 0], [2, 1, 0], [[5, 0], [7, 0], [0, 0]], [1, 2, 9], 16, 5)
    assert ok and table == [[5, 0], [7, 9], [0, 0]] and lens == [5, 17, 0] and cu == [0, 2, 3, 3] and left == 2
    assert slots == [5 * 16 + 3, 5 * 16 + 4, 9 * 16, -1, -1] and pos == [3, 4, 16, 0, 0]


def test_module_exports() -> None:
    assert all(hasattr(paged, n) for n in paged.__all__)


def test_cache_refusals() -> None:
    from kvdlra_b200 import PagedKVCache

    for kw, what in ((dict(max_tokens=0), "max_tokens"), (dict(page_size=24), "page_size"), (dict(storage="int4"), "storage"),
                     (dict(left_padding=torch.tensor([-1])), "left_padding"), (dict(left_padding=torch.zeros(2)), "left_padding")):
        with pytest.raises(ValueError, match=what):
            PagedKVCache(None, **{"max_tokens": 8, "num_layers": 1, **kw})
    cache = PagedKVCache(None, 8, num_layers=2)
    k = torch.zeros(1, 2, 3, 32)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        cache.update(k, k, 0)
    assert cache.get_seq_length() == 0 and cache.get_mask_sizes(3, 0) == (3, 0) and cache.stored_state_numel() == 0
