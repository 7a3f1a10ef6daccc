"""An 8-bit paged KV cache: page tables, the quantising writer, the dense
reader and attention over the pages.

The cache holds every token of requests of their own lengths, as 8-bit codes
(``torch.float8_e4m3fn`` or ``torch.int8``) in pages of ``page_size`` tokens,
with one scale for each (page, KV head): ``x = code * scale``.  It is the
full-length counterpart of :class:`kvdlra_b200.BugStreamingCache`, whose
memory it is compared against, and serves ragged batches.

A serving step is four calls, all on the current stream, with lengths, tables
and slots on the device throughout::

    plan = tables.advance(new_lens, capacity)            # pages, slots, positions
    paged_append(pool, plan.slots, k, v)                 # per layer; max_new= the most new tokens of a request
    out = paged_attention(pool, tables.table, tables.lens, q, cu_q=plan.cu_new, scaling=s)
    tables.release(done)                                 # finished requests

Every call but ``check_status`` can be captured in a CUDA graph.  Bad slots
and page ids are skipped on the device and reported by ``check_status``.
Inference only: there is no gradient through the codes, and inputs that
require one are refused while gradients are recorded, inputs with a tangent always.  The reference has no
counterpart of these operators.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.forward_ad import unpack_dual

from . import _native as N

__all__ = ["PagedPool", "PageTables", "PagePlan", "build_page_tables", "paged_append", "paged_attention",
           "paged_peek", "PAGE_SIZES", "HEAD_DIMS"]

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128, 256)
_STORES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_NAMES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_INT_MAX = 2**31 - 1  # the C calls' sizes; ctypes would cut larger ones
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _call(device: torch.device, fn: object, name: str, *args: object) -> None:
    """``_native.call``, with the device switched only where it is not current."""
    if torch.cuda.current_device() == device.index:
        code = fn(*args)  # type: ignore[operator]
    else:
        with torch.cuda.device(device):
            code = fn(*args)  # type: ignore[operator]
    if code:
        N.check(code, name)


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _dtype(t: Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise NotImplementedError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _ints(t: Tensor, shape: tuple[int, ...], what: str, device: torch.device) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the rest on {device}")


def _table(t: Tensor, batch: int | None, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.stride(1) != 1 or t.shape[1] > _INT_MAX or (batch is not None and t.shape[0] != batch):
        raise ValueError(f"table must be int32 (batch{'' if batch is None else ' ' + str(batch)}, pages) with contiguous rows, got "
                         f"{t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"table is on {t.device}, the rest on {device}")


def _cuda(device: torch.device) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"kvdlra_b200.paged runs on CUDA devices only (no CPU fallback); got a tensor on {device}")


def _no_grad(a: Tensor, b: Tensor | None = None) -> None:
    if (a.requires_grad or (b is not None and b.requires_grad)) and torch.is_grad_enabled():
        raise NotImplementedError("the 8-bit paged cache is inference only: call it under torch.no_grad()")
    if unpack_dual(a).tangent is not None or (b is not None and unpack_dual(b).tangent is not None):
        raise NotImplementedError("the 8-bit paged cache is inference only: it carries no tangents")


def _rows(t: Tensor) -> tuple[Tensor, N.HFView]:
    """``t`` ``(B, H, T, D)`` or packed ``(T, H, D)`` with a contiguous,
    16-byte-aligned last dimension (a copy where it has none), and its C view.
    Strides of dimensions of one element, which are never used, count as 0."""
    st, sh, n = t.stride(), t.shape, 16 // t.element_size()
    if len(sh) == 3:
        tokens, sb, hs, ts = sh[0], 0, st[1] if sh[1] > 1 else 0, st[0] if sh[0] > 1 else 0
    else:
        tokens, sb, hs, ts = sh[2], st[0] if sh[0] > 1 else 0, st[1] if sh[1] > 1 else 0, st[2] if sh[2] > 1 else 0
    ptr = t.data_ptr()
    if st[-1] != 1 or ptr % 16 or sb % n or hs % n or ts % n:
        return _rows(t.clone(memory_format=torch.contiguous_format))
    return t, N.HFView(ptr, sb, hs, ts, tokens)


class PagedPool:
    """One layer's pages: codes ``k``, ``v`` ``(num_pages, H, page_size, D)``
    (any strides that are multiples of 16 bytes, both alike, with contiguous
    ``D``: the page-head-slot and the page-slot-head order are both such) and
    fp32 scales ``k_scale``, ``v_scale`` ``(num_pages, H)``.

    The tensors stay the caller's; :meth:`allocate` makes them.  Scales that
    this package writes are powers of two; attention and peek read any."""

    def __init__(self, k: Tensor, v: Tensor, k_scale: Tensor, v_scale: Tensor, *, status: Tensor | None = None) -> None:
        if k.dtype not in _STORES or v.dtype != k.dtype:
            raise NotImplementedError(f"codes must be float8_e4m3fn or int8, both alike, got {k.dtype} and {v.dtype}")
        _need(k.dim() == 4 and v.shape == k.shape, f"k and v must be (num_pages, H, page_size, D) alike, got {tuple(k.shape)} and {tuple(v.shape)}")
        pages, heads, page, dim = k.shape
        _need(page in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, got {page}")
        _need(dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {dim}")
        _need(pages >= 1 and 1 <= heads <= 1024 and pages * page < 2**31, f"{pages} pages of {page} tokens, {heads} heads")
        st = tuple(s if n > 1 else max(dim, s // 16 * 16) for s, n in zip(k.stride(), k.shape[:3]))
        _need(k.stride(3) == 1 and v.stride() == k.stride() and all(s % 16 == 0 and s >= dim for s in st)
              and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0,
              f"codes need contiguous D and equal strides that are multiples of 16 bytes, got {k.stride()} and {v.stride()}")
        for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _need(s.dtype == torch.float32 and tuple(s.shape) == (pages, heads) and s.stride(1) == 1 and s.stride(0) == k_scale.stride(0)
                  and s.stride(0) >= heads, f"{name} must be float32 ({pages}, {heads}) with contiguous rows, got {s.dtype} {tuple(s.shape)}")
        _need(all(t.device == k.device for t in (v, k_scale, v_scale)), "codes and scales must be on one device")
        _cuda(k.device)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.num_heads, self.page_size, self.head_dim = pages, heads, page, dim
        self.device = k.device
        self.status = torch.zeros(4, dtype=torch.int32, device=k.device) if status is None else status
        self._c = N.PagedPool(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), st[0], st[1], st[2],
                              k_scale.stride(0), pages, page, heads, dim, _STORES[k.dtype], self.status.data_ptr())
        self._ref = C.byref(self._c)
        self._ws: dict[tuple[int, int], int] = {}

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_heads: int, head_dim: int, *, storage: str = "e4m3",
                 device: torch.device | str = "cuda") -> PagedPool:
        """An empty pool; ``storage`` is ``"e4m3"`` or ``"int8"``."""
        if storage not in _NAMES:
            raise ValueError(f"storage must be 'e4m3' or 'int8', got {storage!r}")
        shape = (num_pages, num_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(_NAMES[storage]) for _ in "kv")
        ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in "kv")
        return cls(k, v, ks, vs)

    def heads(self, first: int, count: int) -> PagedPool:
        """KV heads ``[first, first + count)`` of the pool, over the same tensors."""
        _need(0 <= first and count >= 1 and first + count <= self.num_heads, f"heads [{first}, {first + count}) of {self.num_heads}")
        s = slice(first, first + count)
        return PagedPool(self.k[:, s], self.v[:, s], self.k_scale[:, s], self.v_scale[:, s], status=self.status)

    def workspace_bytes(self, dtype: int, num_q_heads: int) -> int:
        key = (dtype, num_q_heads)
        n = self._ws.get(key)
        if n is None:
            with torch.cuda.device(self.device):
                n = int(N.lib().kvd_paged_attention_workspace_bytes(self._ref, dtype, num_q_heads))
            if n == 0:
                raise N.KvdError(N.KVD_ERR_ARG, "kvd_paged_attention_workspace_bytes", N.lib().kvd_last_error().decode())
            self._ws[key] = n
        return n

    def check_status(self) -> None:
        """Raise if a call on this pool met bad slots, bad page ids or values
        that are not finite (synchronises)."""
        _call(self.device, N.lib().kvd_paged_check_status, "kvd_paged_check_status", self.status.data_ptr(), _stream(self.device.index))


class PagePlan(NamedTuple):
    """One step's indices, all int32 on the device."""

    lens: Tensor        # (batch,) cached + new tokens
    cu_new: Tensor      # (batch + 1,) first row of each request's new tokens
    slots: Tensor       # (capacity,) page * page_size + offset; -1 behind the last row
    positions: Tensor   # (capacity,) position of each row in its request; 0 behind the last
    free_count: Tensor  # (1,) pages left on the free stack


def build_page_tables(cached_lens: Tensor, new_lens: Tensor, table: Tensor, free_pages: Tensor, free_count: Tensor, *,
                      page_size: int, capacity: int, in_place: bool = False, status: Tensor | None = None) -> PagePlan:
    """Pages, slots and positions for ``new_lens[b]`` more tokens of each request.

    ``table`` ``(batch, max_pages)`` holds request b's ``cached_lens[b]``
    tokens in its first pages and gets the new pages' ids, taken from the top
    of the stack ``free_pages[:free_count]`` in request order.  ``capacity``
    rows of slots and positions are written.  ``in_place``: the new lengths and
    the free count overwrite ``cached_lens`` and ``free_count``.  If pages,
    columns or rows do not suffice, or a length is negative, nothing is
    allocated, every slot is -1, and ``status`` (int32, 4 words) says so; it says so
    too of a token whose page has no id in ``table``, which gets slot -1."""
    device = cached_lens.device
    batch = cached_lens.shape[0]
    _ints(cached_lens, (batch,), "cached_lens", device)
    _ints(new_lens, (batch,), "new_lens", device)
    _table(table, batch, device)
    _ints(free_pages, (free_pages.shape[0],), "free_pages", device)
    _ints(free_count, (1,), "free_count", device)
    if status is not None:
        _ints(status, (4,), "status", device)
    _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    _need(0 <= capacity <= _INT_MAX, f"capacity must be >= 0 and within 32 bits, got {capacity}")
    _need(not (in_place and batch and new_lens.data_ptr() == cached_lens.data_ptr()),
          "new_lens must have memory of their own: the lengths are overwritten in place")
    _cuda(device)
    # one allocation: slots and positions first, both on 16-byte borders
    cap = (capacity + 3) & ~3
    lib = N.lib()
    ws = lib.kvd_page_tables_workspace_bytes(batch, capacity)
    n = 2 * cap + 2 * batch + 2
    buf = torch.empty(n + ws // 4, dtype=torch.int32, device=device)
    slots, _, positions, _, cu, lens, left, _ = buf.split_with_sizes(
        (capacity, cap - capacity, capacity, cap - capacity, batch + 1, batch, 1, ws // 4))
    if in_place:
        lens, left = cached_lens, free_count
    _call(device, lib.kvd_page_tables, "kvd_page_tables", batch, table.shape[1], page_size, cached_lens.data_ptr(),
          new_lens.data_ptr(), table.data_ptr(), table.stride(0), free_pages.data_ptr(), free_pages.shape[0],
          free_count.data_ptr(), capacity, lens.data_ptr(), left.data_ptr(), cu.data_ptr(), slots.data_ptr(),
          positions.data_ptr(), None if status is None else status.data_ptr(), buf.data_ptr() + 4 * n if ws else None, ws,
          _stream(device.index))
    return PagePlan(lens, cu, slots, positions, left)


class PageTables:
    """Page tables of up to ``batch`` requests over ``num_pages`` pages, and
    the stack of free ones: all on the device.  One set serves every layer's
    pool.  Rows of idle requests have length 0."""

    def __init__(self, batch: int, max_pages: int, num_pages: int, page_size: int, device: torch.device | str = "cuda") -> None:
        _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        _need(batch >= 1 and max_pages >= 1 and num_pages >= 1, f"batch {batch}, {max_pages} pages a request, {num_pages} pages")
        device = torch.device(device)
        _cuda(device)
        self.batch, self.max_pages, self.num_pages, self.page_size = batch, max_pages, num_pages, page_size
        self.table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)  # page 0 on top
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(4, dtype=torch.int32, device=device)
        self.device = self.table.device

    def advance(self, new_lens: Tensor, capacity: int) -> PagePlan:
        """Room for ``new_lens[b]`` more tokens of each request (in place: the plan's
        ``lens`` and ``free_count`` are the tables' own, which later calls overwrite)."""
        return build_page_tables(self.lens, new_lens, self.table, self.free_pages, self.free_count, page_size=self.page_size,
                                 capacity=capacity, in_place=True, status=self.status)

    def release(self, done: Tensor) -> None:
        """Requests with ``done[b]`` (bool) give their pages back and are empty."""
        _need(done.dtype == torch.bool and tuple(done.shape) == (self.batch,) and done.is_contiguous() and done.device == self.device,
              f"done must be a contiguous bool tensor of shape ({self.batch},) on {self.device}, got {done.dtype} {tuple(done.shape)}")
        _call(self.device, N.lib().kvd_page_release, "kvd_page_release", self.batch, self.max_pages, self.page_size, done.data_ptr(),
              self.lens.data_ptr(), self.table.data_ptr(), self.table.stride(0), self.free_pages.data_ptr(), self.num_pages,
              self.free_count.data_ptr(), self.status.data_ptr(), _stream(self.device.index))

    def check_status(self) -> None:
        """Raise if a step did not fit (synchronises)."""
        _call(self.device, N.lib().kvd_paged_check_status, "kvd_paged_check_status", self.status.data_ptr(), _stream(self.device.index))


def paged_append(pool: PagedPool, slots: Tensor, k: Tensor, v: Tensor, *, max_new: int = 0) -> None:
    """Store keys and values ``(B, H, T, D)``, or packed ``(T, H, D)``, at
    ``slots`` (int32, one per row, batch-major).  Negative slots are skipped.
    Rows of one page must follow one another with consecutive slots, one run a call,
    as :func:`build_page_tables` gives them; rows that go back into the page of the row
    before (the same slot twice, a gap) are skipped and reported.  ``max_new``: the most
    rows of one packed request, if known; it only chooses the launch.

    A page's scale is the least power of two with ``|x| <= 448 s`` (e4m3) or
    ``127 s`` (int8); when later tokens need a larger one, the page's codes are
    rounded again (e4m3 loses nothing but subnormals by it).  Infinities are
    stored as the largest code, NaN as 0, and :meth:`PagedPool.check_status`
    raises for both."""
    _need(k.dim() in (3, 4) and k.shape == v.shape and k.dtype == v.dtype, f"k and v must be (B, H, T, D) or (T, H, D) alike, got "
          f"{k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    dtype = _dtype(k, "keys")
    batch, tokens, heads = (1, k.shape[0], k.shape[1]) if k.dim() == 3 else (k.shape[0], k.shape[2], k.shape[1])
    _need(heads == pool.num_heads and k.shape[-1] == pool.head_dim, f"pool holds {pool.num_heads} heads x {pool.head_dim}, got {tuple(k.shape)}")
    _need(k.device == pool.device and v.device == pool.device, f"k and v must be on {pool.device}")
    _ints(slots, (batch * tokens,), "slots", pool.device)
    _need(max_new >= 0, f"max_new must be >= 0, got {max_new}")
    _no_grad(k, v)
    most = min(max_new, _INT_MAX) if k.dim() == 3 else tokens
    k, k_view = _rows(k)  # the copies, if any, live until the call is made: the allocator orders their reuse by stream
    v, v_view = _rows(v)
    _call(pool.device, N.lib().kvd_paged_append_runs, "kvd_paged_append", pool._ref, slots.data_ptr(), batch, dtype, k_view, v_view, most,
          _stream(pool.device.index))


def paged_peek(pool: PagedPool, table: Tensor, lens: Tensor, tokens: int, *, dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """Dense keys and values ``(B, H, tokens, D)`` of each request's first
    ``tokens`` tokens, held to ``dtype``'s range (a code may round up past its
    largest value); zero from its length on."""
    code = _DTYPES.get(dtype)
    if code is None:
        raise NotImplementedError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    _table(table, None, pool.device)
    batch = table.shape[0]
    _ints(lens, (batch,), "lens", pool.device)
    _need(tokens >= 0, f"tokens must be >= 0, got {tokens}")
    kv = torch.empty((2, batch, pool.num_heads, tokens, pool.head_dim), dtype=dtype, device=pool.device)
    k, v = kv.unbind(0)
    if table.shape[1] == 0:
        kv.zero_()
        return k, v
    _call(pool.device, N.lib().kvd_paged_peek, "kvd_paged_peek", pool._ref, batch, table.data_ptr(), table.stride(0), table.shape[1],
          lens.data_ptr(), code, _rows(k)[1], _rows(v)[1], _stream(pool.device.index))
    return k, v


def paged_attention(pool: PagedPool, table: Tensor, lens: Tensor, q: Tensor, *, cu_q: Tensor | None = None, max_q: int = 0,
                    scaling: float | None = None, window: int = 0, starts: Tensor | None = None, return_lse: bool = False,
                    out: Tensor | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """Attention of queries over the requests' pages.

    ``q`` is ``(B, Hq, T, D)``, every request with T query tokens, or packed
    ``(rows, Hq, D)`` with ``cu_q`` ``(B + 1,)`` (int32).  A request's queries
    are its last tokens (its keys and values are stored already): query i of n
    sees tokens up to ``lens[b] - n + i``, from ``starts[b]`` on (left padding)
    and, with ``window > 0``, only the last ``window`` of them.  A query that
    sees nothing gives zeros.  ``max_q``: the most query tokens of one packed
    request, if known; it only chooses kernels.  ``scaling`` is positive, ``D ** -0.5``
    if not given.  Lengths beyond the table's columns end with them; ``cu_q``
    entries that are no offsets into the rows answer nothing.  The pages' codes are
    finite, as :func:`paged_append` writes them.  Sums are fp32: scores and values up to
    2^90 stay within it; the output is held to its type's range.

    Returns ``(B, T, Hq, D)``, or ``(rows, Hq, D)`` packed, in ``q``'s type
    (rows that no request answers are zero, or as they were in ``out``), and with
    ``return_lse`` the natural log of the softmax's sum, fp32, without the last
    dimension (-inf where a query saw nothing)."""
    dtype = _dtype(q, "queries")
    device, dim = pool.device, pool.head_dim
    _table(table, None, device)
    batch = table.shape[0]
    _ints(lens, (batch,), "lens", device)
    packed = cu_q is not None
    _need(q.dim() == (3 if packed else 4) and q.shape[-1] == dim, f"queries must be (B, Hq, T, {dim}), or (rows, Hq, {dim}) with cu_q, got {tuple(q.shape)}")
    hq = q.shape[1]
    _need(hq >= pool.num_heads and hq % pool.num_heads == 0, f"{hq} query heads over {pool.num_heads} KV heads")
    _need(q.device == device, f"queries are on {q.device}, the pool on {device}")
    _need(window >= 0 and max_q >= 0, f"window and max_q must be >= 0, got {window} and {max_q}")
    if packed:
        _ints(cu_q, (batch + 1,), "cu_q", device)  # type: ignore[arg-type]
        shape, tokens = (q.shape[0], hq, dim), q.shape[0]
    else:
        _need(q.shape[0] == batch, f"{q.shape[0]} requests' queries, {batch} rows of the table")
        shape, tokens = (batch, q.shape[2], hq, dim), q.shape[2]
    if starts is not None:
        _ints(starts, (batch,), "starts", device)
    _no_grad(q)
    q, view = _rows(q)
    lse = None
    fill = out is None  # rows that no request answers
    if out is None:
        out = torch.empty_like(q) if packed and q.is_contiguous() else q.new_empty(shape)
    else:
        _need(tuple(out.shape) == shape and out.dtype == q.dtype and out.device == device and out.is_contiguous() and out.data_ptr() % 16 == 0
              and out.untyped_storage().data_ptr() != q.untyped_storage().data_ptr(),
              f"out must be a contiguous {q.dtype} tensor of shape {shape} with memory of its own, got {out.dtype} {tuple(out.shape)}")
    if return_lse:
        lse = q.new_empty(shape[:-1], dtype=torch.float32)
        if packed and not fill:
            lse.fill_(-torch.inf)
    if batch == 0:
        if fill:
            out.zero_()
        if lse is not None:
            lse.fill_(-torch.inf)
        return out if lse is None else (out, lse)
    ws = torch.empty(pool.workspace_bytes(dtype, hq), dtype=torch.uint8, device=device)
    _call(device, N.lib().kvd_paged_attention, "kvd_paged_attention", pool._ref, batch, table.data_ptr(), table.stride(0), table.shape[1],
          lens.data_ptr(), None if starts is None else starts.data_ptr(), None if cu_q is None else cu_q.data_ptr(), dtype,
          view.ptr, view.stride_b, view.stride_h, view.stride_t, tokens, min(max_q, _INT_MAX), hq,
          dim**-0.5 if scaling is None else scaling, min(window, _INT_MAX),
          out.data_ptr(), None if lse is None else lse.data_ptr(), int(fill), ws.data_ptr(), ws.numel(), _stream(device.index))
    return out if lse is None else (out, lse)
