"""A transformers cache over 8-bit pages: the full-length, exact-position
baseline beside :class:`kvdlra_b200.BugStreamingCache`.

It keeps every token of every sequence as 8-bit codes (:mod:`kvdlra_b200.paged`)
and takes the same calls: ``model(..., past_key_values=cache)``,
``model.generate``, ``harness.prefill_chunked`` and ``harness.decode_greedy``.
With :func:`kvdlra_b200.enable_factored_decode` the model's attention reads the
pages; without it ``update`` returns the dense keys and values, as any cache
does, and the model's own attention reads those.

All layers share one set of page tables and have a pool each.  A batch's rows
advance together, from their left padding on; batches of requests with lengths of
their own use :mod:`kvdlra_b200.paged` directly.
"""

from __future__ import annotations

from contextlib import contextmanager
from typing import Any, Iterator

import torch
from torch import Tensor
from transformers.cache_utils import Cache, CacheLayerMixin

from .attention import tag_step, uses_factored_decode
from .paged import PAGE_SIZES, PagedPool, PagePlan, PageTables, paged_append, paged_attention, paged_peek

__all__ = ["PagedKVCache", "PagedKVLayer"]

_MARK = "_kvdlra_checked"


class PagedKVLayer(CacheLayerMixin):  # type: ignore[misc]
    """One layer's pages."""

    is_sliding = False
    is_compileable = False

    def __init__(self, owner: PagedKVCache, index: int) -> None:
        super().__init__()
        self._owner, self._index = owner, index
        self.pool: PagedPool | None = None
        self.cumulative_length = 0
        self._parts: dict[tuple[int, int], PagedPool] = {}

    def lazy_initialization(self, key_states: Tensor, value_states: Tensor) -> None:
        batch, heads, _, dim = key_states.shape
        self._owner._tables_for(batch, key_states.device)
        assert self._owner.tables is not None
        self.dtype, self.device = key_states.dtype, key_states.device
        self.pool = PagedPool.allocate(self._owner.tables.num_pages, self._owner.page_size, heads, dim, storage=self._owner.storage,
                                       device=key_states.device)
        self.is_initialized = True

    def update(self, key_states: Tensor, value_states: Tensor, *args: object, **kwargs: object) -> tuple[Tensor, Tensor]:
        """Store the step's keys and values ``(B, H, q, D)``; returns the dense
        keys and values of all tokens, or the step's own, tagged with the layer,
        for a model whose attention reads the pages."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        assert self.pool is not None
        if key_states.dtype != self.dtype:
            raise ValueError(f"cache dtype is {self.dtype}, got {key_states.dtype}")
        plan = self._owner._step(self.cumulative_length, int(key_states.shape[0]), int(key_states.shape[2]))
        paged_append(self.pool, plan.slots, key_states, value_states)
        self.cumulative_length += int(key_states.shape[2])
        if self._owner._reads_pages():
            return tag_step(key_states.view(key_states.shape), self), value_states
        tables = self._owner.tables
        assert tables is not None
        return paged_peek(self.pool, tables.table, plan.lens, self.cumulative_length, dtype=self.dtype)

    def paged_attention(self, query: Tensor, *, scaling: float | None = None, heads: tuple[int, int] | None = None,
                        window: int = 0) -> Tensor:
        """Attention of the step's queries ``(B, Hq, q, D)`` over the pages;
        ``(B, q, Hq, D)``.  ``heads``: the KV heads that the queries belong to."""
        tables, pool = self._owner.tables, self.pool
        assert tables is not None and pool is not None
        if heads is not None:
            if heads not in self._parts:
                self._parts[heads] = pool.heads(*heads)
            pool = self._parts[heads]
        out = paged_attention(pool, tables.table, tables.lens, query, scaling=scaling, window=window, starts=self._owner.starts)
        assert isinstance(out, Tensor)
        return out

    def check_mask(self, mask: Tensor | None, query: Tensor, *, window: int = 0, causal: bool = True) -> None:
        """Refuse a mask that says anything but what the pages' attention computes:
        causal over the cache's tokens, ``window``, the cache's left padding.  Reading
        it synchronises: a step's mask is marked once it was read.  Under capture it
        is compared on the device, and :meth:`PagedKVCache.check_status` raises."""
        owner = self._owner
        if mask is None:
            if not causal and query.shape[2] > 1:
                raise NotImplementedError("attention over the pages is causal")
            return
        step, seen = getattr(mask, _MARK, (None, None))
        if step is owner._step_mark and seen == window:
            return
        fits = owner._mask_fits(mask, int(query.shape[2]), self.cumulative_length, window)
        if mask.is_cuda and torch.cuda.is_current_stream_capturing():
            assert self.pool is not None
            self.pool.status[1:2].bitwise_or_((~fits).to(torch.int32) * 8)
        elif not bool(fits):
            owner._refused = True
            raise ValueError("the attention mask is not the causal one of the cache's tokens: hidden tokens at the front of a row are "
                             "the cache's left_padding (tokens per row), others are not supported; reset() the cache")
        setattr(mask, _MARK, (owner._step_mark, window))

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        if isinstance(query_length, Tensor):  # tolerate cache_position tensors
            query_length = int(query_length.shape[0])
        return self.cumulative_length + query_length, 0

    def get_seq_length(self) -> int:
        return self.cumulative_length

    def get_max_cache_shape(self) -> int:
        return self._owner.max_tokens

    def reset(self) -> None:
        self.cumulative_length = 0

    def reorder_cache(self, beam_idx: Tensor) -> None:
        raise NotImplementedError("PagedKVCache does not reorder its rows (no beam search)")

    def crop(self, max_length: int) -> None:
        raise NotImplementedError("PagedKVCache does not give back single tokens; reset() empties it")

    def batch_repeat_interleave(self, repeats: int) -> None:
        raise NotImplementedError("PagedKVCache does not repeat its rows")

    def stored_state_numel(self) -> int:
        """The layer's stored floats, in the reference's float-equivalent unit of
        16 bits: two codes to one, a scale two."""
        if self.pool is None or self.cumulative_length == 0:
            return 0
        tables, pool = self._owner.tables, self.pool
        assert tables is not None
        pages = tables.batch * -(-self.cumulative_length // pool.page_size)
        return pages * pool.num_heads * (pool.page_size * pool.head_dim + 2 * 2)


class PagedKVCache(Cache):
    """Every token in 8-bit pages, ``max_tokens`` a row at most.

    ``storage``: ``"e4m3"`` or ``"int8"``.  ``left_padding``: int tensor
    ``(batch,)``, tokens at the front of each row that are padding."""

    def __init__(self, model: Any, max_tokens: int, *, page_size: int = 64, storage: str = "e4m3",
                 left_padding: Tensor | None = None, num_layers: int | None = None) -> None:
        if max_tokens < 1:
            raise ValueError(f"max_tokens must be >= 1, got {max_tokens}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if storage not in ("e4m3", "int8"):
            raise ValueError(f"storage must be 'e4m3' or 'int8', got {storage!r}")
        if left_padding is not None and (left_padding.dim() != 1 or left_padding.dtype.is_floating_point or bool((left_padding < 0).any())):
            raise ValueError("left_padding must be a 1-d tensor of whole numbers >= 0")
        if num_layers is None:
            num_layers = int(model.config.num_hidden_layers)
        self._model_config = getattr(model, "config", None)
        self.max_tokens, self.page_size, self.storage = max_tokens, page_size, storage
        self._left_padding = left_padding
        self.starts: Tensor | None = None
        self.tables: PageTables | None = None
        self._plan: PagePlan | None = None
        self._at: tuple[int, int] | None = None
        self._step_mark, self._refused = object(), False
        super().__init__(layers=[PagedKVLayer(self, i) for i in range(num_layers)])

    def _reads_pages(self) -> bool:
        return uses_factored_decode(self._model_config)

    def _tables_for(self, batch: int, device: torch.device) -> None:
        if self.tables is None:
            if self._left_padding is not None:
                if self._left_padding.shape[0] != batch:
                    raise ValueError(f"left_padding is for {self._left_padding.shape[0]} rows, the batch has {batch}")
                self.starts = self._left_padding.to(device=device, dtype=torch.int32).contiguous()
            width = -(-self.max_tokens // self.page_size)
            self.tables = PageTables(batch, width, batch * width, self.page_size, device)
        elif self.tables.batch != batch:
            raise NotImplementedError(f"PagedKVCache was initialised for batch size {self.tables.batch}, got {batch}")

    def _step(self, length: int, batch: int, tokens: int) -> PagePlan:
        """The step's tables: made by its first layer, used by all."""
        tables = self.tables
        assert tables is not None
        if batch != tables.batch:
            raise NotImplementedError(f"PagedKVCache was initialised for batch size {tables.batch}, got {batch}")
        if self._refused:
            raise RuntimeError("a step of this cache was refused half way: reset() it")
        if self._at != (length, tokens):
            if self._at is not None and length != sum(self._at):
                raise RuntimeError(f"a layer holds {length} tokens, the cache {sum(self._at)}: its layers advance together")
            if length + tokens > self.max_tokens:
                raise ValueError(f"{length + tokens} tokens in a cache for {self.max_tokens}")
            new = torch.full((batch,), tokens, dtype=torch.int32, device=tables.device)  # not kept: a captured step's belongs to its graph
            self._plan = tables.advance(new, batch * tokens)
            self._at = (length, tokens)
            self._step_mark = object()
        assert self._plan is not None
        return self._plan

    def _mask_fits(self, mask: Tensor, tokens: int, length: int, window: int) -> Tensor:
        """Whether a mask ``(1 or B, 1 or heads, tokens, length)``, of truth values or
        to be added, is the pages' own (a truth value on its device).  Rows of padding
        queries, which mean nothing, may say anything."""
        if mask.dim() != 4 or tuple(mask.shape[2:]) != (tokens, length):
            return torch.zeros((), dtype=torch.bool, device=mask.device)
        t, last = torch.arange(length, device=mask.device), torch.arange(length - tokens, length, device=mask.device)[:, None]
        seen = t <= last
        if window:
            seen &= t > last - window
        if self.starts is not None:
            starts = self.starts.to(mask.device)[:, None, None, None]
            seen = seen & (t >= starts)
        # to be added: 0, or so low that nothing is left of the token's weight
        fits = mask == seen if mask.dtype == torch.bool else torch.where(seen, mask == 0, mask <= -1e4)
        if self.starts is not None:
            fits = fits | (last < starts)
        return fits.all()

    @contextmanager
    def ingesting(self) -> Iterator[None]:
        """Chunked pre-fill, as the harness calls it: chunks need no mode here."""
        yield

    def consolidate(self) -> None:
        """Nothing is deferred: a chunk is stored when ``update`` returns."""

    def reset(self) -> None:
        """Empty every layer (the pages stay allocated for reuse)."""
        if self.tables is not None:
            self.tables.release(torch.ones(self.tables.batch, dtype=torch.bool, device=self.tables.device))
        self._plan = self._at = None
        self._refused = False
        for layer in self.layers:
            layer.reset()

    def stored_state_numel(self) -> int:
        return sum(layer.stored_state_numel() for layer in self.layers)

    def check_status(self) -> None:
        """Raise if a kernel met bad indices or values that are not finite
        (synchronises)."""
        if self.tables is not None:
            self.tables.check_status()
        for layer in self.layers:
            if layer.pool is not None:
                layer.pool.check_status()
