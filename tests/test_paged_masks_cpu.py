"""Attention masks in front of the 8-bit paged cache, on the CPU: the device calls
are stood in for by exact dense ones, so that a model's two ways through
``PagedKVCache`` (its own attention over the dense return, the registered function
over the pages) give the same logits, or the second refuses the mask."""

from __future__ import annotations

import pytest
import torch
from transformers import Gemma3ForCausalLM, Gemma3TextConfig, LlamaConfig, LlamaForCausalLM, MistralConfig, MistralForCausalLM

from kvdlra_b200 import PagedKVCache, enable_factored_decode, paged_cache
from kvdlra_b200.attention import factored_attention_forward
from kvdlra_b200.paged import PagePlan


class _Tables:
    def __init__(self, batch, max_pages, num_pages, page_size, device) -> None:
        self.batch, self.num_pages, self.device, self.table = batch, num_pages, device, None
        self.lens = torch.zeros(batch, dtype=torch.int32)

    def advance(self, new, capacity):
        self.lens += new
        return PagePlan(self.lens, None, torch.zeros(capacity), None, None)

    def release(self, done) -> None:
        self.lens.zero_()


class _Pool:
    page_size = 64

    @classmethod
    def allocate(cls, *args, **kw):
        return cls()

    def __init__(self) -> None:
        self.k = self.v = None
        self.status = torch.zeros(4, dtype=torch.int32)


def _append(pool, slots, k, v, **kw) -> None:
    assert slots.numel() == k.shape[0] * k.shape[2]
    pool.k, pool.v = (x if y is None else torch.cat([y, x], 2) for x, y in ((k, pool.k), (v, pool.v)))


def _peek(pool, table, lens, tokens, dtype):
    return pool.k[:, :, :tokens], pool.v[:, :, :tokens]


def _attention(pool, table, lens, q, *, scaling, window, starts):
    """Causal from the bottom right, a window, left padding: what the pages compute."""
    n, total = q.shape[2], int(lens[0])
    k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], 1) for x in (pool.k, pool.v))
    t, last = torch.arange(total), total - n + torch.arange(n)[:, None]
    seen = ((t <= last) & ((t > last - window) if window else True)).expand(q.shape[0], 1, n, total)
    if starts is not None:
        seen = seen & (t >= starts[:, None, None, None])
    x = (q @ k.transpose(2, 3) * scaling).masked_fill(~seen, -torch.inf)
    return (torch.nan_to_num(torch.softmax(x, 3)) @ v).transpose(1, 2)


@pytest.fixture(autouse=True)
def _stand_ins(monkeypatch) -> None:
    for name, fake in (("PageTables", _Tables), ("PagedPool", _Pool), ("paged_append", _append), ("paged_peek", _peek),
                       ("paged_attention", _attention)):
        monkeypatch.setattr(paged_cache, name, fake)


_SIZES = dict(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
              head_dim=16, max_position_embeddings=128)


def _model(kind):
    torch.manual_seed(0)
    if kind == "llama":
        return LlamaForCausalLM(LlamaConfig(**_SIZES)).eval()
    if kind == "mistral":
        return MistralForCausalLM(MistralConfig(sliding_window=8, **_SIZES)).eval()
    config = Gemma3TextConfig(sliding_window=8, layer_types=["sliding_attention", "full_attention", "sliding_attention"], **_SIZES)
    return Gemma3ForCausalLM(config).eval()


def _ids(batch, n, seed=1):
    return torch.randint(1, 64, (batch, n), generator=torch.Generator().manual_seed(seed))


def _run(model, pages, steps, pads=None):
    """Logits of each step through a fresh cache: (ids, kwargs) steps."""
    if pages:
        enable_factored_decode(model)
    else:
        model.set_attn_implementation("sdpa")
    cache = PagedKVCache(model, 100, left_padding=None if pads is None else torch.tensor(pads))
    with torch.no_grad():
        return [model(ids, past_key_values=cache, use_cache=True, **kw).logits for ids, kw in steps]


def _same(model, steps, pads=None) -> None:
    """fp32 through three layers, sums of at most 64 terms in other orders: 1e-4 of
    the largest logit is some 800 half steps."""
    want, got = (_run(model, pages, steps, pads) for pages in (False, True))
    at = 0
    for a, b in zip(want, got):
        n = a.shape[1]
        for r in range(a.shape[0]):
            skip = max(0, (0 if pads is None else pads[r]) - at)  # rows of padding mean nothing
            if skip < n:
                assert float((a[r, skip:] - b[r, skip:]).abs().max()) < 1e-4 * float(a.abs().max())
        at += n


@pytest.mark.parametrize("kind", ["llama", "mistral", "gemma3"])
@pytest.mark.parametrize("sizes", [(20, 1, 1, 5), (8, 1), (9, 1), (3, 30, 1)])
def test_prompts_longer_than_the_window(kind, sizes) -> None:
    steps = [(_ids(2, n, seed=i), {}) for i, n in enumerate(sizes)]
    _same(_model(kind), steps)


@pytest.mark.parametrize("kind", ["llama", "mistral", "gemma3"])
@pytest.mark.parametrize("pads", [[0, 3, 7], [12, 0, 19]])
def test_left_padded_batches(kind, pads) -> None:
    ids, at = _ids(3, 20), torch.arange(20)
    mask = (at[None] >= torch.tensor(pads)[:, None]).long()
    steps, total = [(ids, dict(attention_mask=mask))], mask
    for i, n in enumerate((1, 4, 1)):
        total = torch.cat([total, torch.ones(3, n, dtype=torch.long)], 1)
        steps.append((_ids(3, n, seed=5 + i), dict(attention_mask=total)))
    _same(_model(kind), steps, pads)


def _after_prompt(kind, n, more, **kw):
    """A prompt of n tokens, then `more` tokens under a mask, over the pages."""
    return lambda: _run(_model(kind), True, [(_ids(2, n), {}), (_ids(2, more, seed=2), kw)])


@pytest.mark.parametrize("kind", ["llama", "mistral", "gemma3"])
def test_hidden_tokens_are_refused_at_every_step(kind) -> None:
    for n, more in ((12, 5), (12, 1)):
        mask = torch.ones(2, n + more, dtype=torch.long)
        _after_prompt(kind, n, more, attention_mask=mask)()
        mask[1, n - 2] = 0
        with pytest.raises(ValueError, match="left_padding"):
            _after_prompt(kind, n, more, attention_mask=mask)()
    mask = torch.ones(2, 12, dtype=torch.long)
    mask[0, :2] = 0
    with pytest.raises(ValueError, match="left_padding"):
        _run(_model(kind), True, [(_ids(2, 12), dict(attention_mask=mask))])
    with pytest.raises(ValueError, match="left_padding"):  # padding of another length than the cache was told
        _run(_model(kind), True, [(_ids(2, 12), dict(attention_mask=mask))], pads=[3, 0])


def test_masks_of_four_dimensions() -> None:
    model, n = _model("llama"), 10
    causal = torch.ones(n, n, dtype=torch.bool).tril()[None, None]
    prefix, hole = causal.clone(), causal.clone()
    prefix[..., :4, :4] = True
    hole[..., 6, 3] = False
    low = torch.finfo(torch.float32).min

    def call(mask):
        return _run(model, True, [(_ids(2, n), dict(attention_mask=mask))])[0]

    plain = call(None)
    additive = torch.where(causal, 0.0, low)
    for mask in (causal, causal.expand(2, 1, n, n), additive, torch.where(causal, 0.0, -torch.inf)):
        assert torch.equal(call(mask), plain)
    bias = additive.clone()
    bias[..., 5, 2] = 0.5
    for mask in (prefix, hole, torch.where(prefix, 0.0, low), torch.where(hole, 0.0, low), bias):
        with pytest.raises(ValueError, match="attention mask"):
            call(mask)


def test_a_refused_step_leaves_a_cache_that_says_so() -> None:
    model = _model("llama")
    enable_factored_decode(model)
    cache = PagedKVCache(model, 100)
    mask = torch.ones(2, 6, dtype=torch.long)
    mask[1, 0] = 0
    with torch.no_grad():
        with pytest.raises(ValueError, match="left_padding"):
            model(_ids(2, 6), attention_mask=mask, past_key_values=cache, use_cache=True)
        with pytest.raises(RuntimeError, match="reset"):
            model(_ids(2, 1), past_key_values=cache, use_cache=True)
        cache.reset()
        for layer in cache.layers:
            if layer.pool is not None:
                layer.pool.k = layer.pool.v = None
        got = model(_ids(2, 6), past_key_values=cache, use_cache=True).logits
    assert torch.equal(got, _run(model, True, [(_ids(2, 6), {})])[0])


def test_attention_that_is_not_causal_is_refused() -> None:
    model = _model("llama")
    for layer in model.model.layers:
        layer.self_attn.is_causal = False
    with pytest.raises(NotImplementedError, match="causal"):
        _run(model, True, [(_ids(2, 6), {})])


def test_a_mask_is_read_once_a_step(monkeypatch) -> None:
    """Reading it waits for the device: once for each of the step's masks, not once
    a layer."""
    reads = []
    fits = paged_cache.PagedKVCache._mask_fits
    monkeypatch.setattr(paged_cache.PagedKVCache, "_mask_fits", lambda self, *a: reads.append(0) or fits(self, *a))
    for kind, most in (("llama", 1), ("gemma3", 2)):
        mask = torch.ones(2, 12, dtype=torch.long)
        mask[0, :2] = 0
        full = torch.cat([mask, torch.ones(2, 1, dtype=torch.long)], 1)
        reads.clear()
        _run(_model(kind), True, [(_ids(2, 12), dict(attention_mask=mask)), (_ids(2, 1), dict(attention_mask=full))], pads=[2, 0])
        assert len(reads) == 2 * most
        reads.clear()
        _run(_model(kind), True, [(_ids(2, 4), {}), (_ids(2, 1), {}), (_ids(2, 1), {})])
        assert not reads


@pytest.mark.parametrize("kw, what", [(dict(softcap=30.0), "softcap"), (dict(s_aux=torch.zeros(4)), "s_aux"), (dict(dropout=0.1), "dropout")])
def test_parts_of_attention_that_the_pages_lack_are_refused(kw, what) -> None:
    """Models pass them as keyword arguments; None stands for their absence."""
    model = _model("llama")
    enable_factored_decode(model)
    cache = PagedKVCache(model, 32)
    module = model.model.layers[0].self_attn
    q, k = torch.randn(2, 4, 3, 16), torch.randn(2, 2, 3, 16)
    key, value = cache.update(k, k, 0)
    with torch.no_grad():
        factored_attention_forward(module, q, key, value, None, scaling=0.25, softcap=None, s_aux=None)
        with pytest.raises(NotImplementedError, match=what):
            factored_attention_forward(module, q, key, value, None, scaling=0.25, **kw)
