"""The transformers cache over 8-bit pages behind a random-init Llama: the
harness's chunked prefill and greedy decode, ``model.generate``, padded batches.

The pages hold rounded keys and values, so a run is compared with another that
reads the same pages: the paged attention against the model's own attention over
the dense return of ``update``.  Both read the same numbers; what differs is the
order of sums and the rounding of the attention's output to the model's type, half
a step each, through a few layers: 2e-3 of the largest logit in fp32 and 2e-2 in
bf16, as for the compressed cache."""

from __future__ import annotations

import pytest
import torch

from golden.make_golden import MODEL_CASE, tiny_llama

from kvdlra_b200 import PagedKVCache, enable_factored_decode
from kvdlra_b200.harness import decode_greedy, prefill_chunked
from kvdlra_b200.paged_cache import PagedKVLayer

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _model(dtype):
    torch.manual_seed(0)
    return tiny_llama(MODEL_CASE).to(DEV, dtype)


def _ids(model, batch, tokens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(1, model.config.vocab_size, (batch, tokens), generator=g).to(DEV)


@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-3), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("storage, page_size", [("e4m3", 16), ("int8", 64)])
def test_harness_runs_on_the_pages(dtype, tol, storage, page_size, monkeypatch) -> None:
    model = _model(dtype)
    ids = _ids(model, 2, 150)
    forced = _ids(model, 2, 9, seed=2)
    calls = []
    fn = PagedKVLayer.paged_attention
    monkeypatch.setattr(PagedKVLayer, "paged_attention", lambda self, *a, **k: calls.append(0) or fn(self, *a, **k))
    runs = {}
    for mode in ("sdpa", "paged"):
        if mode == "paged":
            enable_factored_decode(model)
        else:
            model.set_attn_implementation("sdpa")
        cache = PagedKVCache(model, 170, page_size=page_size, storage=storage)
        first = prefill_chunked(model, cache, ids, 64, keep_logits=True)
        _, logits = decode_greedy(model, cache, first, 150, 9, forced=forced)
        runs[mode] = torch.cat([first[:, None], logits], 1).double()
        assert cache.get_seq_length() == 159
        assert calls == [] if mode == "sdpa" else len(calls) == (3 + 9) * model.config.num_hidden_layers
        layer = cache.layers[0]
        d = layer.pool.head_dim
        assert layer.stored_state_numel() == 2 * -(-159 // page_size) * layer.pool.num_heads * (page_size * d + 4)
        cache.check_status()
        cache.reset()
        assert cache.get_seq_length() == 0 and cache.tables.free_count.item() == cache.tables.num_pages
        again = prefill_chunked(model, cache, ids, 64, keep_logits=True)
        assert torch.equal(again, first)
    err = float((runs["paged"] - runs["sdpa"]).abs().max() / runs["sdpa"].abs().max())
    assert err < tol, err


def test_codes_stay_near_the_exact_cache() -> None:
    """int8 pages against transformers' own cache: the keys' and values' step is
    2^-7 of a page's largest, which moves the logits by a few percent at most."""
    model = _model(torch.float32)
    enable_factored_decode(model)
    ids = _ids(model, 1, 100)
    with torch.no_grad():
        exact = model(ids, use_cache=True).logits[:, -1]
        cache = PagedKVCache(model, 128, page_size=16, storage="int8")
        got = prefill_chunked(model, cache, ids, 40, keep_logits=True)
    assert float((got - exact).abs().max() / exact.abs().max()) < 0.1


def test_generate() -> None:
    model = _model(torch.bfloat16)
    enable_factored_decode(model)
    ids = _ids(model, 2, 33)
    cache = PagedKVCache(model, 64)
    out = model.generate(ids, past_key_values=cache, max_new_tokens=12, do_sample=False, attention_mask=torch.ones_like(ids))
    assert out.shape == (2, 45) and cache.get_seq_length() == 44
    cache.check_status()


def test_left_padded_rows_equal_their_unpadded_runs() -> None:
    """A padded batch with ``left_padding``, against each row alone; without it the
    batch is refused."""
    model = _model(torch.float32)
    enable_factored_decode(model)
    pads = [0, 7, 20]
    ids = _ids(model, 3, 40)
    mask = torch.ones_like(ids)
    for b, p in enumerate(pads):
        mask[b, :p] = 0
    pos = (mask.cumsum(1) - 1).clamp(min=0)
    with torch.no_grad():
        cache = PagedKVCache(model, 64, page_size=16, storage="int8", left_padding=torch.tensor(pads))
        got = model(ids, attention_mask=mask, position_ids=pos, past_key_values=cache, use_cache=True).logits[:, -1]
        nxt = _ids(model, 3, 1, seed=3)
        step = model(nxt, attention_mask=torch.cat([mask, mask[:, -1:]], 1), position_ids=pos[:, -1:] + 1, past_key_values=cache,
                     use_cache=True).logits[:, -1]
        for b, p in enumerate(pads):
            one = PagedKVCache(model, 64, page_size=16, storage="int8")
            # pages that begin elsewhere have other scales: compare within the codes' step
            want = model(ids[b : b + 1, p:], past_key_values=one, use_cache=True).logits[:, -1]
            assert float((got[b] - want[0]).abs().max() / want.abs().max()) < 0.1
            want = model(nxt[b : b + 1], position_ids=pos[b : b + 1, -1:] + 1, past_key_values=one, use_cache=True).logits[:, -1]
            assert float((step[b] - want[0]).abs().max() / want.abs().max()) < 0.1
        with pytest.raises(ValueError, match="left_padding"):
            model(ids, attention_mask=mask, position_ids=pos, past_key_values=PagedKVCache(model, 64), use_cache=True)


def test_refusals() -> None:
    model = _model(torch.float32)
    enable_factored_decode(model)
    ids = _ids(model, 2, 20)
    cache = PagedKVCache(model, 24, page_size=16)
    with torch.no_grad():
        model(ids, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="in a cache for 24"):
            model(ids[:, :5], past_key_values=cache, use_cache=True)
        with pytest.raises(NotImplementedError, match="batch size"):
            model(ids[:1, :1], past_key_values=cache, use_cache=True)
    for call in (lambda: cache.crop(3), lambda: cache.reorder_cache(torch.tensor([1, 0])), lambda: cache.batch_repeat_interleave(2)):
        with pytest.raises(NotImplementedError):
            call()
