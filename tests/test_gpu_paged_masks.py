"""Models with sliding windows, padded batches and captured steps on
``PagedKVCache``: attention over the pages against the model's own attention over
the dense return, as in ``test_gpu_paged_cache`` (both read the same numbers: 2e-3
of the largest logit in fp32)."""

from __future__ import annotations

import pytest
import torch
from test_paged_masks_cpu import _SIZES

from transformers import Gemma3ForCausalLM, Gemma3TextConfig, LlamaConfig, LlamaForCausalLM, MistralConfig, MistralForCausalLM

from kvdlra_b200 import PagedKVCache, enable_factored_decode
from kvdlra_b200.harness import prefill_chunked

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
_HEADS = {**_SIZES, "head_dim": 64}


def _model(kind, dtype=torch.float32):
    torch.manual_seed(0)
    if kind == "llama":
        m = LlamaForCausalLM(LlamaConfig(**_HEADS))
    elif kind == "mistral":
        m = MistralForCausalLM(MistralConfig(sliding_window=16, **_HEADS))
    else:
        m = Gemma3ForCausalLM(Gemma3TextConfig(sliding_window=16, layer_types=["sliding_attention", "full_attention", "sliding_attention"],
                                               **_HEADS))
    return m.eval().to(DEV, dtype)


def _ids(batch, n, seed=1):
    return torch.randint(1, 64, (batch, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("kind", ["mistral", "gemma3"])
@pytest.mark.parametrize("pads", [None, [0, 5, 30]])
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-3), (torch.bfloat16, 2e-2)])
def test_sliding_windows(kind, pads, dtype, tol) -> None:
    model, n = _model(kind, dtype), 40
    ids = _ids(3, n)
    mask = torch.ones_like(ids)
    for b, p in enumerate(pads or []):
        mask[b, :p] = 0
    runs = []
    for pages in (False, True):
        if pages:
            enable_factored_decode(model)
        else:
            model.set_attn_implementation("sdpa")
        cache = PagedKVCache(model, 64, page_size=16, storage="int8", left_padding=None if pads is None else torch.tensor(pads))
        total, out = mask, []
        with torch.no_grad():
            for i, m in enumerate((n, 1, 6, 1)):
                if i:
                    total = torch.cat([total, total.new_ones(3, m)], 1)
                x = model(ids if i == 0 else _ids(3, m, seed=7 + i), attention_mask=None if pads is None else total, past_key_values=cache,
                          use_cache=True).logits
                keep = torch.ones(3, m, dtype=torch.bool, device=DEV) if i else mask.bool()
                out.append(x[keep].double())
        cache.check_status()
        runs.append(torch.cat(out))
    assert float((runs[0] - runs[1]).abs().max() / runs[0].abs().max()) < tol


def test_chunked_prompts_longer_than_the_window() -> None:
    model, ids = _model("mistral"), _ids(2, 60)
    got = []
    for pages in (False, True):
        if pages:
            enable_factored_decode(model)
        cache = PagedKVCache(model, 64, page_size=16, storage="int8")
        got.append(prefill_chunked(model, cache, ids, 25, keep_logits=True).double())
        cache.check_status()
    assert float((got[0] - got[1]).abs().max() / got[0].abs().max()) < 2e-3


def test_a_captured_step_compares_its_mask_on_the_device() -> None:
    """The step's graph takes the mask that the model builds in it; one that hides a
    token shows in the status."""
    model, n = _model("llama"), 20
    enable_factored_decode(model)
    ids, nxt = _ids(2, n), _ids(2, 1, seed=3)
    mask, pos = torch.ones(2, n + 1, dtype=torch.long, device=DEV), torch.full((2, 1), n, device=DEV)
    with torch.no_grad():
        cache = PagedKVCache(model, 64, page_size=16)
        model(ids, past_key_values=cache, use_cache=True)
        want = model(nxt, past_key_values=cache, use_cache=True, position_ids=pos).logits
        cache.reset()
        model(ids, past_key_values=cache, use_cache=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = model(nxt, past_key_values=cache, use_cache=True, attention_mask=mask, position_ids=pos).logits
        graph.replay()
        torch.cuda.synchronize()
        assert float((got - want).abs().max()) <= 1e-3 * float(want.abs().max())
        cache.check_status()
        mask[1, 4] = 0
        graph.replay()
        with pytest.raises(RuntimeError, match="bad indices"):
            cache.check_status()
