"""The 8-bit paged KV cache's operators, as a serving program calls them.

* ``tables``: page tables, slot map and positions of one step, from the
  requests' cached and new token counts.
* ``update``: the step's keys and values written into 8-bit pages with a scale
  for each (page, KV head), then read back dense, as a cache's ``update`` does
  for a model whose attention reads dense keys and values.
* ``attend``: attention over the pages, for single tokens, a few tokens and
  chunks, with ragged requests.

``own`` chooses between the plain torch form and ``kvdlra_b200.paged``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_TOP = {"e4m3": 448.0, "int8": 127.0}
_FLOOR = -100  # least exponent of a scale


# ------------------------------------------------------------------- cases


def listed():
    return [
        # one decode step of a few requests: a launch's latency
        dict(name="tables-decode-8", op="tables", batch=8, cached_lo=900, cached_hi=8200, new_lo=1, new_hi=1, page=16, pad=0),
        # a scheduler's largest step: a thousand requests, some idle, some with prompts, into a padded slot map
        dict(name="tables-mixed-1024", op="tables", batch=1024, cached_lo=0, cached_hi=6000, new_lo=0, new_hi=2047, page=32, pad=777),
        # a decode step of a batch on an SDPA model, Llama-3.2-1B heads
        dict(name="update-decode-32", op="update", batch=32, cached=511, new=1, heads=8, dim=64, page=16, store="e4m3", dtype="bf16"),
        # an ingest chunk of 512 tokens at the end of 8192, Llama-3.2-1B heads
        dict(name="update-chunk-512", op="update", batch=1, cached=7680, new=512, heads=8, dim=64, page=16, store="int8", dtype="bf16"),
        # prompts of four requests at once, an odd length, Llama-3.1-8B heads
        dict(name="update-prompt-4x8191", op="update", batch=4, cached=0, new=8191, heads=8, dim=128, page=128, store="e4m3", dtype="fp16"),
        # decode of one sequence, Llama-3.2-1B heads
        dict(name="attend-decode-1x8191", op="attend", batch=1, kv_lo=8191, kv_hi=8191, q_lo=1, q_hi=1, heads_q=32, heads=8, dim=64,
             page=16, store="e4m3", dtype="bf16", window=0),
        # decode of a ragged batch, Llama-3.1-8B heads
        dict(name="attend-decode-64-ragged", op="attend", batch=64, kv_lo=1, kv_hi=32768, q_lo=1, q_hi=1, heads_q=32, heads=8, dim=128,
             page=64, store="int8", dtype="bf16", window=0),
        # decode of one very long sequence: the split over the tokens
        dict(name="attend-decode-1x131072", op="attend", batch=1, kv_lo=131072, kv_hi=131072, q_lo=1, q_hi=1, heads_q=32, heads=8, dim=128,
             page=128, store="e4m3", dtype="fp16", window=0),
        # a few drafted tokens a request, checked at once
        dict(name="attend-draft-96x4", op="attend", batch=96, kv_lo=100, kv_hi=4099, q_lo=4, q_hi=4, heads_q=32, heads=4, dim=128,
             page=32, store="e4m3", dtype="bf16", window=0),
        # an ingest chunk of 512 tokens at the end of 8192, Llama-3.2-1B heads
        dict(name="attend-chunk-512-of-8192", op="attend", batch=1, kv_lo=8192, kv_hi=8192, q_lo=512, q_hi=512, heads_q=32, heads=8, dim=64,
             page=16, store="e4m3", dtype="bf16", window=0),
        # an ingest chunk of 2048 tokens of a long prompt, Llama-3.1-8B heads
        dict(name="attend-chunk-2048-of-32768", op="attend", batch=1, kv_lo=32768, kv_hi=32768, q_lo=2048, q_hi=2048, heads_q=32, heads=8,
             dim=128, page=64, store="int8", dtype="bf16", window=0),
        # decodes and chunks in one batch, a sliding window, one query head a KV head, full precision
        dict(name="attend-mixed-24-window", op="attend", batch=24, kv_lo=16, kv_hi=6001, q_lo=1, q_hi=257, heads_q=8, heads=8, dim=64,
             page=16, store="int8", dtype="fp32", window=1000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tables", "update", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "tables":
        batch = _log(rng, 1, 1024)
        new_hi = rng.choice([1, 1, _log(rng, 2, 2047)])
        return dict(op=op, batch=batch, cached_lo=0, cached_hi=_log(rng, 1, 8200), new_lo=min(new_hi, rng.randint(0, 1)), new_hi=new_hi, page=page,
                    pad=rng.randint(0, 999))
    store, dim = rng.choice(["e4m3", "int8"]), rng.choice([32, 64, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "update":
        heads = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 32)
        most = 32764 * 8 * 128 // (batch * heads * dim)  # no more than the largest listed one
        total = _log(rng, 2, max(2, min(20000, most)))
        new = min(total, rng.choice([1, _log(rng, 1, total), total]))
        return dict(op=op, batch=batch, cached=total - new, new=new, heads=heads, dim=dim, page=page, store=store, dtype=dtype)
    heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    if rng.random() < 0.5:  # single tokens, or a few
        batch, q_hi = _log(rng, 1, 64), rng.choice([1, 1, 2, 5])
        kv_hi = min(_log(rng, 16, 32768), (1 << 20) // batch)
        q_lo, kv_lo = rng.randint(1, q_hi), rng.randint(1, kv_hi)
    else:  # chunks
        batch, q_hi = _log(rng, 1, 6), _log(rng, 6, 1024)
        kv_hi = q_hi + _log(rng, 1, 8192 // batch)
        q_lo, kv_lo = rng.randint(0, q_hi), rng.randint(1, kv_hi)
    if dtype == "fp32" or dim in (32, 256):  # forms away from the served models' run at ordinary lengths
        kv_hi = min(kv_hi, 8192)
        kv_lo = min(kv_lo, kv_hi)
    return dict(op=op, batch=batch, kv_lo=kv_lo, kv_hi=kv_hi, q_lo=q_lo, q_hi=q_hi, heads_q=heads * group, heads=heads, dim=dim, page=page,
                store=store, dtype=dtype, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))


def _spread(lo, hi, n, turn):
    """n lengths over [lo, hi], the same ones for every seed; the first is the largest."""
    return [hi - int((hi - lo + 1) * ((b * turn) % 1.0)) if hi > lo else hi for b in range(n)]


def _lens(case):
    kv = _spread(case["kv_lo"], case["kv_hi"], case["batch"], 0.6180339887)
    q = _spread(case["q_lo"], case["q_hi"], case["batch"], 0.7548776662)
    return kv, q


def _plan_lens(case):
    cached = _spread(case["cached_lo"], case["cached_hi"], case["batch"], 0.6180339887)
    new = _spread(case["new_lo"], case["new_hi"], case["batch"], 0.7548776662)
    return cached, new


# ----------------------------------------------------------------- prepare


def _keys(g, n, heads, dim, dtype):
    """Key- or value-like rows (n, heads, dim): normal, a few strong channels, rows of different size."""
    x = torch.randn(n, heads, dim, generator=g, device="cuda")
    chan = 1.0 + 7.0 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.04)
    row = torch.exp(0.4 * torch.randn(n, 1, 1, generator=g, device="cuda"))
    return (x * chan * row).to(dtype)


def _filled(g, pages, heads, page, dim, store):
    """Pages that hold quantised rows already: codes and power-of-two scales."""
    x = _keys(g, pages * page, heads, dim, torch.float32).view(pages, page, heads, dim).transpose(1, 2).contiguous()
    s = _scale(x.abs().amax((2, 3)), store)
    return _codes(x, s[:, :, None, None], store), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    page = case["page"]
    if case["op"] == "tables":
        cached, new = _plan_lens(case)
        held = [-(-c // page) for c in cached]
        need = sum(-(-(c + t) // page) - h for c, t, h in zip(cached, new, held))
        pages = sum(held) + need + 5
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        width = max(-(-(c + t) // page) for c, t in zip(cached, new)) + 1
        table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
        col = torch.arange(width, device="cuda")[None]
        h = torch.tensor(held, device="cuda")[:, None]
        table[col < h] = order[: sum(held)]
        return dict(case=case, table=table, free=order[sum(held):].contiguous(),
                    count=torch.tensor([pages - sum(held)], dtype=torch.int32, device="cuda"),
                    cached=torch.tensor(cached, dtype=torch.int32, device="cuda"), new=torch.tensor(new, dtype=torch.int32, device="cuda"),
                    capacity=sum(new) + case["pad"])
    heads, dim, store = case["heads"], case["dim"], case["store"]
    dtype = _DTYPE[case["dtype"]]
    if case["op"] == "update":
        lens = [case["cached"] + case["new"]] * case["batch"]
    else:
        lens = _lens(case)[0]
    width = max(1, max(-(-n // page) for n in lens))
    pages = sum(-(-n // page) for n in lens) + 2
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    held = torch.tensor([-(-n // page) for n in lens], device="cuda")[:, None]
    table = torch.zeros(case["batch"], width, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None] < held] = order[: int(held.sum())]
    k, ks = _filled(g, pages, heads, page, dim, store)
    v, vs = _filled(g, pages, heads, page, dim, store)
    s = dict(case=case, table=table, k=k, v=v, ks=ks, vs=vs, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["op"] == "update":
        n, c = case["new"], case["cached"]
        pos = c + torch.arange(n, device="cuda")
        s["slots"] = (table[:, pos // page] * page + pos % page).reshape(-1).to(torch.int32)
        s["tokens"] = c + n
        s["new_k"], s["new_v"] = (_keys(g, case["batch"] * n, heads, dim, dtype).view(case["batch"], n, heads, dim).transpose(1, 2) for _ in "kv")
        return s
    q = _lens(case)[1]
    s["cu"] = torch.tensor([0] + list(np.cumsum(q)), dtype=torch.int32, device="cuda")
    s["q_most"], s["kv_most"] = max(q), max(lens)
    s["q"] = torch.randn(sum(q), case["heads_q"], dim, generator=g, device="cuda").to(dtype)
    s["scaling"] = dim**-0.5
    return s


# -------------------------------------------------------------- plain forms


def _power(e):
    """2^e in 32 bits, for -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale(amax, store):
    """The least power of two s with amax <= top * s (no less than 2^-100)."""
    m, e = torch.frexp(amax / _TOP[store])  # m 2^e with m in [1/2, 1); the quotient's rounding is put right below
    e = torch.where(amax > 0, e - (m == 0.5).to(e.dtype), _FLOOR).clamp(min=_FLOOR)
    return _power(torch.where(amax > _TOP[store] * _power(e), e + 1, e))


def _codes(x, s, store):
    y = (x / s).clamp(-_TOP[store], _TOP[store])
    return y.round().to(torch.int8) if store == "int8" else y.to(torch.float8_e4m3fn)


def _take(codes, at):
    return codes.view(torch.uint8)[at].view(codes.dtype).float()


def _plain_tables(s):
    page, table = s["case"]["page"], s["table"]
    cached, new = s["cached"].long(), s["new"].long()
    total = cached + new
    have, need = (cached + page - 1) // page, (total + page - 1) // page
    cu = torch.zeros(cached.numel() + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new.cumsum(0)
    first = (need - have).cumsum(0) - (need - have)  # new pages of the requests before
    col = torch.arange(table.shape[1], device="cuda")[None]
    at = (s["count"].long() - 1 - first[:, None] - (col - have[:, None])).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where((col >= have[:, None]) & (col < need[:, None]), s["free"][at], table))
    i = torch.arange(s["capacity"], device="cuda")
    b = (torch.searchsorted(cu, i, right=True) - 1).clamp(max=cached.numel() - 1)
    live = i < cu[-1]
    pos = torch.where(live, cached[b] + i - cu[b], 0)
    slot = torch.where(live, table[b, pos // page].long() * page + pos % page, -1)
    return dict(table=table, lens=total.int(), cu=cu.int(), slots=slot.int(), positions=pos.int(), count=(s["count"] - (need - have).sum()).int())


def _plain_append(codes, scale, x, slots, case):
    """x (B, H, n, D) into the pages at slots (B * n,), in place."""
    page, store = case["page"], case["store"]
    pages, heads = scale.shape
    rows = x.transpose(1, 2).reshape(-1, heads, x.shape[3]).float()
    p, off = (slots // page).long(), (slots % page).long()
    amax = torch.zeros_like(scale).scatter_reduce_(0, p[:, None].expand(-1, heads), rows.abs().amax(2), "amax")
    first = torch.full((pages,), page, device="cuda").scatter_reduce_(0, p, off, "amin")  # offset of the call's first token of the page
    s = _scale(amax, store)
    s = torch.where((first > 0)[:, None], torch.maximum(s, scale), s)
    s = torch.where((first < page)[:, None], s, scale)
    old = codes.float() * (scale / s)[:, :, None, None]
    kept = (torch.arange(page, device="cuda")[None] < first[:, None])[:, None, :, None] & (s > scale)[:, :, None, None]
    kept = kept & (first < page)[:, None, None, None]
    one = torch.ones((), device="cuda")
    codes.copy_(torch.where(kept, _codes(old, one, store).float(), codes.float()).to(codes.dtype))
    codes.view(torch.uint8)[p, :, off] = _codes(rows, s[p][:, :, None], store).view(torch.uint8)
    scale.copy_(s)


def _plain_dense(codes, scale, table, tokens, lens):
    """(B, H, tokens, D) in 32 bits; rows behind a request's length are zero."""
    t = table.long()
    x = _take(codes, t) * scale[t][:, :, :, None, None]  # (B, pages, H, page, D)
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :tokens]
    return x * (torch.arange(tokens, device="cuda")[None] < lens[:, None])[:, None, :, None]


def _plain_update(s):
    case = s["case"]
    dtype = _DTYPE[case["dtype"]]
    _plain_append(s["k"], s["ks"], s["new_k"], s["slots"], case)
    _plain_append(s["v"], s["vs"], s["new_v"], s["slots"], case)
    k, v = (_plain_dense(s[a], s[b], s["table"], s["tokens"], s["lens"]).to(dtype) for a, b in (("k", "ks"), ("v", "vs")))
    return dict(k=k, v=v, k_scale=s["ks"], v_scale=s["vs"])


def _plain_attend(s):
    case = s["case"]
    heads, group, dim = case["heads"], case["heads_q"] // case["heads"], case["dim"]
    lens, cu, most = s["lens"].long(), s["cu"].long(), s["q_most"]
    n = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=max(0, s["q"].shape[0] - 1))  # (B, q)
    q = s["q"][at].float().view(len(lens), most, heads, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)  # (B, H, G q, D)
    k = _plain_dense(s["k"], s["ks"], s["table"], s["kv_most"], s["lens"])
    x = (q * s["scaling"]) @ k.transpose(2, 3)
    del k
    t = torch.arange(s["kv_most"], device="cuda")
    last = lens[:, None] - n[:, None] + i  # the last token that query i sees
    seen = (t <= last[:, :, None]) & (t < lens[:, None, None])
    if case["window"]:
        seen = seen & (t > last[:, :, None] - case["window"])
    seen = seen[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = torch.exp(x - top)
    total = x.sum(3, keepdim=True)
    lse = (top + torch.log(total)).squeeze(3)
    v = _plain_dense(s["v"], s["vs"], s["table"], s["kv_most"], s["lens"])
    o = (x @ v) / torch.where(total > 0, total, 1.0)
    o = o.view(len(lens), heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(-1, case["heads_q"], dim)
    lse = lse.view(len(lens), heads, group, most).permute(0, 3, 1, 2).reshape(-1, case["heads_q"])
    live = torch.searchsorted(cu, torch.arange(s["q"].shape[0], device="cuda"), right=True) - 1
    row = live * most + torch.arange(s["q"].shape[0], device="cuda") - cu[live]
    return dict(out=o[row].to(_DTYPE[case["dtype"]]), lse=lse[row])


# ---------------------------------------------------------------------- run


def _pool(s):
    """The pool over the state's pages: made once, as a program makes it when it allocates them."""
    if "pool" not in s:
        from kvdlra_b200.paged import PagedPool

        s["pool"] = PagedPool(s["k"], s["v"], s["ks"], s["vs"])
    return s["pool"]


def _own_tables(s):
    from kvdlra_b200.paged import build_page_tables

    p = build_page_tables(s["cached"], s["new"], s["table"], s["free"], s["count"], page_size=s["case"]["page"], capacity=s["capacity"])
    return dict(table=s["table"], lens=p.lens, cu=p.cu_new, slots=p.slots, positions=p.positions, count=p.free_count)


def _own_update(s):
    from kvdlra_b200.paged import paged_append, paged_peek

    pool = _pool(s)
    paged_append(pool, s["slots"], s["new_k"], s["new_v"])
    k, v = paged_peek(pool, s["table"], s["lens"], s["tokens"], dtype=s["new_k"].dtype)
    return dict(k=k, v=v, k_scale=s["ks"], v_scale=s["vs"])


def _own_attend(s):
    from kvdlra_b200.paged import paged_attention

    out, lse = paged_attention(_pool(s), s["table"], s["lens"], s["q"], cu_q=s["cu"], max_q=s["q_most"], scaling=s["scaling"],
                               window=s["case"]["window"], return_lse=True)
    return dict(out=out, lse=lse)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "update": _own_update, "attend": _own_attend}[op](state)
    return {"tables": _plain_tables, "update": _plain_update, "attend": _plain_attend}[op](state)


# --------------------------------------------------------------------- work


def work(case):
    page = case["page"]
    if case["op"] == "tables":
        cached, new = _plan_lens(case)
        pages = sum(-(-(c + t) // page) + (-c // page) for c, t in zip(cached, new))
        tokens = sum(new) + case["pad"]
        return dict(bytes=4 * (2 * tokens + 2 * pages + 4 * case["batch"]), flops=0)
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "update":
        row = 2 * case["batch"] * case["heads"] * case["dim"]  # keys and values of one token a request
        n, total = case["new"], case["cached"] + case["new"]
        # the new rows read, their codes written; the cached codes read; the dense rows written
        return dict(bytes=row * (n * size + n + case["cached"] + total * size) + 8 * case["batch"] * case["heads"] * -(-total // page), flops=0)
    kv, q = _lens(case)
    win = case["window"]
    seen, bytes_, row = 0, 0, 2 * case["heads"] * case["dim"]
    for n, m in zip(kv, q):
        if not m:
            continue
        # query i (of m) sees tokens (n - m + i - win, n - m + i]
        last = np.arange(n - m, n, dtype=np.int64)
        first = np.maximum(0, last - win + 1) if win else np.zeros_like(last)
        each = np.where(last >= 0, last - first + 1, 0)
        seen += int(each.sum())
        if each.any():
            tokens = n - int(first[last >= 0].min())
            bytes_ += tokens * row + 8 * case["heads"] * -(-tokens // page)
    bytes_ += sum(q) * case["heads_q"] * (2 * case["dim"] * size + 4)
    return dict(bytes=bytes_, flops=4 * seen * case["heads_q"] * case["dim"])


# -------------------------------------------------------------------- exact


def _exact_power(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_scale(amax, store):
    """Power-of-two scales in 64 bits, by counting the powers that are too small."""
    powers = _exact_power(torch.arange(_FLOOR, 128, device="cuda"))
    return _exact_power(_FLOOR + (amax.double()[..., None] > _TOP[store] * powers).sum(-1))


def _exact_round(y, store):
    """The nearest representable value, ties to even, in 64 bits."""
    if store == "int8":
        return y.round().clamp(-127, 127)
    _, e = torch.frexp(y.abs().clamp(min=2.0**-6))  # |y| in [2^(e-1), 2^e): three bits behind the leading one
    step = _exact_power(e - 4)
    return ((y / step).round() * step).clamp(-448, 448)


def _exact_update(s):
    """Page by page of each request, from the definition."""
    case = s["case"]
    page, c, n, store = case["page"], case["cached"], case["new"], case["store"]
    out = {}
    for name, codes, scale, new in (("k", s["k"], s["ks"], s["new_k"]), ("v", s["v"], s["vs"], s["new_v"])):
        dense, scales = [], scale.double()
        for b in range(case["batch"]):
            ids = s["table"][b].long()
            x = _take(codes, ids).double() * scale[ids].double()[:, :, None, None]  # (pages, H, page, D)
            lo = c // page
            y = torch.zeros(ids.numel(), case["heads"], page, case["dim"], dtype=torch.float64, device="cuda")
            flat = y.transpose(1, 2).reshape(-1, case["heads"], case["dim"])
            flat[c : c + n] = new[b].transpose(0, 1).double()
            y = flat.view(ids.numel(), page, case["heads"], case["dim"]).transpose(1, 2)[lo:]
            sc = _exact_scale(y.abs().amax((2, 3)), store)
            if c % page:
                sc[0] = torch.maximum(sc[0], scale[ids[lo]].double())
            old = x[lo].clone()
            fresh = _exact_round(y / sc[:, :, None, None], store) * sc[:, :, None, None]
            if c % page:
                again = _exact_round(old / sc[0][:, None, None], store) * sc[0][:, None, None]
                fresh[0, :, : c % page] = again[:, : c % page]
            x[lo:] = fresh
            scales[ids[lo:]] = sc
            dense.append(x.transpose(0, 1).flatten(1, 2)[:, : c + n])
        out[name] = torch.stack(dense)
        out[name + "_scale"] = scales
    return dict(k=out["k"], v=out["v"], k_scale=out["k_scale"], v_scale=out["v_scale"])


def _exact_attend(s):
    """One request and KV head at a time."""
    case = s["case"]
    group, win = case["heads_q"] // case["heads"], case["window"]
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        if not m or not n:
            continue
        ids = s["table"][b, : -(-n // case["page"])].long()
        for h in range(case["heads"]):
            k = (_take(s["k"][:, h], ids).double() * s["ks"][ids, h].double()[:, None, None]).flatten(0, 1)[:n]
            v = (_take(s["v"][:, h], ids).double() * s["vs"][ids, h].double()[:, None, None]).flatten(0, 1)[:n]
            d = torch.arange(n, device="cuda")[None] - (torch.arange(m, device="cuda")[:, None] + n - m)  # token minus the query's own place
            hide = (d > 0) | (d <= -win) if win else d > 0
            for g in range(group):
                x = s["q"][cu[b] : cu[b + 1], h * group + g].double() @ k.T * s["scaling"]
                x[hide] = -math.inf
                z = torch.logsumexp(x, 1)
                w = torch.exp(x - torch.where(z == -math.inf, 0.0, z)[:, None])
                out[cu[b] : cu[b + 1], h * group + g] = w @ v
                lse[cu[b] : cu[b + 1], h * group + g] = z
    return dict(out=out, lse=lse)


def _exact_tables(s):
    """Request by request, token by token, on the host."""
    page, cached, new = s["case"]["page"], s["cached"].tolist(), s["new"].tolist()
    table, free = s["table"].cpu().numpy().copy(), s["free"].tolist()[: int(s["count"])]
    slots, positions = np.full(s["capacity"], -1, np.int32), np.zeros(s["capacity"], np.int32)
    at, cu = 0, [0]
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(-(-c // page), -(-(c + n) // page)):
            table[b, j] = free.pop()
        p = np.arange(c, c + n)
        slots[at : at + n] = table[b, p // page] * page + p % page
        positions[at : at + n] = p
        at += n
        cu.append(at)
    ints = [table, np.array([c + n for c, n in zip(cached, new)], np.int32), np.array(cu, np.int32), slots, positions, np.array([len(free)], np.int32)]
    return dict(zip(("table", "lens", "cu", "slots", "positions", "count"), (torch.from_numpy(x).cuda() for x in ints)))


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "update": _exact_update, "attend": _exact_attend}[case["op"]](s)
