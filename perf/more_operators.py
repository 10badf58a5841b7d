"""Operators over the paged 4-bit K/V cache that serve whole chunks of new
tokens and bound a sequence's cache, as their speed is measured.

Kinds of cases, each one pass of calls that a serving loop makes for one layer
(chunk, weigh) or once for all layers (evict):

  chunk   attention of several new tokens a sequence over its cached tokens and,
          causally, over each other: prompts behind a cached prefix, a prompt's
          next part, proposed tokens that are verified at once
  weigh   the same, and every token's attention weight, summed over the new rows
          and the query heads of each KV head, added to what it has gathered
  evict   the tokens of largest gathered weight and the most recent ones of every
          layer and KV head moved to the front of their sequence, the pages
          behind them given back

``own`` false: elementary torch operations in float32.  ``own`` true: the calls
of ``popkv_amd.paged``.

Layout: codes uint8 [layers, pages, KVH, P, 2, 64] (K row, V row of a token;
byte j holds dims 2j, low nibble, and 2j + 1), scales float16 [layers, pages,
KVH, P, 2, R, 2] (low, delta of every 128 / R dims), table int32 [B, W] (page
of every P tokens, -1: none), counts int64 [B], refs int32 [pages].  A value is
low + code * delta.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"
# rows of new tokens times keys: what the largest call has, query heads counted
_MOST = 32 * 2048 * 32767


def listed() -> list[dict]:
    return [
        # the smallest call: one new token of one short chat
        dict(name="chunk-one-token", kind="chunk", batch=1, new=1, cached=180, ragged=False, q_heads=32, kv_heads=8,
             group=16, page=32, dtype="fp16"),
        # five proposed tokens and the one before them verified at once, eight chats of different lengths
        dict(name="chunk-verify-8", kind="chunk", batch=8, new=6, cached=8201, ragged=True, q_heads=32, kv_heads=8,
             group=32, page=64, dtype="bf16"),
        # chunked prefill of an 8B-shaped model: the last 2K of a 32K prompt, the largest call
        dict(name="chunk-2k-behind-30k", kind="chunk", batch=1, new=2048, cached=30719, ragged=False, q_heads=32,
             kv_heads=8, group=64, page=64, dtype="bf16"),
        # prompts of different lengths behind cached prefixes of different lengths, eight queries per KV head
        dict(name="chunk-prompts-ragged", kind="chunk", batch=6, new=1001, cached=4100, ragged=True, q_heads=64,
             kv_heads=8, group=32, page=128, dtype="fp16"),
        # a whole prompt with nothing cached
        dict(name="chunk-prompt-8k", kind="chunk", batch=1, new=8191, cached=0, ragged=False, q_heads=32, kv_heads=8,
             group=32, page=64, dtype="bf16"),
        # a small model in float32 without grouped heads
        dict(name="chunk-fp32", kind="chunk", batch=3, new=257, cached=1031, ragged=True, q_heads=8, kv_heads=8,
             group=16, page=32, dtype="fp32"),
        # decode of sixteen bounded caches, the weights gathered token by token
        dict(name="weigh-decode-16", kind="weigh", batch=16, new=1, cached=4200, ragged=True, q_heads=32, kv_heads=8,
             group=64, page=64, dtype="bf16"),
        # a prompt's last 64 tokens say what of its 32K is kept
        dict(name="weigh-window-32k", kind="weigh", batch=1, new=64, cached=32703, ragged=False, q_heads=32,
             kv_heads=8, group=64, page=64, dtype="bf16"),
        # two prompts' next parts, weights gathered all along
        dict(name="weigh-prompts-1k", kind="weigh", batch=2, new=1023, cached=8000, ragged=True, q_heads=32,
             kv_heads=8, group=32, page=64, dtype="fp16"),
        # four prompts cut to 4K once they are cached, every layer of an 8B-shaped model
        dict(name="evict-to-4k", kind="evict", batch=4, tokens=8300, keep=4096, recent=512, layers=32, kv_heads=8,
             group=64, page=64, forked=False),
        # long decodes cut back by an eighth whenever they have grown past it
        dict(name="evict-an-eighth", kind="evict", batch=16, tokens=2304, keep=2016, recent=128, layers=8, kv_heads=8,
             group=32, page=64, forked=False),
        # short beams of a small model, which share the pages of their common prefix
        dict(name="evict-forked", kind="evict", batch=6, tokens=700, keep=230, recent=17, layers=2, kv_heads=2,
             group=16, page=32, forked=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An odd or even size spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("chunk", "chunk", "weigh", "weigh", "evict"))
    group, page = rng.choice((16, 32, 64)), rng.choice((32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    batch = rng.randrange(1, 17)
    if kind != "evict":
        q_heads = kv_heads * rng.choice((1, 2, 3, 4, 8, 16) if kv_heads < 8 else (1, 2, 3, 4, 8))
        new, cached = _log(rng, 1, 4096), rng.choice((0, 1, 1, 1, 1, 1)) * _log(rng, 1, 40000)
        while batch * q_heads * new * (cached + new) > _MOST or batch * (cached + new) > 260000:
            if batch > 1 and rng.random() < 0.5:
                batch = max(1, batch // 2)
            elif cached > new:
                cached = cached * 2 // 3
            else:
                new = new * 2 // 3
        return dict(kind=kind, batch=batch, new=new, cached=cached, ragged=rng.random() < 0.6, q_heads=q_heads,
                    kv_heads=kv_heads, group=group, page=page, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    tokens, layers = _log(rng, 40, 12000), rng.randrange(1, 33)
    # at most about 600 MB of pages
    most = 600_000_000 // (kv_heads * (128 + 1024 // group))
    layers = max(1, min(layers, most // (batch * (tokens + 2 * page))))
    keep = max(1, int(tokens * rng.uniform(0.1, 0.98)))
    return dict(kind=kind, batch=batch, tokens=tokens, keep=keep, recent=rng.randrange(0, keep + 1) // 3, layers=layers,
                kv_heads=kv_heads, group=group, page=page, forked=rng.random() < 0.3)


# ---- inputs


def _lengths(case: dict, seed: int, most: int) -> list[int]:
    """Tokens of every sequence: `most`, or spread below it."""
    n = case["batch"]
    if not case["ragged"] or n == 1:
        return [most] * n
    g = torch.Generator().manual_seed(seed + 1)
    part = torch.rand(n, generator=g).tolist()
    part[0] = 1.0
    return [int(round(most * p)) for p in part]


def _randn(shape, gen) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device=_DEV)


def _outliers(kv_heads: int, gen) -> torch.Tensor:
    """[KVH, 128]: ten in four channels of every KV head, as keys have them, one elsewhere."""
    channels = torch.rand((kv_heads, 128), generator=gen, device=_DEV).argsort(1)[:, :4]
    return torch.ones((kv_heads, 128), device=_DEV).scatter_(1, channels, 10.0)


def _quantise(x: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x float32 [..., 128] -> codes uint8 [..., 64], scales float16 [..., 128 / group, 2]."""
    g = x.unflatten(-1, (-1, group))
    low = g.amin(-1).half()
    delta = ((g.amax(-1) - low.float()) / 15).half()
    step = torch.where(delta == 0, 1.0, delta.float())
    code = ((g - low.float()[..., None]) / step[..., None]).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack((low, delta), -1)


def _filled(case: dict, lengths: list[int], room: int, gen) -> dict:
    """One layer's pool with `lengths` cached tokens, their pages scattered over it, and a table of `room` tokens."""
    page, kvh = case["page"], case["kv_heads"]
    need = [-(-n // page) for n in lengths]
    pages = case["batch"] * max(1, -(-case["cached"] // page)) + 7
    order = torch.rand(pages, generator=gen, device=_DEV).argsort().to(torch.int32)
    table = torch.full((case["batch"], -(-room // page)), -1, dtype=torch.int32, device=_DEV)
    codes = torch.zeros((1, pages, kvh, page, 2, 64), dtype=torch.uint8, device=_DEV)
    scales = torch.zeros((1, pages, kvh, page, 2, 128 // case["group"], 2), dtype=torch.float16, device=_DEV)
    keys, at = _outliers(kvh, gen), 0
    for b, n in enumerate(need):  # whole pages; what lies behind a sequence's last token is never read
        if n:
            mine = order[at:at + n]
            table[b, :n] = mine
            at += n
            for which in (0, 1):
                x = _randn((n, kvh, page, 128), gen)
                codes[0, mine.long(), :, :, which], scales[0, mine.long(), :, :, which] = \
                    _quantise(x if which else x * keys[:, None], case["group"])
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    refs[order[:at].long()] = 1
    return dict(codes=codes, scales=scales, table=table, refs=refs, outliers=keys,
                counts=torch.tensor(lengths, dtype=torch.int64, device=_DEV), lengths=lengths)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    state = dict(case=case, kept={})
    batch, kvh, page = case["batch"], case["kv_heads"], case["page"]
    if case["kind"] == "evict":
        return _prepare_evict(case, seed, state, gen)
    dtype = _DTYPES[case["dtype"]]
    cached = _lengths(case, seed, case["cached"])
    new = _lengths(case, seed + 1, case["new"]) if case["new"] > 1 else [1] * batch
    state.update(_filled(case, cached, case["cached"] + case["new"], gen))
    # [B, rows, heads, 128] as a projection writes them, seen as [B, heads, rows, 128]
    rows = lambda heads: _randn((batch, case["new"], heads, 128), gen)  # noqa: E731
    state.update(q=(rows(case["q_heads"]) * 1.5).to(dtype).transpose(1, 2),
                 k=(rows(kvh) * state.pop("outliers")).to(dtype).transpose(1, 2), v=rows(kvh).to(dtype).transpose(1, 2),
                 new=new, tokens=torch.tensor(new, dtype=torch.int64, device=_DEV))
    if case["kind"] == "weigh":
        # as much as one such call adds in the mean, so that neither hides the other
        share = case["new"] * (case["q_heads"] // kvh) / (case["cached"] + case["new"])
        state["weights"] = torch.rand((batch, kvh, state["table"].shape[1] * page), generator=gen, device=_DEV) * share
    return state


def _prepare_evict(case: dict, seed: int, state: dict, gen) -> dict:
    batch, kvh, page, layers, tokens = (case[x] for x in ("batch", "kv_heads", "page", "layers", "tokens"))
    g = torch.Generator().manual_seed(seed + 2)
    # most sequences have grown past what is kept, some have not
    lengths = [int(torch.randint(min(case["keep"] + 1, tokens), tokens + 1, (1,), generator=g)) if b % 5 != 4 else
               int(torch.randint(0, case["keep"] + 1, (1,), generator=g)) for b in range(batch)]
    lengths[0] = tokens
    need = [-(-n // page) for n in lengths]
    width = -(-tokens // page) + 1
    # a fork's children share their first half of pages, the lengths allowing; free ones are left for their copies
    spare = 5 + (batch * -(-case["keep"] // page) if case["forked"] else 0)
    pages = batch * -(-tokens // page) + spare
    order = torch.rand(pages, generator=gen, device=_DEV).argsort().to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=_DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        if case["forked"] and b % 3:
            shared = min(lengths[b], lengths[b - b % 3]) // page // 2
            table[b, :shared] = table[b - b % 3, :shared]
    refs = torch.bincount(table[table >= 0], minlength=pages).to(torch.int32)
    state.update(table=table, refs=refs, counts=torch.tensor(lengths, dtype=torch.int64, device=_DEV), lengths=lengths)
    state["codes"] = torch.randint(0, 256, (layers, pages, kvh, page, 2, 64), generator=gen, device=_DEV,
                                   dtype=torch.uint8)
    state["scales"] = torch.rand((layers, pages, kvh, page, 2, 128 // case["group"], 2), generator=gen,
                                 device=_DEV).half()
    # weights as attention leaves them: a few tokens gather most, many next to nothing, early ones had longer
    w = _randn((layers, batch, kvh, width * page), gen).mul_(2.5).exp_()
    state["weights"] = w * torch.linspace(2.0, 0.2, width * page, device=_DEV)
    return state


# ---- the plain forms


def _dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """codes uint8 [..., 64], scales [..., R, 2] -> float32 [..., 128]."""
    c = torch.stack((codes & 15, codes >> 4), -1).float().flatten(-2)
    s = scales.float().repeat_interleave(128 // scales.shape[-2], -2)
    return s[..., 0] + c * s[..., 1]


def _gather(s: dict, longest: int) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V float32 [B, KVH, longest, 128] of the table's pages."""
    at = s["table"][:, :-(-longest // s["case"]["page"])].long().clamp(min=0)
    c = s["codes"][0][at].permute(0, 2, 1, 3, 4, 5).flatten(2, 3)[:, :, :longest]
    f = s["scales"][0][at].permute(0, 2, 1, 3, 4, 5, 6).flatten(2, 3)[:, :, :longest]
    return _dequantise(c[..., 0, :], f[..., 0, :, :]), _dequantise(c[..., 1, :], f[..., 1, :, :])


def _plain_chunk(s: dict):
    q, counts, tokens = s["q"].float(), s["counts"], s["tokens"]
    batch, qh, rows, _ = q.shape
    kvh, longest, dev = s["case"]["kv_heads"], max(s["lengths"]), q.device
    t = torch.arange(rows, device=dev)
    real = t[None] < tokens[:, None]  # [B, rows]
    k, v = (torch.where(real[:, None, :, None], x.float(), 0.0) for x in (s["k"], s["v"]))
    visible = (t[None, None] <= t[None, :, None]) & real[:, None]  # [B, row, new token]
    if longest:
        ck, cv = _gather(s, longest)
        live = torch.arange(longest, device=dev)[None] < counts[:, None]
        # what lies behind a sequence's last token is masked: its values have to be finite
        ck, cv = (torch.where(live[:, None, :, None], x, 0.0) for x in (ck, cv))
        k, v = torch.cat((ck, k), 2), torch.cat((cv, v), 2)
        visible = torch.cat((live[:, None].expand(batch, rows, longest), visible), 2)
    # one product a KV head: its query heads' rows together
    logits = q.reshape(batch, kvh, -1, 128) @ k.transpose(2, 3).contiguous()
    logits = logits.unflatten(2, (qh // kvh, rows)).div_(math.sqrt(128))
    logits.masked_fill_(~visible[:, None, None], float("-inf"))
    p = logits.sub_(logits.amax(4, keepdim=True)).exp_()
    p = p.div_(p.sum(4, keepdim=True))
    p.masked_fill_(~real[:, None, None, :, None], 0.0)  # rows behind a sequence's last one
    out = (p.flatten(2, 3) @ v).reshape(batch, qh, rows, 128).to(s["q"].dtype)
    if "weights" not in s:
        return out
    gathered = p.sum((2, 3))
    w = s["weights"]
    w[:, :, :longest] += gathered[:, :, :longest]
    b, i = real.nonzero(as_tuple=True)
    at = counts[b] + i
    w[b, :, at] += gathered[:, :, longest:][b, :, i]
    return dict(out=out, weights=w)


def _plain_evict(s: dict) -> dict:
    case, table, counts = s["case"], s["table"], s["counts"]
    page, keep, dev = case["page"], case["keep"], table.device
    over = counts > keep
    i = torch.arange(table.shape[1] * page, device=dev)
    recent = min(case["recent"], keep)
    n = counts[None, :, None, None]
    w = torch.where(i < n, s["weights"], float("-inf"))
    w = torch.where((i < n) & (i >= n - recent), float("inf"), w)
    # ties: the lowest index
    kept = w.sort(dim=3, descending=True, stable=True).indices[..., :keep].sort(3).values
    b = over.nonzero()[:, 0]
    # pages that another sequence holds too give way to the lowest free ones
    mine = torch.arange(table.shape[1], device=dev) < -(-keep // page)
    held, refs = table[b].long(), s["refs"].long()
    give = mine & (refs[held.clamp(min=0)] > 1) & (held >= 0)
    fresh = (refs == 0).nonzero()[:, 0][:int(give.sum())]
    now = torch.where(mine, held, -1)
    now[give] = fresh
    one = torch.ones(held.numel(), dtype=torch.int64, device=dev)
    refs = refs.scatter_add(0, held[held >= 0], -one[:int((held >= 0).sum())])
    refs = refs.scatter_add(0, now[now >= 0], one[:int((now >= 0).sum())])
    # the kept rows, all read before the first is written
    layer = torch.arange(case["layers"], device=dev)[:, None, None, None]
    head = torch.arange(case["kv_heads"], device=dev)[None, None, :, None]
    source = kept[:, b]
    place = torch.arange(keep, device=dev)
    row = torch.arange(b.numel(), device=dev)[None, :, None, None]
    src, dst = held[row, source // page], now[row, place // page]
    for pool in (s["codes"], s["scales"]):
        pool[layer, dst, head, place % page] = pool[layer, src, head, source % page]
    weights = s["weights"].clone()
    moved = torch.zeros_like(weights[:, b])
    moved[..., :keep] = weights[:, b].gather(3, source)
    weights[:, b] = moved
    out = table.clone()
    out[b] = now.to(torch.int32)
    kept = torch.where(over[None, :, None, None], kept, -1).to(torch.int32)
    return dict(codes=s["codes"].view(torch.int32), scales=s["scales"].view(torch.int32), table=out,
                refs=refs.to(torch.int32), counts=torch.where(over, keep, counts), weights=weights, kept=kept)


# ---- one pass


def run(state: dict):
    case = state["case"]
    if own:
        from popkv_amd import paged, popkv

        cache = paged.PagedKVCache(state["codes"], state["scales"], case["group"])
        pages = paged.PageTable(state["table"], state["counts"], state["refs"], case["page"], max(state["lengths"]))
        if case["kind"] == "evict":
            new, weights, kept = paged.evict_tokens(cache, pages, state["weights"], case["keep"],
                                                    recent=case["recent"])
            return dict(codes=cache.codes.view(torch.int32), scales=cache.scales.view(torch.int32), table=new.table,
                        refs=new.refs, counts=new.counts, weights=weights, kept=kept)
        workspace = state["kept"].setdefault("workspace", popkv.LayerStepWorkspace())
        weights = state.get("weights")
        out = paged.paged_chunk_attention(state["q"], cache, 0, pages, state["k"], state["v"],
                                          tokens=state["tokens"] if case["ragged"] else None, weights=weights,
                                          workspace=workspace)
        return out if weights is None else dict(out=out, weights=weights)
    return (_plain_evict if case["kind"] == "evict" else _plain_chunk)(state)


def work(case: dict) -> dict:
    group, kvh, batch = case["group"], case["kv_heads"], case["batch"]
    row = 128 + 8 * (128 // group)  # bytes of a token of one KV head, K and V
    if case["kind"] == "evict":
        over = sum(b % 5 != 4 for b in range(batch)) * case["layers"] * kvh
        tokens = (case["tokens"] + case["keep"]) / 2
        return {"bytes": over * (2 * row * case["keep"] + 4 * tokens + 8 * case["keep"]), "flops": 0}
    part = 0.6 if case["ragged"] and batch > 1 else 1.0  # what the lengths come to, in the mean
    cached, new = case["cached"] * part, case["new"] * (part if case["new"] > 1 else 1.0)
    size = 4 if case["dtype"] == "fp32" else 2
    moved = cached * kvh * row + 256 * size * new * (case["q_heads"] + kvh)
    if case["kind"] == "weigh":
        moved += 8 * kvh * (cached + new)
    return {"bytes": batch * moved, "flops": 4 * 128 * case["q_heads"] * batch * new * (cached + (new + 1) / 2)}


# ---- from the definition, in 64 bits


def _sequence(s: dict, b: int, n: int, head: int, which: int) -> torch.Tensor:
    """float64 [n, 128]: the K (0) or V (1) rows of sequence b under one KV head."""
    pages = s["table"][b, :-(-n // s["case"]["page"])].long()
    codes = s["codes"][0][pages, head][:, :, which].reshape(-1, 64)[:n]
    low, delta = s["scales"][0][pages, head][:, :, which].double().reshape(-1, 128 // s["case"]["group"], 2)[:n].unbind(2)
    nibble = (codes[..., None].to(torch.int32) >> torch.tensor([0, 4], device=codes.device)) & 15
    c = nibble.reshape(n, low.shape[1], s["case"]["group"]).double()
    return (c * delta[..., None] + low[..., None]).reshape(n, 128)


def exact(case: dict, seed: int):
    if case["kind"] == "evict":
        return None  # rows are chosen, moved and counted: nothing is computed
    s = prepare(case, seed)
    batch, kvh, qh, rows = case["batch"], case["kv_heads"], case["q_heads"], case["new"]
    per = qh // kvh
    out = torch.zeros((batch, qh, rows, 128), dtype=torch.float64, device=_DEV)
    weights = s["weights"].double() if "weights" in s else None
    for b, (n, m) in enumerate(zip(s["lengths"], s["new"])):
        for head in range(kvh if m else 0):
            k, v = (torch.cat((_sequence(s, b, n, head, which), s[x][b, head, :m].double()))
                    for which, x in enumerate("kv"))
            for h in range(head * per, head * per + per):
                for first in range(0, m, 1024):  # rows a time
                    last = min(m, first + 1024)
                    seen = n + last
                    logits = s["q"][b, h, first:last].double() @ k[:seen].T / math.sqrt(128)
                    ahead = torch.arange(seen, device=_DEV)[None] > n + torch.arange(first, last, device=_DEV)[:, None]
                    p = torch.softmax(logits.masked_fill(ahead, float("-inf")), 1)
                    out[b, h, first:last] = p @ v[:seen]
                    if weights is not None:
                        weights[b, head, :seen] += p.sum(0)
    return out if weights is None else dict(out=out, weights=weights)
