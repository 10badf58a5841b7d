"""The operators of the paged 4-bit K/V cache, as the speed of this framework is
measured on them.

Kinds of cases, each one pass of calls that a serving loop makes:

  write    new K/V rows of a batch into the pages of one layer: pages reserved,
           rows quantised into them, the sequences read back as K/V tensors
           (what a prefill that extends a cached prefix attends over)
  dense    attention of one decode step of one layer over every cached token
  indexed  the same over the tokens a retrieval selected for each query head
  fork     sequences forked, kept and freed through the page table, the open
           pages copied in every layer
  compact  live pages moved to the front of the pool in every layer

``own`` false: elementary torch operations in float32 (float64 where a value
lies next to a rounding border).  ``own`` true: the calls of
``popkv_amd.paged``.

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
# a group's extrema are held in this range, so that low + 15 * delta stays finite in float16
_LIMIT = 57344.0


def listed() -> list[dict]:
    return [
        # the smallest call: one new token of thirty-two short chats, finest groups
        dict(name="write-append-32", kind="write", batch=32, tokens=1, cached=180, ragged=True, kv_heads=8, group=16,
             page=32, dtype="fp16"),
        # prompts of different lengths admitted to a running batch, some of them continuing a cached prefix
        dict(name="write-prompts-ragged", kind="write", batch=5, tokens=4001, cached=700, ragged=True, kv_heads=8,
             group=32, page=64, dtype="fp32"),
        # one long prompt of an 8B-shaped model
        dict(name="write-prompt-32k", kind="write", batch=1, tokens=32767, cached=0, ragged=False, kv_heads=8,
             group=64, page=64, dtype="bf16"),
        # a full layer of one chat at a 4K context
        dict(name="dense-4k", kind="dense", batch=1, tokens=4095, ragged=False, q_heads=32, kv_heads=8, group=32,
             page=64, dtype="bf16"),
        # batched serving: eight sequences of 64K, the largest call
        dict(name="dense-8x64k", kind="dense", batch=8, tokens=65535, ragged=False, q_heads=32, kv_heads=8, group=64,
             page=64, dtype="bf16"),
        # continuous batching: sequences of different lengths, eight queries per KV head
        dict(name="dense-ragged-gqa8", kind="dense", batch=5, tokens=20001, ragged=True, q_heads=64, kv_heads=8,
             group=32, page=128, dtype="fp16"),
        # a sparse layer of an 8B-shaped model at 32K, the retrieval's selection of every query head
        dict(name="indexed-32k", kind="indexed", batch=1, tokens=32767, ragged=False, selected=4096, q_heads=32,
             kv_heads=8, group=64, page=64, dtype="bf16"),
        # the same for a ragged batch without grouped heads, in float32, short rows padded with -1
        dict(name="indexed-ragged-fp32", kind="indexed", batch=6, tokens=8269, ragged=True, selected=1001, q_heads=8,
             kv_heads=8, group=16, page=32, dtype="fp32"),
        # four prompts, each answered eight times: forked once their prompt is cached
        dict(name="fork-samples-4x8", kind="fork", batch=32, keep=4, tokens=8100, layers=16, kv_heads=8, group=32,
             page=64, pages=768),
        # beam search over short contexts: some beams live on, some fork, some end
        dict(name="fork-beams-64", kind="fork", batch=64, keep=23, tokens=400, layers=4, kv_heads=2, group=64,
             page=32, pages=1031),
        # half of the pool's pages live, scattered
        dict(name="compact-half", kind="compact", batch=12, tokens=2000, layers=16, kv_heads=8, group=32, page=64,
             pages=640),
        # a large table of small pages, few of them live
        dict(name="compact-sparse", kind="compact", batch=48, tokens=130, layers=2, kv_heads=4, group=16, page=32,
             pages=8200),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An odd or even size spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("write", "write", "dense", "dense", "dense", "indexed", "indexed", "fork", "compact"))
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    group, page = rng.choice((16, 32, 64)), rng.choice((32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    if kind == "write":
        batch = rng.randrange(1, 17)
        return dict(kind=kind, batch=batch, tokens=_log(rng, 1, 24000 // batch), cached=rng.randrange(0, 1000),
                    ragged=rng.random() < 0.6, kv_heads=kv_heads, group=group, page=page, dtype=dtype)
    if kind == "dense":
        batch = rng.randrange(1, 17)
        return dict(kind=kind, batch=batch, tokens=_log(rng, 1, min(65536, 300000 // batch)), ragged=rng.random() < 0.6,
                    q_heads=kv_heads * rng.choice((1, 2, 3, 4, 8, 16)), kv_heads=kv_heads, group=group, page=page,
                    dtype=dtype)
    if kind == "indexed":
        batch = rng.randrange(1, 5)
        return dict(kind=kind, batch=batch, tokens=_log(rng, 300, 32768), ragged=rng.random() < 0.6,
                    selected=_log(rng, 1, 4096 // batch), q_heads=kv_heads * rng.choice((1, 2, 4, 8)),
                    kv_heads=kv_heads, group=group, page=page, dtype=dtype)
    batch, tokens = rng.randrange(2, 33), _log(rng, 40, 2000)
    layers = rng.randrange(1, 13)
    # at most about 500 MB of pages
    most = max(1, 500_000_000 // (layers * kv_heads * page * (128 + 1024 // group)))
    need = batch * (-(-tokens // page) + 2)
    if need > most:
        tokens = max(1, (most // batch - 2) * page)
        need = batch * (-(-tokens // page) + 2)
    pages = min(max(need, most), need + _log(rng, 1, 600))
    case = dict(kind=kind, batch=batch, tokens=tokens, layers=layers, kv_heads=kv_heads, group=group, page=page,
                pages=pages)
    return dict(case, keep=rng.randrange(1, batch + 1)) if kind == "fork" else case


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


def _rows(shape, gen, dtype) -> torch.Tensor:
    """Keys with four outlier channels per KV head (dim 1), or values."""
    x = _randn(shape, gen)
    channels = torch.rand((shape[1], 128), generator=gen, device=_DEV).argsort(1)[:, :4]
    scale = torch.ones((shape[1], 128), device=_DEV).scatter_(1, channels, 10.0)
    return (x * scale[:, None]).to(dtype)


def _quantise(x: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., 128] -> codes uint8 [..., 64], scales float16 [..., 128 / group, 2]."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(-_LIMIT, _LIMIT), g.amax(-1).clamp(-_LIMIT, _LIMIT)
    bad = ~g.isfinite().all(-1)
    low = lo.half()
    delta = ((hi.double() - low.double()) / 15).float().half()
    # float64: a value next to a border between two codes
    step = torch.where(delta == 0, 1.0, delta.double())
    code = ((g.double() - low.double()[..., None]) / step[..., None]).round().clamp(0, 15)
    dead = bad | (delta == 0)
    code = torch.where(dead[..., None], 0.0, code).to(torch.uint8).flatten(-2)
    low = torch.where(bad, float("nan"), low)
    delta = torch.where(bad, 0.0, delta)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack((low, delta), -1)


def _dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """codes uint8 [..., 64], scales [..., R, 2] -> float32 [..., 128]."""
    c = torch.stack((codes & 15, codes >> 4), -1).float().flatten(-2)
    s = scales.float().repeat_interleave(128 // scales.shape[-2], -2)
    return s[..., 0] + c * s[..., 1]


def _page_tables(need: list[int], pages: int, width: int, gen) -> tuple[torch.Tensor, torch.Tensor]:
    """A table whose sequence b holds need[b] pages, scattered over the pool."""
    order = torch.rand(pages, generator=gen, device=_DEV).argsort().to(torch.int32)
    table = torch.full((len(need), width), -1, dtype=torch.int32, device=_DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    refs[order[:at].long()] = 1
    return table, refs


def _filled(case: dict, lengths: list[int], gen) -> dict:
    """One layer's pool with `lengths` cached tokens and room for the batch's longest, and its table."""
    page, group, kvh = case["page"], case["group"], case["kv_heads"]
    need = [-(-n // page) for n in lengths]
    most = -(-max(case["tokens"], 1) // page) if case["kind"] != "write" else \
        -(-(case["cached"] + case["tokens"]) // page)
    pages = case["batch"] * most + 7
    table, refs = _page_tables(need, pages, most + 2, gen)
    codes = torch.zeros((1, pages, kvh, page, 2, 64), dtype=torch.uint8, device=_DEV)
    scales = torch.zeros((1, pages, kvh, page, 2, 128 // group, 2), dtype=torch.float16, device=_DEV)
    for b, n in enumerate(need):  # whole pages; what lies behind a sequence's last token is never read
        if n:
            at = table[b, :n].long()
            for which in (0, 1):
                x = _rows((1, kvh, n * page, 128), gen, torch.float32) if which == 0 else \
                    _randn((1, kvh, n * page, 128), gen)
                c, s = _quantise(x, group)
                codes[0, at, :, :, which] = c[0].unflatten(1, (n, page)).transpose(0, 1)
                scales[0, at, :, :, which] = s[0].unflatten(1, (n, page)).transpose(0, 1)
    return dict(codes=codes, scales=scales, table=table, refs=refs,
                counts=torch.tensor(lengths, dtype=torch.int64, device=_DEV), lengths=lengths)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    state = dict(case=case, kept={})
    kind, page, group, kvh = case["kind"], case["page"], case["group"], case["kv_heads"]
    if kind == "write":
        dtype = _DTYPES[case["dtype"]]
        cached = _lengths(case, seed, case["cached"])
        new = _lengths(case, seed + 1, case["tokens"]) if case["tokens"] > 1 else [1] * case["batch"]
        state.update(_filled(case, cached, gen))
        total = [a + b for a, b in zip(cached, new)]
        shape = (case["batch"], kvh, max(new), 128)
        state.update(k=_rows(shape, gen, dtype), v=_randn(shape, gen).to(dtype), new=new,
                     tokens=torch.tensor(new, dtype=torch.int64, device=_DEV), longest=max(total))
    elif kind in ("dense", "indexed"):
        dtype = _DTYPES[case["dtype"]]
        lengths = _lengths(case, seed, case["tokens"])
        state.update(_filled(case, lengths, gen))
        batch, qh = case["batch"], case["q_heads"]
        state.update(q=(_randn((batch, qh, 128), gen) * 1.5).to(dtype), k=_randn((batch, kvh, 128), gen).to(dtype),
                     v=_randn((batch, kvh, 128), gen).to(dtype),
                     head_to_kv=torch.arange(qh, device=_DEV) // (qh // kvh))
        if kind == "indexed":
            # min(selected - 1, count) distinct tokens of every head, ascending, the current one behind them, -1 after
            most = case["selected"]
            idx = torch.full((batch, qh, most), -1, dtype=torch.int64, device=_DEV)
            for b, n in enumerate(lengths):
                k = min(most - 1, n)
                idx[b, :, :k] = torch.rand((qh, n), generator=gen, device=_DEV).argsort(1)[:, :k].sort(1).values
                idx[b, :, k] = n
            state["indices"] = idx
    else:
        layers, pages, batch = case["layers"], case["pages"], case["batch"]
        g = torch.Generator().manual_seed(seed + 2)
        holders = case["keep"] if kind == "fork" else batch
        lengths = [0] * batch
        for b in range(holders):
            lengths[b] = max(0, case["tokens"] - int(torch.randint(0, case["tokens"] // 2 + 1, (1,), generator=g)))
        need = [-(-n // page) for n in lengths]
        state["table"], state["refs"] = _page_tables(need, pages, -(-case["tokens"] // page) + 1, gen)
        state["counts"] = torch.tensor(lengths, dtype=torch.int64, device=_DEV)
        state["lengths"] = lengths
        state["codes"] = torch.randint(0, 256, (layers, pages, kvh, page, 2, 64), generator=gen, device=_DEV,
                                       dtype=torch.uint8)
        state["scales"] = torch.rand((layers, pages, kvh, page, 2, 128 // group, 2), generator=gen, device=_DEV).half()
        if kind == "fork":
            # the kept sequences stay in their places, each other place forks one of them or stays empty; every
            # seventh kept one ends where there are several
            parents = [b if holders < 3 or b % 7 != 6 else -1 for b in range(holders)]
            alive = [p for p in parents if p >= 0]
            for b in range(holders, batch):
                parents.append(alive[int(torch.randint(0, len(alive), (1,), generator=g))] if b % 11 != 10 else -1)
            state["parents"] = torch.tensor(parents, dtype=torch.int64, device=_DEV)
    return state


# ---- the plain forms


def _plain_write(s: dict) -> dict:
    page, table, counts = s["case"]["page"], s["table"].clone(), s["counts"]
    codes, scales = s["codes"][0], s["scales"][0]
    total = counts + s["tokens"]
    # the missing pages of every sequence, in order, take the lowest free ones
    slot = torch.arange(table.shape[1], device=table.device)
    missing = (table < 0) & (slot < ((total + page - 1) // page)[:, None])
    free = (s["refs"] == 0).nonzero()[:, 0]
    take = free[:int(missing.sum())]
    table[missing] = take.to(torch.int32)
    refs = s["refs"].index_fill(0, take, 1)
    # the new rows
    i = torch.arange(s["k"].shape[2], device=table.device)
    b, t = (i[None] < s["tokens"][:, None]).nonzero(as_tuple=True)
    at = counts[b] + t
    where = table[b, at // page].long()
    kc, ks = _quantise(s["k"][b, :, t], s["case"]["group"])
    vc, vs = _quantise(s["v"][b, :, t], s["case"]["group"])
    codes[where, :, at % page] = torch.stack((kc, vc), 2)
    scales[where, :, at % page] = torch.stack((ks, vs), 2)
    # and the sequences back
    k, v = _gather(codes, scales, table, s["longest"])
    live = torch.arange(s["longest"], device=table.device)[None] < total[:, None]
    k, v = (torch.where(live[:, None, :, None], x, 0.0).to(s["k"].dtype) for x in (k, v))
    return dict(k=k, v=v, table=table, refs=refs, counts=total)


def _gather(codes, scales, table, longest) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V float32 [B, KVH, longest, 128] of the table's pages."""
    width = -(-longest // codes.shape[2])
    at = table[:, :width].long().clamp(min=0)
    c = codes[at].permute(0, 2, 1, 3, 4, 5).flatten(2, 3)[:, :, :longest]
    f = scales[at].permute(0, 2, 1, 3, 4, 5, 6).flatten(2, 3)[:, :, :longest]
    return _dequantise(c[..., 0, :], f[..., 0, :, :]), _dequantise(c[..., 1, :], f[..., 1, :, :])


def _plain_dense(s: dict) -> torch.Tensor:
    q, kvh = s["q"].float(), s["case"]["kv_heads"]
    longest = max(s["lengths"])
    k, v = _gather(s["codes"][0], s["scales"][0], s["table"], max(longest, 1))
    live = torch.arange(k.shape[2], device=q.device)[None] < s["counts"][:, None]
    qg = q.unflatten(1, (kvh, -1))
    # one product a KV head, without a copy of the cache for every query head
    cached = (k @ qg.transpose(2, 3).contiguous()).transpose(2, 3) / math.sqrt(128)
    cached = torch.where(live[:, None, None], cached, float("-inf"))
    current = (qg * s["k"].float()[:, :, None]).sum(-1, keepdim=True) / math.sqrt(128)
    logits = torch.cat((cached, current), 3)
    p = (logits - logits.amax(3, keepdim=True)).exp()
    p = p / p.sum(3, keepdim=True)
    out = p[..., :-1].contiguous() @ v + p[..., -1:] * s["v"].float()[:, :, None]
    return out.flatten(1, 2).to(s["q"].dtype)


def _plain_indexed(s: dict) -> torch.Tensor:
    q, idx, counts = s["q"].float(), s["indices"], s["counts"]
    batch, qh = q.shape[:2]
    head = s["head_to_kv"][None, :, None]
    b = torch.arange(batch, device=q.device)[:, None, None]
    cached = (idx >= 0) & (idx < counts[:, None, None])
    current = (idx == counts[:, None, None])[..., None]
    at = torch.where(cached, idx, 0)
    page = s["case"]["page"]
    where = s["table"][b, at // page].long().clamp(min=0)
    c, f = s["codes"][0][where, head, at % page], s["scales"][0][where, head, at % page]
    k = torch.where(current, s["k"].float()[b, head], _dequantise(c[..., 0, :], f[..., 0, :, :]))
    v = torch.where(current, s["v"].float()[b, head], _dequantise(c[..., 1, :], f[..., 1, :, :]))
    logits = (k * q[:, :, None]).sum(-1) / math.sqrt(128)
    logits = torch.where(cached | current[..., 0], logits, float("-inf"))
    p = (logits - logits.amax(2, keepdim=True)).exp()
    p = p / p.sum(2, keepdim=True)
    return (p[..., None] * v).sum(2).to(s["q"].dtype)


def _plain_fork(s: dict) -> dict:
    page, parents, old = s["case"]["page"], s["parents"], s["table"]
    batch, width = old.shape
    pages = s["refs"].numel()
    alive = parents >= 0
    p = parents.clamp(min=0)
    counts = torch.where(alive, s["counts"][p], 0)
    slots = torch.arange(batch, device=old.device)
    same = (parents[:, None] == parents[None]) & alive[:, None]
    first = alive & (same.to(torch.uint8).argmax(1) == slots)  # the lowest place with that parent
    i = torch.arange(width, device=old.device)[None]
    full = counts // page
    keep = alive[:, None] & (first[:, None] | (i < full[:, None]))
    table = torch.where(keep, old[p], -1)
    refs = s["refs"].long()
    refs = refs.scatter_add(0, table[table >= 0].long(), torch.ones_like(table[table >= 0].long()))
    refs = refs.scatter_add(0, old[old >= 0].long(), -torch.ones_like(old[old >= 0].long()))
    # the open pages of the others go to the lowest free pages
    needy = (alive & ~first & (counts % page > 0)).nonzero()[:, 0]
    fresh = (refs == 0).nonzero()[:, 0][:needy.numel()]
    source = old[p[needy], full[needy]].long()
    table[needy, full[needy]] = fresh.to(torch.int32)
    refs = refs.index_fill(0, fresh, 1)
    s["codes"][:, fresh] = s["codes"][:, source]
    s["scales"][:, fresh] = s["scales"][:, source]
    return dict(codes=_words(s["codes"]), scales=_words(s["scales"]), table=table, refs=refs.to(torch.int32),
                counts=counts)


def _plain_compact(s: dict) -> dict:
    live = s["refs"] > 0
    n = int(live.sum())
    i = torch.arange(live.numel(), device=live.device)
    source, target = (live & (i >= n)).nonzero()[:, 0], (~live & (i < n)).nonzero()[:, 0]
    moved = torch.where(live, i, -1).to(torch.int32)
    moved[source] = target.to(torch.int32)
    table = torch.where(s["table"] >= 0, moved[s["table"].long().clamp(min=0)], -1)
    refs = torch.zeros_like(s["refs"])
    refs[moved[live].long()] = s["refs"][live]
    s["codes"][:, target] = s["codes"][:, source]
    s["scales"][:, target] = s["scales"][:, source]
    return dict(codes=_words(s["codes"]), scales=_words(s["scales"]), table=table, refs=refs, map=moved)


def _words(pool: torch.Tensor) -> torch.Tensor:
    """The pool's codes or scales as the words that move (their bits are compared)."""
    return pool.view(torch.int32)


# ---- one pass


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        from popkv_amd import paged, popkv

        cache = paged.PagedKVCache(state["codes"], state["scales"], state["case"]["group"])
        pages = paged.PageTable(state["table"], state["counts"], state["refs"], state["case"]["page"],
                                max(state["lengths"]))
        kept = state["kept"]
        if kind == "write":
            new = paged.reserve_pages(pages, state["tokens"], bound=state["longest"])
            paged.write_tokens(cache, 0, new, state["k"], state["v"], tokens=state["tokens"])
            new.advance(state["tokens"], bound=state["longest"])
            k, v = paged.read_tokens(cache, 0, new, dtype=state["k"].dtype)
            return dict(k=k, v=v, table=new.table, refs=new.refs, counts=new.counts)
        if kind == "dense":
            workspace = kept.setdefault("workspace", popkv.LayerStepWorkspace())
            return paged.paged_attention_step(state["q"], cache, 0, pages, state["k"], state["v"], workspace=workspace)
        if kind == "indexed":
            workspace = kept.setdefault("workspace", popkv.LayerStepWorkspace())
            return paged.paged_indexed_attention(state["q"], cache, 0, pages, state["k"], state["v"],
                                                 state["indices"], state["head_to_kv"], workspace=workspace)
        if kind == "fork":
            new = paged.fork_sequences(cache, pages, state["parents"])
            return dict(codes=_words(cache.codes), scales=_words(cache.scales), table=new.table, refs=new.refs,
                        counts=new.counts)
        new, moved = paged.compact_pages(cache, pages)
        return dict(codes=_words(cache.codes), scales=_words(cache.scales), table=new.table, refs=new.refs, map=moved)
    return {"write": _plain_write, "dense": _plain_dense, "indexed": _plain_indexed, "fork": _plain_fork,
            "compact": _plain_compact}[kind](state)


def work(case: dict) -> dict:
    kind, group, kvh, batch = case["kind"], case["group"], case["kv_heads"], case["batch"]
    row = 128 + 8 * (128 // group)  # bytes of a token of one KV head, K and V
    size = {"bf16": 2, "fp16": 2, "fp32": 4}.get(case.get("dtype"), 2)
    part = 0.6 if case.get("ragged") and batch > 1 else 1.0  # what the lengths come to, in the mean
    tokens = case["tokens"] * batch * part
    if kind == "write":
        new = tokens if case["tokens"] > 1 else batch
        total = new + case["cached"] * batch * part
        return {"bytes": kvh * (new * (512 * size // 2 + row) + total * (row + 512 * size // 2)),
                "flops": kvh * 256 * (6 * new + 2 * total)}
    if kind == "dense":
        return {"bytes": tokens * kvh * row, "flops": 4 * 128 * case["q_heads"] * tokens}
    if kind == "indexed":
        picked = batch * case["q_heads"] * min(case["selected"], case["tokens"] + 1)
        return {"bytes": min(picked, tokens * kvh) * row + picked * 8, "flops": 4 * 128 * picked}
    held = 0.75 * case["tokens"] / case["page"]
    page_bytes = case["layers"] * kvh * case["page"] * row
    if kind == "fork":
        moved = max(0.0, batch - case["keep"])
    else:
        live = min(case["pages"], batch * held)
        moved = live * (1 - live / case["pages"])
    return {"bytes": 2 * moved * page_bytes + 8 * case["pages"], "flops": 0}


# ---- from the definition, in 64 bits


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 [..., 128] of codes [..., 64] and scales [..., R, 2]."""
    nibble = (codes[..., None].to(torch.int32) >> torch.tensor([0, 4], device=codes.device)) & 15
    groups = scales.shape[-2]
    c = nibble.reshape(*codes.shape[:-1], groups, 128 // groups).double()
    low, delta = scales.double().unbind(-1)
    return (c * delta[..., None] + low[..., None]).reshape(*codes.shape[:-1], 128)


def _sequence(s: dict, b: int, n: int, head: int, which: int) -> torch.Tensor:
    """float64 [n, 128]: the K (0) or V (1) rows of sequence b under one KV head."""
    pages = s["table"][b, :-(-n // s["case"]["page"])].long()
    codes = s["codes"][0][pages, head][:, :, which].reshape(-1, 64)[:n]
    scales = s["scales"][0][pages, head][:, :, which].reshape(-1, 128 // s["case"]["group"], 2)[:n]
    return _values(codes, scales)


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    logits = (k * q).sum(1) / math.sqrt(128)
    w = torch.exp(logits - logits.max())
    return (w[:, None] * v).sum(0) / w.sum()


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, group, page = case["kind"], case["group"], case["page"]
    if kind in ("fork", "compact"):
        return None  # pages are copied and counted: nothing is computed
    if kind == "write":
        rows = [torch.zeros((case["batch"], case["kv_heads"], s["longest"], 128), dtype=torch.float64, device=_DEV)
                for _ in range(2)]
        for b, (n, m) in enumerate(zip(s["lengths"], s["new"])):
            for which, (out, x) in enumerate(zip(rows, (s["k"], s["v"]))):
                for head in range(case["kv_heads"]):
                    out[b, head, :n] = _sequence(s, b, n, head, which) if n else 0
                g = x[b, :, :m].double().reshape(case["kv_heads"], m, 128 // group, group)
                low = g.min(3).values.clamp(-_LIMIT, _LIMIT).to(torch.float32).to(torch.float16).double()
                top = g.max(3).values.clamp(-_LIMIT, _LIMIT)
                delta = ((top - low) / 15).to(torch.float32).to(torch.float16).double()
                code = torch.nan_to_num((g - low[..., None]) / delta[..., None]).round().clamp(0, 15)
                out[b, :, n:n + m] = (low[..., None] + code * delta[..., None]).reshape(case["kv_heads"], m, 128)
        return dict(k=rows[0], v=rows[1], table=None, refs=None, counts=None)
    qh = case["q_heads"]
    if case["batch"] * qh > 400:
        return None
    out = torch.zeros((case["batch"], qh, 128), dtype=torch.float64, device=_DEV)
    per = qh // case["kv_heads"]
    for b, n in enumerate(s["lengths"]):
        for head in range(case["kv_heads"]):
            k = torch.cat((_sequence(s, b, n, head, 0), s["k"][b, head].double()[None]))
            v = torch.cat((_sequence(s, b, n, head, 1), s["v"][b, head].double()[None]))
            for h in range(head * per, head * per + per):
                pick = s["indices"][b, h] if kind == "indexed" else None
                rows = pick[pick >= 0] if kind == "indexed" else slice(None)
                out[b, h] = _attend(s["q"][b, h].double(), k[rows], v[rows])
    return out
