"""The paged cache's refusals, before any device call, and its host-side
bookkeeping."""
from __future__ import annotations

import pytest
import torch

from popkv_amd import _native, paged


def pool(**kw):
    return paged.allocate_paged_cache(2, 6, 2, device="cpu", **kw)


def table(cache, batch=3, tokens=200):
    return paged.PageTable.create(batch, tokens, cache)


def test_allocation_and_its_refusals():
    cache = pool(page_tokens=32, dim_group_size=16)
    assert (cache.layers, cache.pages, cache.kv_heads, cache.page_tokens) == (2, 6, 2, 32)
    assert tuple(cache.codes.shape) == (2, 6, 2, 32, 2, 64) and tuple(cache.scales.shape) == (2, 6, 2, 32, 2, 8, 2)
    for kw in (dict(page_tokens=16), dict(page_tokens=48), dict(page_tokens=512)):
        with pytest.raises(ValueError, match="page_tokens"):
            pool(**kw)
    with pytest.raises(ValueError, match="dim_group_size"):
        pool(dim_group_size=128)
    for shape in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError, match="positive"):
            paged.allocate_paged_cache(*shape, device="cpu")
    for batch, tokens in ((0, 5), (2, 0)):
        with pytest.raises(ValueError, match="at least one"):
            paged.PageTable.create(batch, tokens, cache)


def test_page_table_counts():
    t = table(pool())
    assert t.batch == 3 and t.capacity == 256 and t.bound == 0
    t.advance()
    t.advance(4)
    assert t.counts.tolist() == [5, 5, 5] and t.bound == 5
    with pytest.raises(ValueError, match="bound"):
        t.advance(torch.tensor([1, 2, 3]))
    t.advance(torch.tensor([1, 2, 300]), bound=305)
    assert t.counts.tolist() == [6, 7, 305] and t.bound == 256


def test_pool_and_table_refusals():
    cache = pool()
    t = table(cache)
    k = torch.zeros(3, 2, 1, 128)
    call = lambda c, p: paged.write_tokens(c, 0, p, k, k)  # noqa: E731
    with pytest.raises(ValueError, match="codes"):
        call(paged.PagedKVCache(cache.codes.int(), cache.scales, 32), t)
    with pytest.raises(ValueError, match="codes"):
        call(paged.PagedKVCache(cache.codes.transpose(0, 1), cache.scales, 32), t)
    with pytest.raises(ValueError, match="scales"):
        call(paged.PagedKVCache(cache.codes, cache.scales, 16), t)
    with pytest.raises(ValueError, match="scales"):
        call(paged.PagedKVCache(cache.codes, cache.scales.float(), 32), t)
    with pytest.raises(ValueError, match="dim_group_size"):
        call(paged.PagedKVCache(cache.codes, cache.scales, 8), t)
    with pytest.raises(ValueError, match="another page size"):
        call(pool(page_tokens=32), t)
    with pytest.raises(ValueError, match="another page size"):
        call(cache, paged.PageTable(t.table, t.counts, t.refs[:4].contiguous(), 64))
    for bad in (paged.PageTable(t.table.long(), t.counts, t.refs, 64), paged.PageTable(t.table.t(), t.counts, t.refs, 64),
                paged.PageTable(t.table[0], t.counts, t.refs, 64)):
        with pytest.raises(ValueError, match="table must"):
            call(cache, bad)
    with pytest.raises(ValueError, match="counts"):
        call(cache, paged.PageTable(t.table, t.counts.int(), t.refs, 64))
    with pytest.raises(ValueError, match="counts"):
        call(cache, paged.PageTable(t.table, t.counts[:2], t.refs, 64))
    with pytest.raises(ValueError, match="refs"):
        call(cache, paged.PageTable(t.table, t.counts, t.refs.long(), 64))
    with pytest.raises(ValueError, match="layer"):
        paged.write_tokens(cache, 2, t, k, k)
    with pytest.raises(ValueError, match="layer"):
        paged.read_tokens(cache, -1, t)
    with pytest.raises(RuntimeError, match="CUDA device"):
        call(cache, t)


def test_write_and_read_refusals():
    cache = pool()
    t = table(cache)
    k = torch.zeros(3, 2, 5, 128)
    for bad in (k[:2], k[:, :1], k[..., :64], torch.zeros(2, 128)):
        with pytest.raises(ValueError, match="new keys"):
            paged.write_tokens(cache, 0, t, bad, k)
    with pytest.raises(ValueError, match="share"):
        paged.write_tokens(cache, 0, t, k, k[:, :, :4])
    with pytest.raises(ValueError, match="share"):
        paged.write_tokens(cache, 0, t, k, k.half())
    with pytest.raises(RuntimeError, match="not supported"):
        paged.write_tokens(cache, 0, t, k.double(), k.double())
    for bad in (torch.ones(3, dtype=torch.int32), torch.ones(2, dtype=torch.int64), torch.ones(3, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tokens"):
            paged.write_tokens(cache, 0, t, k, k, tokens=bad)
    with pytest.raises(ValueError, match="status"):
        paged.write_tokens(cache, 0, t, k, k, status=torch.zeros(1))
    with pytest.raises(ValueError, match="rows"):
        paged.read_tokens(cache, 0, t, rows=-1)
    with pytest.raises(RuntimeError, match="not supported"):
        paged.read_tokens(cache, 0, t, dtype=torch.int32)
    with pytest.raises(ValueError, match="out"):
        paged.read_tokens(cache, 0, t, out=(k, k.half()))
    with pytest.raises(ValueError, match="out"):
        paged.read_tokens(cache, 0, t, out=(k[:, :1], k[:, :1]))
    for bad in (k[:, :, :4].contiguous(), k[:2], k[0]):
        with pytest.raises(ValueError, match="out"):
            paged.read_tokens(cache, 0, t, out=(k, bad))
        if bad.shape != (3, 2, 4, 128):
            with pytest.raises(ValueError, match="out"):
                paged.read_tokens(cache, 0, t, out=(bad, bad))
    with pytest.raises(ValueError, match="row count"):
        paged.read_tokens(cache, 0, t, rows=4, out=(k, k))


def test_attention_refusals():
    cache = pool()
    t = table(cache)
    t.bound = 100
    q, k = torch.zeros(3, 8, 128), torch.zeros(3, 2, 128)
    idx, mapping = torch.zeros(3, 8, 4, dtype=torch.int64), torch.zeros(8, dtype=torch.int64)
    dense = lambda q, k, v, **kw: paged.paged_attention_step(q, cache, 0, t, k, v, **kw)  # noqa: E731
    pick = lambda *a, **kw: paged.paged_indexed_attention(q, cache, 0, t, k, k, *a, **kw)  # noqa: E731
    for bad in (q[:2], q[..., :64], q[0]):
        with pytest.raises(ValueError, match="q must"):
            dense(bad, k, k)
    with pytest.raises(ValueError, match="multiple"):
        dense(q[:, :3], k, k)
    with pytest.raises(ValueError, match="1 to 16"):
        dense(torch.zeros(3, 34, 128), k, k)
    with pytest.raises(ValueError, match="current k"):
        dense(q, k[:, :1], k)
    with pytest.raises(ValueError, match="current v"):
        dense(q, k, k[:2])
    with pytest.raises(ValueError, match="max_tokens"):
        dense(q, k, k, max_tokens=99)
    with pytest.raises(ValueError, match="out"):
        dense(q, k, k, out=q[:, :4])
    for call in (lambda **kw: dense(q, k, k, **kw), lambda **kw: pick(idx, mapping, **kw)):
        with pytest.raises(ValueError, match="one of the operands"):
            call(out=q)
    with pytest.raises(RuntimeError, match="share a dtype"):
        dense(q, k.half(), k)
    with pytest.raises(RuntimeError, match="share a dtype"):
        dense(q, k, k, out=q.half())
    with pytest.raises(RuntimeError, match="not supported"):
        dense(q.double(), k.double(), k.double())
    for bad in (idx[0], idx[:2], idx[:, :4], idx[..., :0]):
        with pytest.raises(ValueError, match="indices"):
            pick(bad, mapping)
    with pytest.raises(ValueError, match="valid mask"):
        pick(idx, mapping, torch.ones(3, 8, 3))
    with pytest.raises(ValueError, match="head_to_kv"):
        pick(idx, mapping[:4])
    with pytest.raises(RuntimeError, match="CUDA device"):
        pick(idx, mapping)
    with pytest.raises(RuntimeError, match="CUDA device"):
        dense(q, k, k)


def test_page_call_refusals():
    cache = pool()
    t, other = table(cache), table(cache)
    parents = torch.arange(3)
    with pytest.raises(ValueError, match="negative"):
        paged.reserve_pages(t, -1)
    with pytest.raises(RuntimeError, match="no entries left"):
        paged.reserve_pages(t, 1, bound=257)
    for bad in (parents.int(), parents[:2]):
        with pytest.raises(ValueError, match="parents"):
            paged.fork_sequences(cache, t, bad)
    other.counts = t.counts
    for call in (lambda out: paged.reserve_pages(t, out=out), lambda out: paged.fork_sequences(cache, t, parents, out=out),
                 lambda out: paged.compact_pages(cache, t, out=out)):
        with pytest.raises(ValueError, match="share all of them or none"):
            call(other)
        with pytest.raises(ValueError, match="shape"):
            call(table(cache, batch=4))
        with pytest.raises(RuntimeError, match="CUDA device"):
            call(None)


# ---------------------------------------------------------------- the C entries

P = 1 << 20  # an aligned address that no refused call follows


def refused(name, args, text, **change):
    names = list(args)
    full = {**args, **change}
    with pytest.raises(RuntimeError, match=text):
        _native.call(name, *(full[n] for n in names))


POOL = dict(codes=P, scales=P, pages=4, kv_heads=2, page_tokens=64, group=32)
TABLE = dict(table=P, width=4, counts=P, batch=2)


def pool_and_table_refusals(name, args):
    for key in ("codes", "scales", "table", "counts"):
        refused(name, args, "null pointer", **{key: None})
    refused(name, args, "page or KV head", pages=0)
    refused(name, args, "page or KV head", pages=(1 << 30) + 1)
    refused(name, args, "page or KV head", kv_heads=0)
    refused(name, args, "page_tokens", page_tokens=48)
    refused(name, args, "dim_group_size", group=128)
    refused(name, args, "16-byte", codes=P + 8)
    refused(name, args, "batch or page table", batch=0)
    refused(name, args, "batch or page table", batch=65536)
    refused(name, args, "batch or page table", width=0)
    refused(name, args, "batch or page table", width=1 << 25)


def test_c_write_and_read_refusals():
    args = dict(k=P, v=P, dtype=2, kb=1280, kh=640, kt=128, vb=1280, vh=640, vt=128, rows=5, tokens=None, **POOL, **TABLE,
                status=None, stream=None)
    pool_and_table_refusals("popkv_paged_write", args)
    refused("popkv_paged_write", args, "null pointer", k=None)
    refused("popkv_paged_write", args, "fp32/fp16/bf16", dtype=3)
    refused("popkv_paged_write", args, "row count", rows=-1)
    refused("popkv_paged_write", args, "16-byte", kt=129)
    refused("popkv_paged_write", args, "16-byte", vb=-128)
    refused("popkv_paged_write", args, "16-byte", v=P + 4)
    args = dict(k=P, v=P, dtype=2, rows=5, fill=0, **POOL, **TABLE, stream=None)
    pool_and_table_refusals("popkv_paged_read", args)
    refused("popkv_paged_read", args, "null pointer", v=None)
    refused("popkv_paged_read", args, "row count", rows=-1)
    refused("popkv_paged_read", args, "fp32/fp16/bf16", dtype=-1)
    refused("popkv_paged_read", args, "16-byte", k=P + 2)


def test_c_attention_refusals():
    lib = _native.lib()
    need = lib.popkv_paged_attention_workspace_bytes(2, 8, 2, 256)
    args = dict(q=P, dtype=2, **POOL, **TABLE, most=256, ck=P, cv=P, q_heads=8, out=P, ws=P, bytes=need, stream=None)
    pool_and_table_refusals("popkv_paged_attention", args)
    for key in ("q", "ck", "cv", "out", "ws"):
        refused("popkv_paged_attention", args, "null pointer", **{key: None})
        refused("popkv_paged_attention", args, "16-byte", **{key: P + 8})
    refused("popkv_paged_attention", args, "fp32/fp16/bf16", dtype=7)
    for heads in (0, 7, 34):
        refused("popkv_paged_attention", args, "1 to 16", q_heads=heads)
    refused("popkv_paged_attention", args, "token count", most=-1)
    refused("popkv_paged_attention", args, "workspace bytes", bytes=need - 1)
    need = lib.popkv_paged_indexed_attention_workspace_bytes(2, 8, 100)
    args = dict(q=P, dtype=2, **POOL, **TABLE, ck=P, cv=P, idx=P, index=0, mask=None, map=P, q_heads=8, selected=100,
                out=P, ws=P, bytes=need, stream=None)
    pool_and_table_refusals("popkv_paged_indexed_attention", args)
    for key in ("q", "ck", "cv", "idx", "map", "out", "ws"):
        refused("popkv_paged_indexed_attention", args, "null pointer", **{key: None})
    refused("popkv_paged_indexed_attention", args, "int64 or int32", index=2)
    refused("popkv_paged_indexed_attention", args, "too many heads", q_heads=0)
    refused("popkv_paged_indexed_attention", args, "selection", selected=0)
    refused("popkv_paged_indexed_attention", args, "workspace bytes", bytes=need - 1)
    assert lib.popkv_paged_attention_workspace_bytes(0, 8, 2, 256) == 0
    assert lib.popkv_paged_indexed_attention_workspace_bytes(2, 8, 0) == 0


def test_c_page_call_refusals():
    lib = _native.lib()
    need = lib.popkv_page_reserve_workspace_bytes(2, 4)
    args = dict(table=P, counts=P, refs_in=P, table_out=2 * P, counts_out=2 * P, refs_out=2 * P, width=4, batch=2,
                pages=4, page_tokens=64, tokens=None, each=1, status=None, ws=P, bytes=need, stream=None)
    for key in ("table", "counts", "refs_in", "table_out", "counts_out", "refs_out", "ws"):
        refused("popkv_page_reserve", args, "null pointer", **{key: None})
    refused("popkv_page_reserve", args, "page count", pages=0)
    refused("popkv_page_reserve", args, "page_tokens", page_tokens=16)
    refused("popkv_page_reserve", args, "token count", each=-1)
    for key in ("table_out", "counts_out", "refs_out"):
        refused("popkv_page_reserve", args, "or none of them", **{key: P})
    refused("popkv_page_reserve", args, "workspace bytes", bytes=need - 1)
    refused("popkv_page_reserve", args, "batch or page table", batch=0)
    need = lib.popkv_page_fork_workspace_bytes(2, 4)
    pool_args = dict(codes=P, scales=P, layers=3, pages=4, kv_heads=2, page_tokens=64, group=32)
    tables = dict(table=P, counts=P, refs_in=P, table_out=2 * P, counts_out=2 * P, refs_out=2 * P, width=4, batch=2)
    fork = dict(**pool_args, **tables, parents=P, status=None, ws=P, bytes=need, stream=None)
    compact = dict(**pool_args, **tables, map=P, ws=P, bytes=lib.popkv_page_compact_workspace_bytes(4), stream=None)
    for name, args, own in (("popkv_page_fork", fork, "parents"), ("popkv_page_compact", compact, "map")):
        pool_and_table_refusals(name, args)
        for key in (own, "refs_in", "table_out", "counts_out", "refs_out", "ws"):
            refused(name, args, "null pointer", **{key: None})
        refused(name, args, "layer count", layers=0)
        refused(name, args, "or none of them", refs_out=P)
        refused(name, args, "workspace bytes", bytes=args["bytes"] - 1)


def test_c_no_rows_are_no_work():
    """An empty tensor has no address: a call without rows is done, whatever
    its row pointers, and still refuses a bad pool, table, type or row count."""
    write = dict(k=None, v=None, dtype=2, kb=0, kh=0, kt=128, vb=0, vh=0, vt=128, rows=0, tokens=None, **POOL, **TABLE,
                 status=None, stream=None)
    read = dict(k=None, v=None, dtype=2, rows=0, fill=1, **POOL, **TABLE, stream=None)
    for name, args in (("popkv_paged_write", write), ("popkv_paged_read", read)):
        _native.call(name, *args.values())
        _native.call(name, *{**args, "k": P + 2, "v": P + 4}.values())
        pool_and_table_refusals(name, args)
        refused(name, args, "fp32/fp16/bf16", dtype=3)
        refused(name, args, "row count", rows=-1)
        refused(name, args, "null pointer", rows=1)


def test_outputs_that_overlap_operands():
    """Workgroups read the operands while others write: an output that shares
    memory with one is refused wherever in it that begins."""
    cache = pool()
    t = table(cache)
    t.bound = 100
    idx, mapping = torch.zeros(3, 8, 4, dtype=torch.int64), torch.zeros(8, dtype=torch.int64)
    flat = torch.zeros(9 * 8 * 128)
    rows = lambda first, heads: flat[first * 128:(first + 3 * heads) * 128].view(3, heads, 128)  # noqa: E731
    q, k, v = rows(0, 8), rows(24, 2), rows(30, 2)
    for first in (1, 23, 24, 27, 29, 30, 35):
        for call in (lambda out: paged.paged_attention_step(q, cache, 0, t, k, v, out=out),
                     lambda out: paged.paged_indexed_attention(q, cache, 0, t, k, v, idx, mapping, out=out)):
            with pytest.raises(ValueError, match="one of the operands"):
                call(rows(first, 8))
    for call in (lambda out: paged.paged_attention_step(q, cache, 0, t, k, v, out=out),
                 lambda out: paged.paged_indexed_attention(q, cache, 0, t, k, v, idx, mapping, out=out)):
        with pytest.raises(RuntimeError, match="CUDA device"):  # behind the last of them
            call(rows(36, 8))
    x = torch.zeros(2 * 3 * 2 * 5 * 128 + 128)
    part = lambda first: x[first:first + 3 * 2 * 5 * 128].view(3, 2, 5, 128)  # noqa: E731
    for second in (0, 128, 3 * 2 * 5 * 128 - 128):
        for out in ((part(0), part(second)), (part(second), part(0))):
            with pytest.raises(ValueError, match="overlap"):
                paged.read_tokens(cache, 0, t, out=out)
    with pytest.raises(RuntimeError, match="CUDA device"):
        paged.read_tokens(cache, 0, t, out=(part(0), part(3 * 2 * 5 * 128)))
    none = torch.zeros(3, 2, 0, 128)
    with pytest.raises(RuntimeError, match="CUDA device"):  # no rows: nothing to overlap
        paged.read_tokens(cache, 0, t, out=(none, none))


def test_output_tables_that_overlap_the_input():
    """An output table of its own shares no memory with the input's, not even a
    part of a tensor."""
    cache = pool()
    raw = (torch.full((4, 4), -1, dtype=torch.int32), torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32))
    at = lambda i, j, n: paged.PageTable(raw[0][i:i + 3], raw[1][j:j + 3], raw[2][n:n + 6], 64)  # noqa: E731
    pages = at(0, 0, 0)
    apart = table(cache)
    for table_at, counts_at, refs_at in ((1, None, None), (None, 1, None), (None, None, 2), (1, 1, 1)):
        other = at(table_at or 0, counts_at or 0, refs_at or 0)
        out = paged.PageTable(apart.table if table_at is None else other.table,
                              apart.counts if counts_at is None else other.counts,
                              apart.refs if refs_at is None else other.refs, 64)
        for call in (lambda: paged.reserve_pages(pages, out=out),
                     lambda: paged.fork_sequences(cache, pages, torch.arange(3), out=out),
                     lambda: paged.compact_pages(cache, pages, out=out)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    for out in (at(0, 0, 0), apart):  # in place by another name, and apart
        with pytest.raises(RuntimeError, match="CUDA device"):
            paged.reserve_pages(pages, out=out)


def test_a_refused_call_leaves_its_output_as_it_was():
    cache = pool()
    pages, out = table(cache), table(cache)
    pages.bound, out.bound = 100, 7
    for call in (lambda: paged.reserve_pages(pages, out=out),
                 lambda: paged.fork_sequences(cache, pages, torch.arange(3), out=out),
                 lambda: paged.compact_pages(cache, pages, out=out)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()
        assert out.bound == 7
