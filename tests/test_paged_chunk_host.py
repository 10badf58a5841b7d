"""Refusals of the paged cache's chunk attention and eviction, before any device call."""
from __future__ import annotations

import pytest
import torch

from popkv_amd import _native, paged

from test_paged_host import P, POOL, TABLE, pool, pool_and_table_refusals, refused, table


def operands(batch=3, q_heads=4, kv_heads=2, rows=5, dtype=torch.float32):
    return [torch.zeros(batch, h, rows, 128, dtype=dtype) for h in (q_heads, kv_heads, kv_heads)]


def test_chunk_refusals():
    cache = pool()
    t = table(cache)
    t.bound = 100
    q, k, v = operands()

    def call(q=q, k=k, v=v, layer=0, **kw):
        return paged.paged_chunk_attention(q, cache, layer, t, k, v, **kw)

    for bad in (q[:2], q[..., :64], q[0], q[:, :, 0]):
        with pytest.raises(ValueError, match="q must"):
            call(q=bad)
    for heads in (0, 3):
        with pytest.raises(ValueError, match="multiple"):
            call(q=q[:, :heads])
    for bad in (k[:, :1], k[:2], k[:, :, :4], k[..., :64], k[:, :, 0]):
        with pytest.raises(ValueError, match="new k and v"):
            call(k=bad)
        with pytest.raises(ValueError, match="new k and v"):
            call(v=bad)
    with pytest.raises(RuntimeError, match="share a dtype"):
        call(k=k.half())
    with pytest.raises(RuntimeError, match="not supported"):
        call(*operands(dtype=torch.float64))
    for bad in (torch.ones(3, dtype=torch.int32), torch.ones(2, dtype=torch.int64), torch.ones(3, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tokens"):
            call(tokens=bad)
    with pytest.raises(ValueError, match="max_tokens"):
        call(max_tokens=99)
    with pytest.raises(ValueError, match="layer"):
        call(layer=2)
    w = torch.zeros(3, 2, t.capacity)
    for bad in (w[:, :1], w[:2], w[:, :, :100], w.double(), w.transpose(0, 1).contiguous().transpose(0, 1), w[..., None]):
        with pytest.raises(ValueError, match="weights must"):
            call(weights=bad)
    with pytest.raises(RuntimeError, match="CUDA device"):
        call(weights=w)


def test_chunk_outputs():
    """An output's rows are contiguous, aligned and apart, and shares nothing with the
    operands, wherever in them it begins."""
    cache = pool()
    t = table(cache)
    q, k, v = operands()
    call = lambda out, q=q, **kw: paged.paged_chunk_attention(q, cache, 0, t, k, v, out=out, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="shaped like q"):
        call(torch.zeros(3, 4, 4, 128))
    with pytest.raises(RuntimeError, match="share a dtype"):
        call(torch.zeros(3, 4, 5, 128, dtype=torch.float16))
    for bad in (torch.zeros(3, 4, 1, 128).expand(3, 4, 5, 128), torch.zeros(3, 1, 5, 128).expand(3, 4, 5, 128),
                torch.zeros(4000).as_strided((3, 4, 5, 128), (640, 128, 64, 1))):
        with pytest.raises(ValueError, match="rows must not overlap"):
            call(bad)
    for bad in (torch.zeros(3, 4, 128, 5).transpose(2, 3), torch.zeros(3 * 4 * 5 * 128 + 1)[1:].view(3, 4, 5, 128),
                torch.zeros(3, 4, 5, 130)[..., :128]):
        with pytest.raises(ValueError, match="contiguous and 16-byte aligned"):
            call(bad)
    flat = torch.zeros(3 * 4 * 5 * 128 * 2)
    view = lambda first: flat[first:first + 3 * 4 * 5 * 128].view(3, 4, 5, 128)  # noqa: E731
    for first in (0, 128, 3 * 4 * 5 * 128 - 128):
        with pytest.raises(ValueError, match="nor overlap one"):
            call(view(first), q=view(0))
    for bad in (k, v):
        with pytest.raises(ValueError, match="nor overlap one"):
            paged.paged_chunk_attention(k.new_zeros(3, 2, 5, 128), cache, 0, t, k, v, out=bad)
    w = torch.zeros(3 * 2 * t.capacity + 3 * 4 * 5 * 128)
    inside = w[128:128 + 3 * 4 * 5 * 128].view(3, 4, 5, 128)
    with pytest.raises(ValueError, match="weights must not overlap"):
        call(None, q=inside, weights=w[:3 * 2 * t.capacity].view(3, 2, -1))
    with pytest.raises(ValueError, match="weights must not overlap"):
        call(inside, weights=w[:3 * 2 * t.capacity].view(3, 2, -1))
    # behind the last refusal: the device
    for good in (view(0), torch.zeros(3, 5, 4, 128).transpose(1, 2), torch.zeros(3, 5, 4, 192)[..., :128].transpose(1, 2),
                 torch.zeros(5, 4, 3, 128).transpose(0, 2)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call(good)


def test_token_weights():
    cache = pool()
    t = table(cache)
    w = paged.allocate_token_weights(cache, t)
    assert w.shape == (2, 3, 2, 256) and w.dtype == torch.float32 and not w.any()


def test_evict_refusals():
    cache = pool()
    t, other = table(cache), table(cache)
    w = paged.allocate_token_weights(cache, t)
    call = lambda w=w, keep=5, **kw: paged.evict_tokens(cache, t, w, keep, **kw)  # noqa: E731
    for bad in (w[:1], w[:, :2], w[..., :200], w.double(), w.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="weights must"):
            call(bad)
        with pytest.raises(ValueError, match="weights must"):
            call(weights_out=bad)
    for kw in (dict(keep=-1), dict(recent=-1)):
        with pytest.raises(ValueError, match="negative"):
            call(**kw)
    for bad in (torch.ones(3, dtype=torch.int32), torch.ones(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="keeps"):
            call(keeps=bad)
    with pytest.raises(ValueError, match="status"):
        call(status=torch.zeros(1))
    flat = torch.zeros(w.numel() + 64)
    with pytest.raises(ValueError, match="weights_out"):
        call(flat[:w.numel()].view(w.shape), weights_out=flat[64:].view(w.shape))
    other.counts = t.counts
    with pytest.raises(ValueError, match="share all of them or none"):
        call(out=other)
    with pytest.raises(ValueError, match="shape"):
        call(out=table(cache, batch=4))
    with pytest.raises(RuntimeError, match="CUDA device"):
        call(keep=10 ** 9, recent=10 ** 9, weights_out=w, out=t)


# ---------------------------------------------------------------- the C entries

def test_c_chunk_refusals():
    lib = _native.lib()
    name = "popkv_paged_chunk_attention"
    need = lib.popkv_paged_chunk_attention_workspace_bytes(2, 2, 8, 2, 5, 256, 1)
    args = dict(q=P, dtype=2, qb=5120, qh=640, qt=128, k=P, kb=1280, kh=640, kt=128, v=P, vb=1280, vh=640, vt=128, rows=5,
                tokens=None, **POOL, **TABLE, most=256, q_heads=8, out=P, ob=5120, oh=640, ot=128, fill=1, weights=P,
                stride=256, ws=P, bytes=need, stream=None)
    pool_and_table_refusals(name, args)
    for key in ("q", "k", "v", "out", "ws"):
        refused(name, args, "null pointer", **{key: None})
        refused(name, args, "16-byte", **{key: P + 8})
    for key in ("qb", "qh", "qt", "kb", "kh", "kt", "vb", "vh", "vt", "ob", "oh", "ot"):
        refused(name, args, "16-byte", **{key: 129})
        refused(name, args, "16-byte", **{key: -128})
    refused(name, args, "4-byte", weights=P + 2)
    refused(name, args, "weight stride", stride=0)
    refused(name, args, "fp32/fp16/bf16", dtype=3)
    for heads in (0, 7, 65538):
        refused(name, args, "multiple", q_heads=heads)
    refused(name, args, "token count", most=-1)
    for rows in (-1, 1 << 29):
        refused(name, args, "row count", rows=rows)
    refused(name, args, "row count", rows=(1 << 25) + 1)
    refused(name, args, "workspace bytes", bytes=need - 1)
    # an empty chunk is done, whatever its pointers
    _native.call(name, *{**args, "rows": 0, "q": None, "out": None, "ws": None}.values())
    for bad in ((3, 2, 8, 2, 5, 256, 1), (2, 0, 8, 2, 5, 256, 1), (2, 2, 7, 2, 5, 256, 1), (2, 2, 8, 2, 0, 256, 1)):
        assert lib.popkv_paged_chunk_attention_workspace_bytes(*bad) == 0


def test_c_evict_refusals():
    lib = _native.lib()
    name = "popkv_page_evict"
    need = lib.popkv_page_evict_workspace_bytes(2, 4, 4)
    args = dict(codes=P, scales=P, layers=3, pages=4, kv_heads=2, page_tokens=64, group=32, table=P, counts=P, refs_in=P,
                table_out=2 * P, counts_out=2 * P, refs_out=2 * P, width=4, batch=2, w=P, w_out=P, stride=256, keeps=None,
                keep=100, recent=5, kept=P, status=None, ws=P, bytes=need, stream=None)
    pool_and_table_refusals(name, args)
    for key in ("refs_in", "table_out", "counts_out", "refs_out", "w", "w_out", "kept", "ws"):
        refused(name, args, "null pointer", **{key: None})
    refused(name, args, "layer count", layers=0)
    refused(name, args, "token count", keep=-1)
    refused(name, args, "token count", recent=-1)
    refused(name, args, "cover the page table", stride=255)
    refused(name, args, "fit the page table", keep=257)
    refused(name, args, "or none of them", refs_out=P)
    refused(name, args, "too many", layers=65535, batch=65535, width=1)
    # a launch of so many heads would fail once the table is already the new one
    refused(name, args, "too many", layers=1, batch=32768, kv_heads=128, width=1)
    refused(name, args, "workspace bytes", bytes=need - 1)
    refused(name, args, "16-byte", ws=P + 8)
    assert lib.popkv_page_evict_workspace_bytes(0, 4, 4) == 0
