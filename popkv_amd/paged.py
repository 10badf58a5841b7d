"""A paged 4-bit K/V cache for batched decode: rows quantised into pages that
sequences share, attention that reads them, and the pages' bookkeeping.

``popkv_amd.batch`` keeps each layer's K/V in static caches [B, KVH, rows, 128]
of the model dtype: every sequence owns its rows, for its longest length.
Here the layers of a model share one pool of pages, each of ``page_tokens``
tokens of every KV head, and a sequence holds the pages that its tokens need;
K and V take 4 bits a value with an fp16 (low, delta) per group of
``dim_group_size`` dimensions, 144 to 192 bytes a token and KV head instead of
512.  The reference has no counterpart (its caches are one sequence's rows,
popkv.py:105-111).

  * ``PagedKVCache``: the pool of a model; ``allocate_paged_cache`` makes one;
  * ``PageTable``: which pages each sequence of a batch holds, its token count
    and the pages' reference counts, all on the device, so that a captured
    decode step stays valid while the sequences grow; shared by the layers;
  * ``reserve_pages``, ``write_tokens``, ``PageTable.advance``: room for new
    tokens, their rows quantised into one layer, the counts moved on;
  * ``paged_attention_step`` / ``paged_indexed_attention``: the dense layers'
    attention (``popkv.dense_attention_step``) and the sparse layers' attention
    over selected tokens (``sparse_kernels.indexed_attention_split``), for a
    batch, reading the pages;
  * ``read_tokens``: the cached rows back in a float dtype, for a prefill that
    extends a cached prefix;
  * ``fork_sequences``: beams, several answers to one prompt, sequences that
    end; ``compact_pages``: the live pages to the front of the pool.

A decode step of a batch:

    reserve_pages(pages, 1, out=pages)              # once a step
    for every layer:
        attend (the current token's K/V given beside the cache)
        write_tokens(cache, layer, pages, k, v)
    pages.advance()

A page that a sequence still fills is its alone; full pages may be shared.
``status`` (int32, on the device) collects bits where a call could not do all
of its work: 1 a page table row is full, 4 no free page is left (or a token's
page is missing), 8 a fork's parent lies outside the batch.  Poll it after
steps, as for ``batch.append_batched``.  Implementation limits: head_dim 128;
1 to 16 query heads per KV head in the dense attention.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native as nat
from .popkv import LayerStepWorkspace

PAGE_TOKENS = (32, 64, 128, 256)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_INDEX_CODES = {torch.int64: nat.INDEX_I64, torch.int32: nat.INDEX_I32}


@dataclass
class PagedKVCache:
    """The pool: ``codes`` uint8 [layers, pages, KVH, page_tokens, 2, 64] (a
    token's K row, then its V row; byte j holds dims 2j, low nibble, and
    2j + 1) and ``scales`` float16 [layers, pages, KVH, page_tokens, 2,
    128 / dim_group_size, 2] ((low, delta); a value is low + code * delta)."""
    codes: torch.Tensor
    scales: torch.Tensor
    dim_group_size: int

    @property
    def layers(self) -> int:
        return int(self.codes.shape[0])

    @property
    def pages(self) -> int:
        return int(self.codes.shape[1])

    @property
    def kv_heads(self) -> int:
        return int(self.codes.shape[2])

    @property
    def page_tokens(self) -> int:
        return int(self.codes.shape[3])


@dataclass
class PageTable:
    """``table`` int32 [B, width] (the page of every ``page_tokens`` tokens,
    -1 where there is none), ``counts`` int64 [B] cached tokens, ``refs`` int32
    [pages] (0: free), and ``bound``, the most tokens any sequence holds as far
    as the host knows (it sizes launches; the counts themselves stay on the
    device)."""
    table: torch.Tensor
    counts: torch.Tensor
    refs: torch.Tensor
    page_tokens: int
    bound: int = 0

    @classmethod
    def create(cls, batch: int, max_tokens: int, cache: PagedKVCache) -> "PageTable":
        """An empty table of ``batch`` sequences of at most ``max_tokens``."""
        if batch <= 0 or max_tokens <= 0:
            raise ValueError("a page table needs at least one sequence and one token")
        dev, width = cache.codes.device, -(-int(max_tokens) // cache.page_tokens)
        return cls(torch.full((batch, width), -1, dtype=torch.int32, device=dev),
                   torch.zeros(batch, dtype=torch.int64, device=dev),
                   torch.zeros(cache.pages, dtype=torch.int32, device=dev), cache.page_tokens)

    @property
    def batch(self) -> int:
        return int(self.table.shape[0])

    @property
    def capacity(self) -> int:
        """Tokens a sequence can hold."""
        return int(self.table.shape[1]) * self.page_tokens

    def advance(self, tokens: int | torch.Tensor = 1, *, bound: int | None = None) -> None:
        """Every sequence gained ``tokens`` tokens (an int64 [B] on the device
        for different numbers, with the new ``bound``)."""
        if isinstance(tokens, torch.Tensor):
            if bound is None:
                raise ValueError("give the new bound with tokens on the device")
        elif bound is None:
            bound = self.bound + int(tokens)
        self.counts.add_(tokens)
        self.bound = min(int(bound), self.capacity)


def allocate_paged_cache(layers: int, pages: int, kv_heads: int, *, page_tokens: int = 64, dim_group_size: int = 32,
                         device: torch.device | str = "cuda") -> PagedKVCache:
    """A pool of ``pages`` pages in each of ``layers`` layers."""
    if layers <= 0 or pages <= 0 or kv_heads <= 0:
        raise ValueError("layers, pages and KV heads must be positive")
    if page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}")
    if dim_group_size not in (16, 32, 64):
        raise ValueError("dim_group_size must be one of 16, 32, 64")
    shape = (layers, pages, kv_heads, page_tokens, 2)
    return PagedKVCache(torch.zeros(*shape, 64, dtype=torch.uint8, device=device),
                        torch.zeros(*shape, 128 // dim_group_size, 2, dtype=torch.float16, device=device),
                        dim_group_size)


def _check_pool(cache: PagedKVCache) -> None:
    g = cache.dim_group_size
    if g not in (16, 32, 64):
        raise ValueError("dim_group_size must be one of 16, 32, 64")
    codes, scales = cache.codes, cache.scales
    if codes.ndim != 6 or codes.dtype != torch.uint8 or tuple(codes.shape[4:]) != (2, 64) or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous uint8 [layers, pages, KV heads, page tokens, 2, 64]")
    if tuple(scales.shape) != (*codes.shape[:5], 128 // g, 2) or scales.dtype != torch.float16 \
            or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous float16 {[*codes.shape[:5], 128 // g, 2]}")
    if cache.page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}")


def _check_table(pages: PageTable, what: str = "page table") -> None:
    t = pages.table
    if t.ndim != 2 or t.dtype != torch.int32 or not t.is_contiguous() or t.numel() == 0:
        raise ValueError(f"{what}: table must be a contiguous int32 [batch, width]")
    if tuple(pages.counts.shape) != (int(t.shape[0]),) or pages.counts.dtype != torch.int64 \
            or not pages.counts.is_contiguous():
        raise ValueError(f"{what}: counts must be a contiguous int64 [batch]")
    if pages.refs.ndim != 1 or pages.refs.dtype != torch.int32 or not pages.refs.is_contiguous() \
            or pages.refs.numel() == 0:
        raise ValueError(f"{what}: refs must be a contiguous int32 [pages]")
    if pages.page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}")


def _check_cache(cache: PagedKVCache, pages: PageTable) -> None:
    _check_pool(cache)
    _check_table(pages)
    if pages.page_tokens != cache.page_tokens or int(pages.refs.numel()) != cache.pages:
        raise ValueError("the page table belongs to a pool of another page size or page count")


def _check_layer(cache: PagedKVCache, layer: int) -> None:
    if not 0 <= layer < cache.layers:
        raise ValueError(f"layer must be in [0, {cache.layers})")


def _check_status(status: torch.Tensor | None) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 tensor of at least one element")


def _on_device(first: torch.Tensor, *tensors: torch.Tensor | None) -> torch.device:
    """Every operand on the first one's CUDA device (RuntimeError, as
    elsewhere in the package)."""
    dev = first.device
    if dev.type != "cuda":
        raise RuntimeError("the paged cache must be on a CUDA device")
    for t in tensors:
        if t is not None and t.device != dev:
            raise RuntimeError(f"every operand must be on the paged cache's device {dev}, got {t.device}")
    return dev


def _tokens(tokens: torch.Tensor, batch: int) -> torch.Tensor:
    if tuple(tokens.shape) != (batch,) or tokens.dtype != torch.int64:
        raise ValueError(f"tokens must be an int64 [{batch}] tensor")
    return tokens.contiguous()


def _pool_args(cache: PagedKVCache, layer: int, pages: PageTable) -> tuple:
    return (cache.codes.data_ptr() + layer * cache.codes.stride(0),
            cache.scales.data_ptr() + layer * cache.scales.stride(0) * 2, cache.pages, cache.kv_heads,
            cache.page_tokens, cache.dim_group_size, pages.table.data_ptr(), int(pages.table.shape[1]),
            pages.counts.data_ptr(), pages.batch)


def _rows4(x: torch.Tensor, batch: int, kv_heads: int, what: str) -> torch.Tensor:
    """K or V rows as [B, KVH, rows, 128] with contiguous, 16-byte aligned
    rows; a [B, KVH, 128] is one row."""
    if x.ndim == 3:
        x = x.unsqueeze(2)
    if x.ndim != 4 or int(x.shape[0]) != batch or int(x.shape[1]) != kv_heads or int(x.shape[3]) != 128:
        raise ValueError(f"{what} must be [{batch}, {kv_heads}, rows, 128] or [{batch}, {kv_heads}, 128]")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{x.dtype} is not supported; expected fp32/fp16/bf16")
    size = x.element_size()
    if x.stride(3) != 1 or x.data_ptr() % 16 or any(s * size % 16 or s < 0 for s in x.stride()[:3]):
        x = x.contiguous()
    return x


def _new_table(pages: PageTable, out: PageTable | None) -> PageTable:
    """The table a call writes: `out`, or a new one."""
    if out is None:
        return PageTable(torch.empty_like(pages.table), torch.empty_like(pages.counts), torch.empty_like(pages.refs),
                         pages.page_tokens, pages.bound)
    if out is not pages:
        _check_table(out, "out")
        if out.table.shape != pages.table.shape or out.refs.shape != pages.refs.shape \
                or out.page_tokens != pages.page_tokens:
            raise ValueError("out must have the page table's shape")
        same = [a.data_ptr() == b.data_ptr() for a, b in ((out.table, pages.table), (out.counts, pages.counts),
                                                          (out.refs, pages.refs))]
        if any(same) and not all(same):
            raise ValueError("out shares some of the page table's tensors: share all of them or none")
        out.bound = pages.bound
    return out


def reserve_pages(pages: PageTable, tokens: int | torch.Tensor = 1, *, bound: int | None = None,
                  status: torch.Tensor | None = None, out: PageTable | None = None) -> PageTable:
    """Pages for ``tokens`` more tokens of every sequence (an int, or an int64
    [B] on the device).  Missing pages are taken lowest first, sequences in
    order; a sequence whose share the pool or the table does not hold gets none
    and sets ``status`` (bit 4, bit 1).  Counts stay: ``advance`` moves them
    once the rows are written.  Returns a new page table, or writes ``out``
    (which may be ``pages``: in place).  ``bound``: the most tokens a sequence
    will hold, checked against the table's width."""
    _check_table(pages)
    _check_status(status)
    if bound is not None and bound > pages.capacity:
        raise RuntimeError("the page table has no entries left")
    each = 0
    if isinstance(tokens, torch.Tensor):
        tokens = _tokens(tokens, pages.batch)
    else:
        each, tokens = int(tokens), None
        if each < 0:
            raise ValueError("tokens must not be negative")
    new = _new_table(pages, out)
    dev = _on_device(pages.table, pages.counts, pages.refs, tokens, status, new.table, new.counts, new.refs)
    nbytes = int(nat.lib().popkv_page_reserve_workspace_bytes(pages.batch, int(pages.refs.numel())))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_reserve", pages.table.data_ptr(), pages.counts.data_ptr(), pages.refs.data_ptr(),
                 new.table.data_ptr(), new.counts.data_ptr(), new.refs.data_ptr(), int(pages.table.shape[1]),
                 pages.batch, int(pages.refs.numel()), pages.page_tokens, nat.ptr(tokens), each, nat.ptr(status),
                 ws.data_ptr(), nbytes, nat.stream_of(dev))
    return new


def write_tokens(cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor, v: torch.Tensor, *,
                 tokens: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Quantise new K/V rows ([B, KVH, rows, 128], any strides with contiguous
    rows, or [B, KVH, 128]: one row) of one layer into the sequences' pages:
    row t of sequence b becomes its token ``counts[b] + t``, for t <
    ``tokens[b]`` (int64 [B] on the device; None: all rows).  The pages come
    from ``reserve_pages``; a row without one is not written and sets
    ``status`` (bit 4, or bit 1 past the table's end)."""
    _check_cache(cache, pages)
    _check_layer(cache, layer)
    _check_status(status)
    k = _rows4(k, pages.batch, cache.kv_heads, "new keys")
    v = _rows4(v, pages.batch, cache.kv_heads, "new values")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("new keys and values must share shape and dtype")
    if tokens is not None:
        tokens = _tokens(tokens, pages.batch)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, k, v, tokens, status)
    with nat.on_device(dev):
        nat.call("popkv_paged_write", k.data_ptr(), v.data_ptr(), nat.dtype_code(k), *k.stride()[:3], *v.stride()[:3],
                 int(k.shape[2]), nat.ptr(tokens), *_pool_args(cache, layer, pages), nat.ptr(status),
                 nat.stream_of(dev))


def read_tokens(cache: PagedKVCache, layer: int, pages: PageTable, *, dtype: torch.dtype = torch.bfloat16,
                rows: int | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """One layer's cached rows as K, V [B, KVH, rows, 128] (``rows``: default
    ``pages.bound``).  Rows past a sequence's count are zero in new tensors and
    left as they are in ``out``."""
    _check_cache(cache, pages)
    _check_layer(cache, layer)
    if out is None:
        rows = pages.bound if rows is None else int(rows)
        if rows < 0:
            raise ValueError("rows must not be negative")
        if dtype not in _FLOATS:
            raise RuntimeError(f"{dtype} is not supported; expected fp32/fp16/bf16")
        shape = (pages.batch, cache.kv_heads, rows, 128)
        k, v = (torch.empty(shape, dtype=dtype, device=cache.codes.device) for _ in range(2))
    else:
        k, v = out
        if k.ndim != 4 or tuple(k.shape) != (pages.batch, cache.kv_heads, int(k.shape[2]), 128) \
                or v.shape != k.shape or v.dtype != k.dtype or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError(f"out must be two contiguous [{pages.batch}, {cache.kv_heads}, rows, 128] tensors")
        if rows is not None and rows != int(k.shape[2]):
            raise ValueError("rows must be out's row count")
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, k, v)
    with nat.on_device(dev):
        nat.call("popkv_paged_read", k.data_ptr(), v.data_ptr(), nat.dtype_code(k), int(k.shape[2]),
                 1 if out is None else 0, *_pool_args(cache, layer, pages), nat.stream_of(dev))
    return k, v


def _step_operands(q: torch.Tensor, cache: PagedKVCache, pages: PageTable, k: torch.Tensor, v: torch.Tensor,
                   out: torch.Tensor | None) -> int:
    batch, kv_heads = pages.batch, cache.kv_heads
    if q.ndim != 3 or int(q.shape[0]) != batch or int(q.shape[2]) != 128:
        raise ValueError(f"q must be [{batch}, query heads, 128]")
    q_heads = int(q.shape[1])
    if q_heads <= 0 or q_heads % kv_heads != 0:
        raise ValueError("query heads must be a positive multiple of the KV heads")
    for t, what in ((k, "current k"), (v, "current v")):
        if tuple(t.shape) != (batch, kv_heads, 128):
            raise ValueError(f"{what} must be [{batch}, {kv_heads}, 128]")
    if out is not None and (tuple(out.shape) != tuple(q.shape) or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor shaped like q")
    if any(t.dtype != q.dtype for t in (k, v, out) if t is not None):
        raise RuntimeError("queries, current K/V and out must share a dtype")
    nat.dtype_code(q)
    return q_heads


def _aligned(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def paged_attention_step(q: torch.Tensor, cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor,
                         v: torch.Tensor, *, max_tokens: int | None = None,
                         workspace: LayerStepWorkspace | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one decode step of one layer over every cached token and
    the current one: q [B, QH, 128], current k/v [B, KVH, 128] -> [B, QH, 128],
    query head h reading KV head h // (QH / KVH); 1 to 16 query heads per KV
    head.  ``max_tokens`` (default ``pages.bound``) bounds the device counts
    for the launch -- give the largest count a captured graph will see.  The
    workspace holds merge tickets and split states: do not share it with
    ``popkv_layer_step``."""
    _check_cache(cache, pages)
    _check_layer(cache, layer)
    q_heads = _step_operands(q, cache, pages, k, v, out)
    if q_heads // cache.kv_heads > 16:
        raise ValueError("paged attention supports 1 to 16 query heads per KV head")
    most = pages.bound if max_tokens is None else int(max_tokens)
    if most < pages.bound:
        raise ValueError("max_tokens must cover the page table's bound")
    most = min(most, pages.capacity)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, q, k, v, out)
    qc, kc, vc = _aligned(q), _aligned(k), _aligned(v)
    output = torch.empty_like(qc) if out is None else out
    nbytes = int(nat.lib().popkv_paged_attention_workspace_bytes(pages.batch, q_heads, cache.kv_heads, most))
    ws = (workspace or LayerStepWorkspace()).get(nbytes, dev, pages.batch * cache.kv_heads)
    with nat.on_device(dev):
        nat.call("popkv_paged_attention", qc.data_ptr(), nat.dtype_code(qc), *_pool_args(cache, layer, pages), most,
                 kc.data_ptr(), vc.data_ptr(), q_heads, output.data_ptr(), ws.data_ptr(), ws.numel(),
                 nat.stream_of(dev))
    return output


def paged_indexed_attention(q: torch.Tensor, cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor,
                            v: torch.Tensor, indices: torch.Tensor, head_to_kv: torch.Tensor,
                            valid_mask: torch.Tensor | None = None, *, workspace: LayerStepWorkspace | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over selected tokens, the sparse layers' counterpart of
    ``paged_attention_step``: indices [B, QH, selected] (int64 or int32), the
    current token named by ``counts[b]``, as a retrieval step returns them
    (``batch.popkv_layer_step_batched(return_indices=True)``, whose -1 entries
    pad short rows).  Indices outside [0, counts[b]] and entries whose
    ``valid_mask`` is False are left out, an index named twice counts twice,
    and a row with nothing left is zero.  head_to_kv: [QH] KV head indices.
    The workspace as for ``paged_attention_step``."""
    _check_cache(cache, pages)
    _check_layer(cache, layer)
    q_heads = _step_operands(q, cache, pages, k, v, out)
    if indices.ndim != 3 or tuple(indices.shape[:2]) != (pages.batch, q_heads) or int(indices.shape[2]) < 1:
        raise ValueError(f"indices must be [{pages.batch}, {q_heads}, selected tokens]")
    if valid_mask is not None and valid_mask.shape != indices.shape:
        raise ValueError("valid mask must match indices")
    if head_to_kv.ndim != 1 or int(head_to_kv.numel()) != q_heads:
        raise ValueError(f"head_to_kv must be a vector of {q_heads} KV head indices")
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, q, k, v, out, indices, valid_mask)
    qc, kc, vc = _aligned(q), _aligned(k), _aligned(v)
    idx = (indices if indices.dtype in _INDEX_CODES else indices.long()).contiguous()
    mask = None if valid_mask is None else valid_mask.to(torch.bool).contiguous().view(torch.uint8)
    mapping = head_to_kv.to(device=dev, dtype=torch.int64).contiguous()
    output = torch.empty_like(qc) if out is None else out
    selected = int(idx.shape[2])
    nbytes = int(nat.lib().popkv_paged_indexed_attention_workspace_bytes(pages.batch, q_heads, selected))
    ws = (workspace or LayerStepWorkspace()).get(nbytes, dev, pages.batch * q_heads)
    with nat.on_device(dev):
        nat.call("popkv_paged_indexed_attention", qc.data_ptr(), nat.dtype_code(qc),
                 *_pool_args(cache, layer, pages), kc.data_ptr(), vc.data_ptr(), idx.data_ptr(),
                 _INDEX_CODES[idx.dtype], nat.ptr(mask), mapping.data_ptr(), q_heads, selected, output.data_ptr(),
                 ws.data_ptr(), ws.numel(), nat.stream_of(dev))
    return output


def fork_sequences(cache: PagedKVCache, pages: PageTable, parents: torch.Tensor, *,
                   status: torch.Tensor | None = None, out: PageTable | None = None) -> PageTable:
    """Sequence b becomes a copy of sequence ``parents[b]`` (int64 [B] on the
    device; all at once), or empty for -1.  ``parents[b] == b`` keeps a
    sequence; -1 gives its pages back; the same parent for several sequences
    forks it: they share its full pages, and all but the lowest of them get a
    copy of its open page, in every layer.  Pages reserved ahead stay with the
    lowest child.  A child for whose copy no page is free is left empty and
    sets ``status`` bit 4; a parent outside the batch empties the sequence and
    sets bit 8.  Returns a new page table, or writes ``out`` (which may be
    ``pages``); the old one must not be written through any more."""
    _check_cache(cache, pages)
    _check_status(status)
    if tuple(parents.shape) != (pages.batch,) or parents.dtype != torch.int64:
        raise ValueError(f"parents must be an int64 [{pages.batch}] tensor")
    new = _new_table(pages, out)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, pages.refs, parents, status, new.table,
                     new.counts, new.refs)
    parents = parents.contiguous()
    width = int(pages.table.shape[1])
    nbytes = int(nat.lib().popkv_page_fork_workspace_bytes(pages.batch, width))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_fork", cache.codes.data_ptr(), cache.scales.data_ptr(), cache.layers, cache.pages,
                 cache.kv_heads, cache.page_tokens, cache.dim_group_size, pages.table.data_ptr(),
                 pages.counts.data_ptr(), pages.refs.data_ptr(), new.table.data_ptr(), new.counts.data_ptr(),
                 new.refs.data_ptr(), width, pages.batch, parents.data_ptr(), nat.ptr(status), ws.data_ptr(), nbytes,
                 nat.stream_of(dev))
    return new


def compact_pages(cache: PagedKVCache, pages: PageTable, *, out: PageTable | None = None
                  ) -> tuple[PageTable, torch.Tensor]:
    """The n live pages (refs > 0) to places 0 .. n - 1 of the pool, in every
    layer: those at n or later move, in order, to the free places before n.
    Returns the new page table (or ``out``, which may be ``pages``) and the
    int32 [pages] map of where each live page is now (-1: it was free), for
    whoever holds pages outside this table."""
    _check_cache(cache, pages)
    new = _new_table(pages, out)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, pages.refs, new.table, new.counts, new.refs)
    page_map = torch.empty_like(pages.refs)
    nbytes = int(nat.lib().popkv_page_compact_workspace_bytes(cache.pages))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_compact", cache.codes.data_ptr(), cache.scales.data_ptr(), cache.layers, cache.pages,
                 cache.kv_heads, cache.page_tokens, cache.dim_group_size, pages.table.data_ptr(),
                 pages.counts.data_ptr(), pages.refs.data_ptr(), new.table.data_ptr(), new.counts.data_ptr(),
                 new.refs.data_ptr(), int(pages.table.shape[1]), pages.batch, page_map.data_ptr(), ws.data_ptr(),
                 nbytes, nat.stream_of(dev))
    return new, page_map
