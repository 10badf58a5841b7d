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
  * ``paged_chunk_attention``: several new tokens a sequence at once, over the
    cached tokens and, causally, each other: a prompt behind a cached prefix, a
    prompt's next part, proposed tokens to verify; it can gather every token's
    attention weight (``allocate_token_weights``) as it goes;
  * ``evict_tokens``: sequences cut, in every layer and KV head by itself, to their
    most recent tokens and those that gathered the largest weights;
  * ``read_tokens``: the cached rows back in a float dtype;
  * ``fork_sequences``: beams, several answers to one prompt, sequences that
    end; ``compact_pages``: the live pages to the front of the pool.

A decode step of a batch:

    reserve_pages(pages, 1, out=pages)              # once a step
    for every layer:
        attend (the current token's K/V given beside the cache)
        write_tokens(cache, layer, pages, k, v)
    pages.advance()

A prompt, or a part of one, is the same with ``paged_chunk_attention``, ``tokens``
of every sequence reserved, written and advanced; a bounded cache gives that call
``weights=w[layer]`` (one token is a chunk too) and calls
``evict_tokens(cache, pages, w, keep, out=pages, weights_out=w)`` once the
sequences have grown past ``keep`` by some.  Proposed tokens are verified without
``weights``, as many as were accepted advanced over, and before that gathered by a
second call with ``tokens`` of them: a row adds to every token that it sees, also if
its own token is rejected.

A page that a sequence still fills is its alone; full pages may be shared.
``status`` (int32, on the device) collects bits where a call could not do all
of its work: 1 a page table row is full, 4 no free page is left (or a token's
page is missing), 8 a fork's parent lies outside the batch.  Poll it after
steps, as for ``batch.append_batched``.  Implementation limits: head_dim 128;
1 to 16 query heads per KV head in ``paged_attention_step``.  The retrieval's
packed planes are not part of the pages: forks and compactions leave them as they
are; ``evict_tokens`` says which tokens it kept.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _native as nat
from .popkv import LayerStepWorkspace

PAGE_TOKENS = (32, 64, 128, 256)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_INDEX_CODES = {torch.int64: nat.INDEX_I64, torch.int32: nat.INDEX_I32}
_TICKET_KIB = 256  # the zero region of an attention workspace, of any call


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
    as the host knows (the counts themselves stay on the device).  It sizes
    launches, and the dense attention leaves out what lies past it; ``advance``
    moves it and no other call does.  A program that knows better sets it: higher
    after replays of a captured step, which move the counts alone, lower once its
    long sequences have ended."""
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
        for different numbers, with the new ``bound``).  Negative numbers take
        tokens back, but not into a page that a fork shares: what is written
        there next would be every holder's."""
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


# (The checks below run at every call of a decode loop, which the host can
# bound: each reads a shape once.)

def _check_table(pages: PageTable, what: str = "page table") -> tuple[int, int, int]:
    """Shapes and types of a page table (ValueError): (batch, width, pages)."""
    table, counts, refs = pages.table, pages.counts, pages.refs
    shape, batches, held = table.shape, counts.shape, refs.shape
    if len(shape) != 2 or table.dtype is not torch.int32 or not table.is_contiguous() or not table.numel():
        raise ValueError(f"{what}: table must be a contiguous int32 [batch, width]")
    batch, width = shape
    if len(batches) != 1 or batches[0] != batch or counts.dtype is not torch.int64 or not counts.is_contiguous():
        raise ValueError(f"{what}: counts must be a contiguous int64 [batch]")
    if len(held) != 1 or refs.dtype is not torch.int32 or not held[0] or not refs.is_contiguous():
        raise ValueError(f"{what}: refs must be a contiguous int32 [pages]")
    if pages.page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}")
    return batch, width, held[0]


def _check_cache(cache: PagedKVCache, pages: PageTable, layer: int = 0) -> tuple[int, int, int, tuple]:
    """Shapes and types of a pool and its page table (ValueError): batch,
    width, KV heads, and the C entries' arguments for a layer, from the codes
    to the batch."""
    batch, width, count = _check_table(pages)
    codes, scales, g = cache.codes, cache.scales, cache.dim_group_size
    if g != 16 and g != 32 and g != 64:
        raise ValueError("dim_group_size must be one of 16, 32, 64")
    shape = codes.shape
    if len(shape) != 6 or codes.dtype is not torch.uint8 or shape[4] != 2 or shape[5] != 64 \
            or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous uint8 [layers, pages, KV heads, page tokens, 2, 64]")
    layers, held, kv_heads, page_tokens, _, _ = shape
    want = (layers, held, kv_heads, page_tokens, 2, 128 // g, 2)
    if scales.shape != want or scales.dtype is not torch.float16 or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous float16 {list(want)}")
    if pages.page_tokens != page_tokens or count != held:
        raise ValueError("the page table belongs to a pool of another page size or page count")
    if not 0 <= layer < layers:
        raise ValueError(f"layer must be in [0, {layers})")
    rows = layer * held * kv_heads * page_tokens
    return batch, width, kv_heads, (codes.data_ptr() + rows * 128, scales.data_ptr() + rows * (1024 // g), held,
                                    kv_heads, page_tokens, g, pages.table.data_ptr(), width, pages.counts.data_ptr(),
                                    batch)


def _check_status(status: torch.Tensor | None) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 tensor of at least one element")


def _on_device(first: torch.Tensor, *tensors: torch.Tensor | None) -> torch.device:
    """Every operand on the first one's CUDA device (RuntimeError, as
    elsewhere in the package)."""
    index = first.get_device()
    if index < 0:
        raise RuntimeError("the paged cache must be on a CUDA device")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"every operand must be on the paged cache's device {first.device}, got {t.device}")
    return first.device


@lru_cache(maxsize=4096)
def _workspace_bytes(call: str, *sizes: int) -> int:
    return getattr(nat.lib(), call + "_workspace_bytes")(*sizes)


def _tokens(tokens: torch.Tensor, batch: int) -> torch.Tensor:
    if tokens.shape != (batch,) or tokens.dtype is not torch.int64:
        raise ValueError(f"tokens must be an int64 [{batch}] tensor")
    return tokens.contiguous()


def _rows(x: torch.Tensor, batch: int, kv_heads: int, what: str) -> tuple[torch.Tensor, int, int, int, int]:
    """K or V rows [B, KVH, rows, 128], or [B, KVH, 128] for one row, with
    contiguous and 16-byte aligned rows (a copy where they are not): the
    tensor, its row count and its strides."""
    shape = x.shape
    n = len(shape)
    if (n != 4 and n != 3) or shape[0] != batch or shape[1] != kv_heads or shape[-1] != 128:
        raise ValueError(f"{what} must be [{batch}, {kv_heads}, rows, 128] or [{batch}, {kv_heads}, 128]")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{x.dtype} is not supported; expected fp32/fp16/bf16")
    rows = shape[2] if n == 4 else 1
    if not x.is_contiguous() or x.data_ptr() % 16:
        strides, unit = x.stride(), 16 // x.element_size()
        if strides[-1] == 1 and x.data_ptr() % 16 == 0 and not any(s % unit for s in strides[:-1]):
            return x, rows, strides[0], strides[1], strides[2] if n == 4 else 128
        x = _aligned(x)
    return x, rows, kv_heads * rows * 128, rows * 128, 128


def _new_table(pages: PageTable, out: PageTable | None) -> PageTable:
    """The table a call writes: `out`, whose bound follows once the call is
    made, or a new one."""
    if out is pages:
        return pages
    if out is None:
        return PageTable(torch.empty_like(pages.table), torch.empty_like(pages.counts), torch.empty_like(pages.refs),
                         pages.page_tokens, pages.bound)
    _check_table(out, "out")
    if out.table.shape != pages.table.shape or out.refs.shape != pages.refs.shape \
            or out.page_tokens != pages.page_tokens:
        raise ValueError("out must have the page table's shape")
    both = ((out.table, pages.table), (out.counts, pages.counts), (out.refs, pages.refs))
    same = [a.data_ptr() == b.data_ptr() for a, b in both]
    if any(same) and not all(same):
        raise ValueError("out shares some of the page table's tensors: share all of them or none")
    if not any(same) and any(_overlap(a, b) for a, b in both):
        raise ValueError("out's tensors must not overlap the page table's")
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
    batch, width, count = _check_table(pages)
    _check_status(status)
    if bound is not None and bound > pages.capacity:
        raise RuntimeError("the page table has no entries left")
    each = 0
    if isinstance(tokens, torch.Tensor):
        tokens = _tokens(tokens, batch)
    else:
        each, tokens = min(int(tokens), pages.capacity + 1), None  # (more than fit are as good as one more)
        if each < 0:
            raise ValueError("tokens must not be negative")
    new = _new_table(pages, out)
    dev = _on_device(pages.table, pages.counts, pages.refs, tokens, status, new.table, new.counts, new.refs)
    nbytes = _workspace_bytes("popkv_page_reserve", batch, count)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_reserve", pages.table.data_ptr(), pages.counts.data_ptr(), pages.refs.data_ptr(),
                 new.table.data_ptr(), new.counts.data_ptr(), new.refs.data_ptr(), width, batch, count,
                 pages.page_tokens, nat.ptr(tokens), each, nat.ptr(status), ws.data_ptr(), nbytes, nat.stream_of(dev))
    new.bound = pages.bound
    return new


def write_tokens(cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor, v: torch.Tensor, *,
                 tokens: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Quantise new K/V rows ([B, KVH, rows, 128], any strides with contiguous
    rows, or [B, KVH, 128]: one row) of one layer into the sequences' pages:
    row t of sequence b becomes its token ``counts[b] + t``, for t <
    ``tokens[b]`` (int64 [B] on the device; None: all rows).  The pages come
    from ``reserve_pages``; a row without one is not written and sets
    ``status`` (bit 4, or bit 1 past the table's end)."""
    batch, _, kv_heads, pool = _check_cache(cache, pages, layer)
    _check_status(status)
    k, rows, *k_strides = _rows(k, batch, kv_heads, "new keys")
    v, v_rows, *v_strides = _rows(v, batch, kv_heads, "new values")
    if rows != v_rows or k.dtype != v.dtype:
        raise ValueError("new keys and values must share shape and dtype")
    if tokens is not None:
        tokens = _tokens(tokens, batch)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, k, v, tokens, status)
    with nat.on_device(dev):
        nat.call("popkv_paged_write", k.data_ptr(), v.data_ptr(), nat.dtype_code(k), *k_strides, *v_strides, rows,
                 nat.ptr(tokens), *pool, nat.ptr(status), nat.stream_of(dev))


def read_tokens(cache: PagedKVCache, layer: int, pages: PageTable, *, dtype: torch.dtype = torch.bfloat16,
                rows: int | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """One layer's cached rows as K, V [B, KVH, rows, 128] (``rows``: default
    ``pages.bound``).  Rows past a sequence's count are zero in new tensors and
    left as they are in ``out`` (two tensors that share no memory)."""
    batch, _, kv_heads, pool = _check_cache(cache, pages, layer)
    if out is None:
        rows = pages.bound if rows is None else int(rows)
        if rows < 0:
            raise ValueError("rows must not be negative")
        if dtype not in _FLOATS:
            raise RuntimeError(f"{dtype} is not supported; expected fp32/fp16/bf16")
        k = torch.empty((batch, kv_heads, rows, 128), dtype=dtype, device=cache.codes.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        if k.ndim != 4 or k.shape != (batch, kv_heads, k.shape[2], 128) or v.shape != k.shape or v.dtype != k.dtype \
                or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError(f"out must be two contiguous [{batch}, {kv_heads}, rows, 128] tensors")
        if rows is not None and rows != int(k.shape[2]):
            raise ValueError("rows must be out's row count")
        if _overlap(k, v):
            raise ValueError("out's two tensors must not overlap")
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, k, v)
    with nat.on_device(dev):
        nat.call("popkv_paged_read", k.data_ptr(), v.data_ptr(), nat.dtype_code(k), k.shape[2],
                 1 if out is None else 0, *pool, nat.stream_of(dev))
    return k, v


def _step_operands(q: torch.Tensor, batch: int, kv_heads: int, k: torch.Tensor, v: torch.Tensor,
                   out: torch.Tensor | None) -> tuple[int, int]:
    """Shapes and types of a step's operands: (query heads, dtype code)."""
    shape = q.shape
    if len(shape) != 3 or shape[0] != batch or shape[2] != 128:
        raise ValueError(f"q must be [{batch}, query heads, 128]")
    _, q_heads, _ = shape
    if q_heads <= 0 or q_heads % kv_heads != 0:
        raise ValueError("query heads must be a positive multiple of the KV heads")
    want = (batch, kv_heads, 128)
    if k.shape != want:
        raise ValueError(f"current k must be [{batch}, {kv_heads}, 128]")
    if v.shape != want:
        raise ValueError(f"current v must be [{batch}, {kv_heads}, 128]")
    dtype = q.dtype
    if out is not None:
        if out.shape != shape or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor shaped like q")
        if _overlap(out, q) or _overlap(out, k) or _overlap(out, v):  # (workgroups still read them)
            raise ValueError("out must not be one of the operands, nor overlap one")
    if k.dtype != dtype or v.dtype != dtype or (out is not None and out.dtype != dtype):
        raise RuntimeError("queries, current K/V and out must share a dtype")
    return q_heads, nat.dtype_code(q)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether contiguous `a` shares bytes with b (one with other strides is
    read through a copy: only its own first element counts)."""
    first, second = a.data_ptr(), b.data_ptr()
    if first == second:
        return a.numel() > 0 and b.numel() > 0
    return b.is_contiguous() and first < second + b.numel() * b.element_size() \
        and second < first + a.numel() * a.element_size()


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x contiguous and 16-byte aligned."""
    if not x.is_contiguous():
        return x.contiguous()  # (an allocation of its own)
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
    workspace holds merge tickets and split states: share it only with this
    module's attention calls, ordered on one stream.  It grows with the calls; a
    captured graph goes on using the buffer that it was captured with, so let
    the largest call come first, or keep a workspace for each graph.  ``out``
    shares no memory with the operands."""
    batch, width, kv_heads, pool = _check_cache(cache, pages, layer)
    q_heads, dtype = _step_operands(q, batch, kv_heads, k, v, out)
    if q_heads > 16 * kv_heads:
        raise ValueError("paged attention supports 1 to 16 query heads per KV head")
    most = pages.bound if max_tokens is None else int(max_tokens)
    if most < pages.bound:
        raise ValueError("max_tokens must cover the page table's bound")
    most = min(most, width * pages.page_tokens)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, q, k, v, out)
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    output = torch.empty_like(q) if out is None else out
    nbytes = _workspace_bytes("popkv_paged_attention", batch, q_heads, kv_heads, most)
    ws = (workspace or LayerStepWorkspace()).get(nbytes, dev, _TICKET_KIB)
    with nat.on_device(dev):
        nat.call("popkv_paged_attention", q.data_ptr(), dtype, *pool, most, k.data_ptr(), v.data_ptr(), q_heads,
                 output.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_of(dev))
    return output


def paged_indexed_attention(q: torch.Tensor, cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor,
                            v: torch.Tensor, indices: torch.Tensor, head_to_kv: torch.Tensor,
                            valid_mask: torch.Tensor | None = None, *, workspace: LayerStepWorkspace | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over selected tokens, the sparse layers' counterpart of
    ``paged_attention_step``: indices [B, QH, selected] (int64 or int32), the
    current token named by ``counts[b]``, as a retrieval returns them
    (``topk.select_with_current``, or, over its own 16-bit caches,
    ``batch.popkv_layer_step_batched(return_indices=True)``, whose -1 entries
    pad short rows).  Indices outside [0, counts[b]] and entries whose
    ``valid_mask`` is False are left out, an index named twice counts twice,
    and a row with nothing left is zero.  head_to_kv: [QH] KV head indices.
    The workspace and ``out`` as for ``paged_attention_step``."""
    batch, _, kv_heads, pool = _check_cache(cache, pages, layer)
    q_heads, dtype = _step_operands(q, batch, kv_heads, k, v, out)
    shape = indices.shape
    if len(shape) != 3 or shape[0] != batch or shape[1] != q_heads or shape[2] < 1:
        raise ValueError(f"indices must be [{batch}, {q_heads}, selected tokens]")
    if valid_mask is not None and valid_mask.shape != shape:
        raise ValueError("valid mask must match indices")
    if head_to_kv.ndim != 1 or head_to_kv.shape[0] != q_heads:
        raise ValueError(f"head_to_kv must be a vector of {q_heads} KV head indices")
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, q, k, v, out, indices, valid_mask)
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    idx = (indices if indices.dtype in _INDEX_CODES else indices.long()).contiguous()
    mask = None if valid_mask is None else valid_mask.to(torch.bool).contiguous().view(torch.uint8)
    if head_to_kv.dtype is not torch.int64 or head_to_kv.device != dev or not head_to_kv.is_contiguous():
        head_to_kv = head_to_kv.to(device=dev, dtype=torch.int64).contiguous()
    output = torch.empty_like(q) if out is None else out
    selected = shape[2]
    nbytes = _workspace_bytes("popkv_paged_indexed_attention", batch, q_heads, selected)
    ws = (workspace or LayerStepWorkspace()).get(nbytes, dev, _TICKET_KIB)
    with nat.on_device(dev):
        nat.call("popkv_paged_indexed_attention", q.data_ptr(), dtype, *pool, k.data_ptr(), v.data_ptr(),
                 idx.data_ptr(), _INDEX_CODES[idx.dtype], nat.ptr(mask), head_to_kv.data_ptr(), q_heads, selected,
                 output.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_of(dev))
    return output


def allocate_token_weights(cache: PagedKVCache, pages: PageTable) -> torch.Tensor:
    """What tokens have gathered, nothing yet: float32 [layers, B, KVH,
    ``pages.capacity``] for ``paged_chunk_attention`` and ``evict_tokens``.  After
    ``fork_sequences`` the children's are ``weights[:, parents]`` (zero for -1)."""
    return torch.zeros((cache.layers, pages.batch, cache.kv_heads, pages.capacity), dtype=torch.float32,
                       device=cache.codes.device)


def _span(x: torch.Tensor) -> tuple[int, int]:
    """The addresses from x's first byte to behind its last."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def _chunk_out(q: torch.Tensor, out: torch.Tensor | None, operands: tuple[torch.Tensor, ...]) -> torch.Tensor:
    """The tensor a chunk's rows go to: `out`, its rows contiguous, aligned, apart
    from each other and from the operands; or a new one laid out like q."""
    if out is None:
        out = torch.empty_like(q)  # (q's order of dimensions, where it has no gaps)
        return out if out.stride(3) == 1 else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape:
        raise ValueError("out must be shaped like q")
    if out.dtype != q.dtype:
        raise RuntimeError("queries, new K/V and out must share a dtype")
    if not out.numel():
        return out
    reach = 1
    for stride, n in sorted((s, n) for s, n in zip(out.stride(), out.shape) if n > 1):
        if stride < reach:
            raise ValueError("out's rows must not overlap")
        reach = stride * (n - 1) + reach
    unit = 16 // out.element_size()
    if out.stride(3) != 1 or out.data_ptr() % 16 or any(s % unit for s, n in zip(out.stride()[:3], out.shape) if n > 1):
        raise ValueError("out's rows must be contiguous and 16-byte aligned")
    first, last = _span(out)
    for x in operands:
        if x.numel():
            a, b = _span(x)
            if first < b and a < last:  # (workgroups still read them)
                raise ValueError("out must not be one of the operands, nor overlap one")
    return out


def paged_chunk_attention(q: torch.Tensor, cache: PagedKVCache, layer: int, pages: PageTable, k: torch.Tensor,
                          v: torch.Tensor, *, tokens: torch.Tensor | None = None,
                          weights: torch.Tensor | None = None, max_tokens: int | None = None,
                          workspace: LayerStepWorkspace | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a chunk of new tokens of one layer: q [B, QH, rows, 128], their
    k/v [B, KVH, rows, 128], not cached yet (any strides with contiguous rows) ->
    [B, QH, rows, 128].  Row t of sequence b, t < ``tokens[b]`` (int64 [B] on the
    device; None: all rows), attends over b's cached tokens and the chunk's tokens 0
    .. t; query head h reads KV head h // (QH / KVH).  Rows past ``tokens[b]`` are
    zero in a new tensor and left as they are in ``out``.  ``write_tokens`` and
    ``advance`` with the same ``tokens`` follow.  (Decoding sequences beside a long piece
    of a prompt are faster in a call of their own: the longest chunk sets the layout.)

    ``weights`` (contiguous float32 [B, KVH, ``pages.capacity``], a layer of
    ``allocate_token_weights``): every token's attention weight, summed over the rows
    and the query heads of its KV head, is added to its place, token t of the chunk at
    ``counts[b] + t``.  Every row counts that ``tokens`` holds, so give the accepted ones of
    proposals alone.  What tokens that are taken back later (``advance`` of a negative
    number) gathered stays at their places, which have to be cleared, and what their rows
    added to older tokens stays in those sums.

    Rounded are, for fp16 rows, cached values (to fp16); for bf16 rows also the weights
    (fp16 on cached tokens, bf16 on new ones) and, without ``weights``, cached keys, so that
    with ``weights`` a bf16 result has other bits.  The error's norm against float64: bf16
    1.6e-3 to 2.1e-3 (its own rounding 1.66e-3), fp16 2.0e-4 to 2.9e-4 (2.1e-4), float32 2e-7
    to 2.5e-6 with the logits' size, as plain float32 products.  New values beyond 2^90 may
    leave the range of the float32 sums.  One token of every sequence laid out as a decode
    step's, without ``tokens`` and ``weights``, is ``paged_attention_step``, to the bit.

    ``max_tokens`` and ``workspace`` as for ``paged_attention_step``.  The workspace takes up
    to 70 MB of partial states, and with ``weights`` 18 KB (float32 42 KB) more for every 32
    rows of a KV head: 39 MB for 2048 tokens of 32 heads, 89 MB in float32.  ``out`` shares no
    memory with the operands."""
    batch, width, kv_heads, pool = _check_cache(cache, pages, layer)
    shape = q.shape
    if len(shape) != 4 or shape[0] != batch or shape[3] != 128:
        raise ValueError(f"q must be [{batch}, query heads, rows, 128]")
    _, q_heads, rows, _ = shape
    if q_heads <= 0 or q_heads % kv_heads != 0:
        raise ValueError("query heads must be a positive multiple of the KV heads")
    want = (batch, kv_heads, rows, 128)
    if k.shape != want or v.shape != want:
        raise ValueError(f"new k and v must be {list(want)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("queries, new K/V and out must share a dtype")
    dtype = nat.dtype_code(q)
    if tokens is not None:
        tokens = _tokens(tokens, batch)
    most = pages.bound if max_tokens is None else int(max_tokens)
    if most < pages.bound:
        raise ValueError("max_tokens must cover the page table's bound")
    capacity = width * pages.page_tokens
    most = min(most, capacity)
    if weights is not None:
        if weights.shape != (batch, kv_heads, capacity) or weights.dtype is not torch.float32 \
                or not weights.is_contiguous():
            raise ValueError(f"weights must be a contiguous float32 [{batch}, {kv_heads}, {capacity}]")
        if any(_overlap(weights, x) for x in (q, k, v)) or (out is not None and _overlap(weights, out)):
            raise ValueError("weights must not overlap another operand")
    output = _chunk_out(q, out, (q, k, v))
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, q, k, v, tokens, weights, out)
    if rows == 0:
        return output
    q, _, *q_strides = _rows(q, batch, q_heads, "q")
    k, _, *k_strides = _rows(k, batch, kv_heads, "new keys")
    v, _, *v_strides = _rows(v, batch, kv_heads, "new values")
    nbytes = _workspace_bytes("popkv_paged_chunk_attention", dtype, batch, q_heads, kv_heads, rows, most,
                              0 if weights is None else 1)
    ws = (workspace or LayerStepWorkspace()).get(nbytes, dev, _TICKET_KIB)
    o_strides = [s if n > 1 else 0 for s, n in zip(output.stride()[:3], shape)]
    with nat.on_device(dev):
        nat.call("popkv_paged_chunk_attention", q.data_ptr(), dtype, *q_strides, k.data_ptr(), *k_strides, v.data_ptr(),
                 *v_strides, rows, nat.ptr(tokens), *pool, most, q_heads, output.data_ptr(), *o_strides,
                 1 if out is None else 0, nat.ptr(weights), capacity, ws.data_ptr(), ws.numel(), nat.stream_of(dev))
    return output


def evict_tokens(cache: PagedKVCache, pages: PageTable, weights: torch.Tensor, keep: int, *, recent: int = 0,
                 keeps: torch.Tensor | None = None, status: torch.Tensor | None = None,
                 out: PageTable | None = None, weights_out: torch.Tensor | None = None
                 ) -> tuple[PageTable, torch.Tensor, torch.Tensor]:
    """Sequences of more than ``keep`` tokens are cut to ``keep`` (``keeps``, int64 [B]
    on the device: to that many each, ``keep`` at most).  Every layer and KV head
    keeps the last ``recent`` tokens and, of the others, those of the largest
    ``weights`` (float32 [layers, B, KVH, ``pages.capacity``]; NaN is the largest, of
    equal ones the first is kept), in their order at the front of the sequence; the
    pages behind are given back, reserved ones too.  A page of the front that a fork
    shares is not written: a free one takes its place.  Free are the pages that were
    free before the call; those that it gives back serve the next one.  A sequence that
    needs more than are left (the ones behind it go on), or one of whose tokens' pages
    is missing, stays as it was and sets ``status`` bit 4.

    Returns the new page table (or ``out``, which may be ``pages``), the kept tokens'
    weights, zero behind them (or ``weights_out``, which may be ``weights``), and where
    each kept token was, int32 [layers, B, KVH, keep] (-1 past a sequence's share and
    for sequences that were not cut), for whoever holds more about the tokens.  The
    bound stays: once no ``status`` is set, it may be lowered to ``keep``.  The old
    table is spent.

    ``counts`` then say how many tokens are held, and no longer at which position the
    next one stands: a model whose keys carry positions (rotary ones) counts them itself.
    Kept keys stay as they were written."""
    batch, width, kv_heads, pool = _check_cache(cache, pages)
    _check_status(status)
    capacity = width * pages.page_tokens
    want = (cache.codes.shape[0], batch, kv_heads, capacity)
    for x in (weights, weights_out):
        if x is not None and (x.shape != want or x.dtype is not torch.float32 or not x.is_contiguous()):
            raise ValueError(f"weights must be a contiguous float32 {list(want)}")
    keep, recent = min(int(keep), capacity), min(int(recent), capacity)
    if keep < 0 or recent < 0:
        raise ValueError("keep and recent must not be negative")
    if keeps is not None and (keeps.shape != (batch,) or keeps.dtype is not torch.int64):
        raise ValueError(f"keeps must be an int64 [{batch}] tensor")
    if weights_out is not None and weights_out.data_ptr() != weights.data_ptr() and _overlap(weights_out, weights):
        raise ValueError("weights_out must be weights or not overlap them")
    new = _new_table(pages, out)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, pages.refs, weights, weights_out, keeps,
                     status, new.table, new.counts, new.refs)
    moved = torch.empty_like(weights) if weights_out is None else weights_out
    kept = torch.empty((*want[:3], keep), dtype=torch.int32, device=dev)
    if keeps is not None:
        keeps = keeps.contiguous()
    nbytes = _workspace_bytes("popkv_page_evict", batch, width, pool[2])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_evict", pool[0], pool[1], want[0], pool[2], kv_heads, pool[4], pool[5], pool[6], pool[8],
                 pages.refs.data_ptr(), new.table.data_ptr(), new.counts.data_ptr(), new.refs.data_ptr(), width, batch,
                 weights.data_ptr(), moved.data_ptr(), capacity, nat.ptr(keeps), keep, recent, kept.data_ptr(),
                 nat.ptr(status), ws.data_ptr(), nbytes, nat.stream_of(dev))
    new.bound = pages.bound
    return new, moved, kept


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
    ``pages``); the old one is spent: pages that its ended sequences gave back
    may hold other tokens already."""
    batch, width, kv_heads, pool = _check_cache(cache, pages)
    _check_status(status)
    if parents.shape != (batch,) or parents.dtype is not torch.int64:
        raise ValueError(f"parents must be an int64 [{batch}] tensor")
    new = _new_table(pages, out)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, pages.refs, parents, status, new.table,
                     new.counts, new.refs)
    parents = parents.contiguous()
    nbytes = _workspace_bytes("popkv_page_fork", batch, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_fork", pool[0], pool[1], cache.codes.shape[0], pool[2], kv_heads, pool[4], pool[5],
                 pool[6], pool[8], pages.refs.data_ptr(), new.table.data_ptr(), new.counts.data_ptr(),
                 new.refs.data_ptr(), width, batch, parents.data_ptr(), nat.ptr(status), ws.data_ptr(), nbytes,
                 nat.stream_of(dev))
    new.bound = pages.bound
    return new


def compact_pages(cache: PagedKVCache, pages: PageTable, *, out: PageTable | None = None
                  ) -> tuple[PageTable, torch.Tensor]:
    """The n live pages (refs > 0) to places 0 .. n - 1 of the pool, in every
    layer: those at n or later move, in order, to the free places before n.
    Returns the new page table (or ``out``, which may be ``pages``) and the
    int32 [pages] map of where each live page is now (-1: it was free), for
    whoever holds pages outside this table; the old table is spent."""
    batch, width, kv_heads, pool = _check_cache(cache, pages)
    new = _new_table(pages, out)
    dev = _on_device(cache.codes, cache.scales, pages.table, pages.counts, pages.refs, new.table, new.counts, new.refs)
    page_map = torch.empty_like(pages.refs)
    nbytes = _workspace_bytes("popkv_page_compact", pool[2])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with nat.on_device(dev):
        nat.call("popkv_page_compact", pool[0], pool[1], cache.codes.shape[0], pool[2], kv_heads, pool[4], pool[5],
                 pool[6], pool[8], pages.refs.data_ptr(), new.table.data_ptr(), new.counts.data_ptr(),
                 new.refs.data_ptr(), width, batch, page_map.data_ptr(), ws.data_ptr(), nbytes, nat.stream_of(dev))
    new.bound = pages.bound
    return new, page_map
