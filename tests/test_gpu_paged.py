"""The paged 4-bit K/V cache against plain float64: rows written and read back,
dense and indexed attention over the pages, the pages' bookkeeping, and a
decode loop of all of them together."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from popkv_amd import paged, popkv, popkv_cuda, topk

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# one unit in the last place of the output type: its rounding, and a neighbour
# where the fp32 result sits on a tie
ULP = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}
# fp32 sums and exponentials of logits up to about 30 in magnitude: relative
# error about 30 * 2^-23 of values up to about 5 (as for the dense layer)
FP32 = 4e-5


# ---------------------------------------------------------------- the format, in float64

def quantise(x: np.ndarray, group: int):
    """x float64 [..., 128] -> codes [..., 128] (0 .. 15), low, delta float16 [..., R]."""
    g = x.reshape(*x.shape[:-1], 128 // group, group)
    bad = ~np.isfinite(g).all(-1)
    safe = np.where(bad[..., None], 0.0, g)
    low = np.clip(safe.min(-1), -57344, 57344).astype(np.float32).astype(np.float16)
    top = np.clip(safe.max(-1), -57344, 57344)
    delta = ((top - low.astype(np.float64)) / 15).astype(np.float32).astype(np.float16)
    step = np.where(delta == 0, 1.0, delta.astype(np.float64))[..., None]
    code = np.clip(np.rint((safe - low.astype(np.float64)[..., None]) / step), 0, 15)
    code = np.where((bad | (delta == 0))[..., None], 0, code)
    low = np.where(bad, np.float16("nan"), low)
    delta = np.where(bad, np.float16(0), delta)
    return code.reshape(x.shape).astype(np.uint8), low, delta


def values(code, low, delta):
    group = 128 // low.shape[-1]
    low, delta = (np.repeat(t.astype(np.float64), group, -1) for t in (low, delta))
    return low + code * delta


def dequantised(x: torch.Tensor, group: int) -> torch.Tensor:
    return torch.from_numpy(values(*quantise(x.double().cpu().numpy(), group)))


def unpack(cache: paged.PagedKVCache):
    c = cache.codes.cpu().numpy()
    s = cache.scales.cpu().numpy()
    return np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], 128), s[..., 0], s[..., 1]


def make(lengths, kv_heads, *, group=32, page=64, layers=1, spare=3, max_tokens=None, seed=0, poison=True):
    """A pool and table whose sequences may hold `lengths` tokens, pages
    scattered; unwritten content is NaN scales and set bits."""
    most = max_tokens or max(max(lengths), 1)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    cache = paged.allocate_paged_cache(layers, pages, kv_heads, page_tokens=page, dim_group_size=group, device=DEV)
    if poison:
        cache.codes.fill_(0xA5)
        cache.scales.fill_(float("nan"))
    table = paged.PageTable.create(len(lengths), most, cache)
    order = np.random.default_rng(seed).permutation(pages)
    at = 0
    for b, n in enumerate(need):
        table.table[b, :n] = torch.from_numpy(order[at:at + n].astype(np.int32)).to(DEV)
        at += n
    table.refs[torch.from_numpy(order[:at]).to(DEV)] = 1
    return cache, table


def fill(cache, table, layer, lengths, gen, dtype=torch.float32, scale=1.0):
    """Writes `lengths` random rows; returns the float64 K, V that the pages stand for."""
    rows = max(max(lengths), 1)
    shape = (len(lengths), cache.kv_heads, rows, 128)
    k, v = (torch.randn(shape, generator=gen).to(dtype) * scale for _ in range(2))
    tokens = torch.tensor(lengths, dtype=torch.int64, device=DEV)
    paged.write_tokens(cache, layer, table, k.to(DEV), v.to(DEV), tokens=tokens)
    return dequantised(k, cache.dim_group_size), dequantised(v, cache.dim_group_size)


# ---------------------------------------------------------------- write, read

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("page,cached,new", [(32, [0], [1]), (64, [0, 63, 64], [1, 1, 1]), (32, [5, 0, 31], [70, 0, 1]),
                                             (256, [300, 17], [1, 515]), (128, [1], [127])])
def test_written_rows_are_the_formats(dtype, group, page, cached, new):
    """Codes and scales bit for bit, every other row of the pool untouched,
    and the rows read back."""
    gen = torch.Generator().manual_seed(page + len(new))
    total = [a + b for a, b in zip(cached, new)]
    cache, table = make(total, 3, group=group, page=page, layers=2)
    table.counts.copy_(torch.tensor(cached))
    rows = max(new)
    k = (torch.randn(len(new), rows, 3, 128, generator=gen) * 3).to(dtype).to(DEV).transpose(1, 2)  # strided heads
    v = torch.randn(len(new), 3, rows, 128, generator=gen).to(dtype).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = [x.copy() for x in unpack(cache)]
    tab = table.table.cpu().numpy()
    for which, x in enumerate((k, v)):
        code, low, delta = quantise(x.double().cpu().numpy(), group)
        for b, n in enumerate(new):
            for t in range(n):
                at = cached[b] + t
                where = (1, tab[b, at // page], slice(None), at % page, which)
                want[0][where], want[1][where], want[2][where] = code[b, :, t], low[b, :, t], delta[b, :, t]
    paged.write_tokens(cache, 1, table, k, v, tokens=torch.tensor(new, device=DEV), status=status)
    got = unpack(cache)
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1], equal_nan=True) and np.array_equal(got[2], want[2], equal_nan=True)
    assert int(status) == 0
    table.advance(torch.tensor(new, device=DEV), bound=max(total))
    mark = 7.0
    outs = tuple(torch.full((len(new), 3, max(total) + 2, 128), mark, dtype=dtype, device=DEV) for _ in range(2))
    paged.read_tokens(cache, 1, table, out=outs)
    fresh = paged.read_tokens(cache, 1, table, dtype=dtype)
    for x, out, one in zip((k, v), outs, fresh):
        for b, n in enumerate(new):
            exact = dequantised(x[b, :, :n], group)
            got = out[b, :, cached[b]:total[b]].cpu()
            # fp32 holds low + code * delta with one rounding; then the type's
            assert torch.equal(got, exact.float().to(dtype))
            assert torch.equal(one[b, :, cached[b]:total[b]].cpu(), got)
            assert (out[b, :, total[b]:] == mark).all() and (one[b, :, total[b]:] == 0).all()


@pytest.mark.parametrize("group", (16, 32, 64))
def test_values_at_the_borders_of_codes(group):
    """Halfway between two codes and the fp32 neighbours of those: the exact
    quotient decides, ties to even."""
    rng = np.random.default_rng(group)
    x = np.zeros((64, 128), np.float32)
    for t in range(64):
        low, delta = np.float16(rng.normal() * 3), np.float16(rng.uniform(1e-3, 2.0))
        for g in range(128 // group):
            half = np.float64(low) + (rng.integers(0, 15, group) + 0.5) * np.float64(delta)
            row = half.astype(np.float32)
            row = np.nextafter(row, rng.choice([-np.inf, np.inf], group).astype(np.float32)) if t % 2 else row
            row[0], row[1] = low, np.float32(np.float64(low) + 15 * np.float64(delta))
            x[t, g * group:(g + 1) * group] = row
    cache, table = make([64], 1, group=group)
    rows = torch.from_numpy(x)[None, None].to(DEV)
    paged.write_tokens(cache, 0, table, rows, rows)
    code, low, delta = quantise(x.astype(np.float64), group)
    got = unpack(cache)
    page = int(table.table[0, 0])
    for which in (0, 1):
        assert np.array_equal(got[0][0, page, 0, :64, which], code)
        assert np.array_equal(got[1][0, page, 0, :64, which], low)
        assert np.array_equal(got[2][0, page, 0, :64, which], delta)


def test_extreme_rows():
    """Constants, zeros, tiny and huge values, and groups with a NaN or an
    infinity (NaN when read back, their neighbours whole)."""
    x = torch.randn(12, 128, generator=torch.Generator().manual_seed(1))
    x[0] = 0.0
    x[1] = -2.5
    x[2] *= 1e-9
    x[3] *= 1e30
    x[4] = 57344.0
    x[5, :64], x[5, 64:] = -57344.0, 65000.0
    x[6, 3] = float("nan")
    x[7, 40] = float("inf")
    x[8, 100] = float("-inf")
    x[9, 127] = 1e38
    x[10] = 1e-40
    x[11] *= 1e-5
    cache, table = make([12], 1)
    paged.write_tokens(cache, 0, table, x[None, None].to(DEV), x[None, None].to(DEV))
    table.advance(12)
    want = dequantised(x, 32)
    for out in paged.read_tokens(cache, 0, table, dtype=torch.float32):
        got = out[0, 0].cpu()
        assert torch.equal(got.isnan(), want.isnan()) and want.isnan().sum() == 3 * 32
        assert torch.equal(got.nan_to_num(), want.nan_to_num().float())


def test_rows_without_a_page():
    """A missing page, a page outside the pool and rows past the table write
    nothing, set their bits and read back as zeros."""
    cache, table = make([64, 64, 64], 2, page=32, spare=0)
    before = (cache.codes.clone(), cache.scales.clone())
    table.table[0, 0] = -1
    table.table[1, 1] = cache.pages
    table.counts.copy_(torch.tensor([0, 40, 64]))
    rows = torch.randn(3, 2, 8, 128, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for tokens, bits in (([8, 0, 0], 4), ([0, 8, 0], 4), ([0, 0, 8], 1)):
        status.zero_()
        paged.write_tokens(cache, 0, table, rows, rows, tokens=torch.tensor(tokens, device=DEV), status=status)
        assert int(status) == bits
    assert torch.equal(cache.codes, before[0]) and torch.equal(cache.scales.view(torch.int16), before[1].view(torch.int16))
    table.counts.copy_(torch.tensor([32, 0, 0]))
    table.bound = 32
    k, v = paged.read_tokens(cache, 0, table)
    assert not k.any() and not v.any()


def test_single_token_rows_and_negative_counts():
    """[B, KVH, 128] is one row; a negative device count is taken as zero."""
    cache, table = make([1, 1], 2)
    x = torch.randn(2, 2, 128, device=DEV)
    table.counts.fill_(-5)
    paged.write_tokens(cache, 0, table, x, -x)
    table.counts.fill_(1)
    k, v = paged.read_tokens(cache, 0, table, dtype=torch.float32, rows=1)
    want = dequantised(x, 32).float()
    assert torch.equal(k[:, :, 0].cpu(), want)
    assert torch.equal(v[:, :, 0].cpu(), dequantised(-x, 32).float())


def test_a_pool_past_32_bit_offsets():
    """Pages whose bytes lie beyond 2^32 of the layer's pool."""
    pages = 17_000  # 256 KiB of codes each: 4.4 GB
    cache = paged.allocate_paged_cache(1, pages, 8, page_tokens=256, dim_group_size=64, device=DEV)
    table = paged.PageTable.create(1, 512, cache)
    table.table.copy_(torch.tensor([[pages - 1, pages - 300]]))
    gen = torch.Generator().manual_seed(2)
    k, v = fill(cache, table, 0, [300], gen)
    table.advance(300)
    q, ck, cv = (torch.randn(1, n, 128, generator=gen).to(DEV) for n in (8, 8, 8))
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv)
    want = attend(q, k, v, ck, cv, [300])
    assert (got.cpu().double() - want).abs().max() < FP32
    idx = torch.arange(301, device=DEV).expand(1, 8, 301).contiguous()
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(8, device=DEV))
    assert (got.cpu().double() - want).abs().max() < FP32
    # and moved from there to the front
    new, page_map = paged.compact_pages(cache, table_with_refs(table))
    assert new.table.tolist() == [[1, 0]] and int(page_map[pages - 1]) == 1
    assert torch.equal(paged.paged_attention_step(q, cache, 0, new, ck, cv).cpu(),
                       paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu())


def table_with_refs(table):
    held = table.table[table.table >= 0].long()
    table.refs.zero_()
    table.refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    return table


# ---------------------------------------------------------------- attention

def attend(q, k, v, ck, cv, lengths, pick=None, head_to_kv=None):
    """float64 attention [B, QH, 128]; pick[b][h]: the token numbers (the
    current one named by its count), default all."""
    q, ck, cv = (t.cpu().double() for t in (q, ck, cv))
    out = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // ck.shape[1]
    for b, n in enumerate(lengths):
        for h in range(q.shape[1]):
            g = h // group if head_to_kv is None else int(head_to_kv[h])
            keys, vals = torch.cat([k[b, g, :n], ck[b, g, None]]), torch.cat([v[b, g, :n], cv[b, g, None]])
            if pick is not None:
                rows = torch.tensor(pick[b][h], dtype=torch.long)
                if not len(rows):
                    continue
                keys, vals = keys[rows], vals[rows]
            out[b, h] = torch.softmax(keys @ q[b, h] / math.sqrt(128), 0) @ vals
    return out


def allowed(want, dtype, q, k, v, ck, cv):
    """Largest error per element of the 16-bit dense kernel: the output's
    rounding, the fp32 work, and K, V and the weights rounded to fp16 (half a
    step, 2^-11 of the value): a logit is off by at most 2^-11 sum|q k| /
    sqrt(128), the weights by twice that in proportion, and each of V's and the
    weights' roundings by 2^-11 of the largest value."""
    bound = ULP[dtype] * want.abs() + FP32
    if dtype == torch.float32:
        return bound
    group = q.shape[1] // ck.shape[1]
    q = q.cpu().double().abs()
    keys = torch.cat([k, ck.cpu().double()[:, :, None]], 2).abs().amax(2)  # [B, KVH, 128]
    logit = 2.0 ** -11 * (q * keys.repeat_interleave(group, 1)).sum(-1, keepdim=True) / math.sqrt(128)
    top = torch.cat([v, cv.cpu().double()[:, :, None]], 2).abs().amax((2, 3)).repeat_interleave(group, 1)[..., None]
    return bound + top * (2 * logit + 2 * 2.0 ** -11)


LENGTHS = [[0], [1], [31, 32, 33], [64, 0, 65, 1], [255, 256, 257], [300] * 9, [4097, 20, 0, 1500], [20011]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (2, 2), (3, 2), (4, 2), (7, 1), (8, 2), (16, 1)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_dense_attention(dtype, group, kv_heads, lengths):
    """No token, tile and page edges, splits of several sequences, more query
    heads than a wave's rows; one workspace used twice with equal bits."""
    dims, page = (16, 32, 64)[len(lengths) % 3], (32, 64, 128, 256)[group % 4]
    gen = torch.Generator().manual_seed(sum(lengths) + group)
    cache, table = make(lengths, kv_heads, group=dims, page=page, max_tokens=max(lengths) + 1)
    k, v = fill(cache, table, 0, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
    q = (torch.randn(len(lengths), kv_heads * group, 128, generator=gen) * 2).to(dtype).to(DEV)
    ck, cv = (torch.randn(len(lengths), kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    ws = popkv.LayerStepWorkspace()
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws)
    want = attend(q, k, v, ck, cv, lengths)
    err = (got.cpu().double() - want).abs()
    bound = allowed(want, dtype, q, k, v, ck, cv)
    assert (err <= bound).all(), float((err / bound).max())
    assert torch.equal(paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws), got)
    # a looser launch bound cuts other splits: the same result to rounding
    loose = paged.paged_attention_step(q, cache, 0, table, ck, cv, max_tokens=max(lengths) + 5000)
    assert ((loose.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_attention_of_large_batches(dtype):
    """More sequences than a wave has lanes, most of them empty or short."""
    lengths = [(i * 37) % 90 if i % 3 else 0 for i in range(150)]
    gen = torch.Generator().manual_seed(3)
    cache, table = make(lengths, 1, page=32)
    k, v = fill(cache, table, 0, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
    q = torch.randn(150, 2, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = (torch.randn(150, 1, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want = attend(q, k, v, ck, cv, lengths)
    err = (paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double() - want).abs()
    assert (err <= allowed(want, dtype, q, k, v, ck, cv)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_attention_leaves_out_what_has_no_page(dtype):
    """A dropped page (an evicted window) and a page outside the pool."""
    gen = torch.Generator().manual_seed(4)
    cache, table = make([200, 130], 2)
    k, v = fill(cache, table, 0, [200, 130], gen)
    table.advance(torch.tensor([200, 130], device=DEV), bound=200)
    table.table[0, 0], table.table[1, 1] = -1, cache.pages + 5
    q = torch.randn(2, 8, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = (torch.randn(2, 2, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    pick = [[list(range(64, 201))] * 8, [list(range(64)) + [128, 129, 130]] * 8]
    want = attend(q, k, v, ck, cv, [200, 130], pick)
    err = (paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double() - want).abs()
    assert (err <= allowed(want, dtype, q, k, v, ck, cv)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (1, 4, 16))
@pytest.mark.parametrize("first,last", [(0, 1), (0, 32), (96, 700), (0, 700)])
def test_dense_attention_keeps_nan(dtype, group, first, last):
    """NaN keys or values in live rows of one KV head: NaN in its group's
    outputs, none elsewhere."""
    gen = torch.Generator().manual_seed(first + last)
    cache, table = make([700], 2)
    k = torch.randn(1, 2, 700, 128, generator=gen)
    v = torch.randn(1, 2, 700, 128, generator=gen)
    k[0, 1, first:last, 5] = float("nan")
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(700)
    q = torch.randn(1, 2 * group, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = (torch.randn(1, 2, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv)
    assert got[0, group:].isnan().all() and not got[0, :group].isnan().any()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_dense_attention_of_large_and_small_queries(dtype):
    """Query magnitudes outside fp16's range, and rows of very different
    magnitudes in one group (bf16 and fp32 hold them)."""
    gen = torch.Generator().manual_seed(6)
    cache, table = make([500], 1)
    k, v = fill(cache, table, 0, [500], gen, scale=1e-2)
    table.advance(500)
    q = torch.randn(1, 4, 128, generator=gen)
    q[0, 1] *= 1e5
    q[0, 2] *= 1e-12
    q[0, 3, ::2] *= 1e-6
    k2 = k.clone()
    q = q.to(dtype).to(DEV)
    ck, cv = (torch.randn(1, 1, 128, generator=gen).to(dtype).to(DEV) * 1e-2 for _ in range(2))
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double()
    want = attend(q, k2, v, ck, cv, [500])
    bound = allowed(want, dtype, q, k, v, ck, cv)
    # row 1's logits reach thousands: fp32 keeps them to 2^-22 of their size
    size = (q.cpu().double().abs() * k.abs().amax(2)).sum(-1, keepdim=True) / math.sqrt(128)
    bound = bound + 2 * size * 2.0 ** -22 * v.abs().max()
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 64))
@pytest.mark.parametrize("scale", (1e-2, 1e-3, 1e-4))
def test_attention_over_small_values(dtype, group, scale):
    """Keys and values whose scales, and the parts they are split in, lie among
    fp16's subnormals: the format's own values, no worse."""
    gen = torch.Generator().manual_seed(30)
    cache, table = make([900], 2, group=group)
    k, v = fill(cache, table, 0, [900], gen, scale=scale)
    table.advance(900)
    q = torch.randn(1, 8, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = ((torch.randn(1, 2, 128, generator=gen) * scale).to(dtype).to(DEV) for _ in range(2))
    want = attend(q, k, v, ck, cv, [900])
    # the type's step (or a subnormal's), the fp32 work on values of this size,
    # and for bf16 V and the weights in fp16: half a step of the largest value
    # each, or half of fp16's least
    bound = ULP[dtype] * want.abs() + FP32 * scale + (2.0 ** -24 if dtype == torch.float16 else 0)
    if dtype == torch.bfloat16:
        bound = bound + v.abs().max() * 2 * 2.0 ** -11 + 2.0 ** -25
    err = (paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    idx = torch.arange(901, device=DEV).expand(1, 8, 901).contiguous()
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(8, device=DEV) // 4)
    bound = ULP[dtype] * want.abs() + FP32 * scale + (2.0 ** -24 if dtype == torch.float16 else 0)
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_strided_and_unaligned_operands():
    """Queries, current rows, indices and rows to write as views, at odd offsets;
    `out` given."""
    gen = torch.Generator().manual_seed(31)
    cache, table = make([100, 60], 2)
    raw = torch.randn(2, 2, 100, 131, generator=gen).to(torch.bfloat16).to(DEV)
    rows_k, rows_v = raw[..., 1:129], raw[..., 3:131]  # rows neither contiguous nor aligned
    paged.write_tokens(cache, 0, table, rows_k, rows_v, tokens=torch.tensor([100, 60], device=DEV))
    table.advance(torch.tensor([100, 60], device=DEV), bound=100)
    k, v = dequantised(rows_k, 32), dequantised(rows_v, 32)
    q = torch.randn(8, 2, 129, generator=gen).to(DEV).transpose(0, 1)[..., 1:]
    c = torch.randn(2, 2, 2, 129, generator=gen).to(DEV)[..., 1:]
    ck, cv = c[0], c[1]
    out = torch.full((2, 8, 128), float("nan"), device=DEV)
    want = attend(q, k, v, ck, cv, [100, 60])
    assert paged.paged_attention_step(q, cache, 0, table, ck, cv, out=out) is out
    assert ((out.cpu().double() - want).abs() <= ULP[torch.float32] * want.abs() + FP32).all()
    idx = torch.arange(202, device=DEV).view(1, 1, 202).expand(2, 8, 202)[..., ::2]  # every second token
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(8) // 4, idx >= 0,
                                        out=out.view(2, 8, 128))
    want = attend(q, k, v, ck, cv, [100, 60], [[list(range(0, 101, 2))] * 8, [list(range(0, 61, 2))] * 8])
    assert ((got.cpu().double() - want).abs() <= ULP[torch.float32] * want.abs() + FP32).all()


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_counts_past_the_launch_bound(dtype):
    """A device count above max_tokens is taken as max_tokens, one past the
    table as the table's capacity, a negative one as zero."""
    gen = torch.Generator().manual_seed(32)
    cache, table = make([96, 96, 96], 1, page=32)
    k, v = fill(cache, table, 0, [96, 96, 96], gen)
    table.counts.copy_(torch.tensor([90, 10 ** 12, -4]))
    table.bound = 70
    q, ck, cv = (torch.randn(3, n, 128, generator=gen).to(dtype).to(DEV) for n in (2, 1, 1))
    for most, lengths in ((70, [70, 70, 0]), (96, [90, 96, 0])):
        want = attend(q, k, v, ck, cv, lengths)
        got = paged.paged_attention_step(q, cache, 0, table, ck, cv, max_tokens=most)
        assert ((got.cpu().double() - want).abs() <= allowed(want, dtype, q, k, v, ck, cv)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", (torch.int64, torch.int32))
@pytest.mark.parametrize("lengths,selected,kv_heads,group", [([700, 33, 0], 1, 2, 4), ([700, 33, 0], 129, 2, 4),
                                                             ([1000], 900, 1, 3), ([64] * 5, 64, 3, 1),
                                                             ([5000, 4000], 2500, 2, 8),
                                                             ([300, 0, 90, 400, 33] * 2, 400, 4, 4)])
def test_indexed_attention(dtype, index, lengths, selected, kv_heads, group):
    """Selections with padding, masked entries, repeats, the current token
    never, once and twice, numbers outside the sequence, and rows that keep
    nothing (zero)."""
    gen = torch.Generator().manual_seed(selected)
    dims, page = (16, 32, 64)[selected % 3], (32, 64, 128)[group % 3]
    cache, table = make(lengths, kv_heads, group=dims, page=page, max_tokens=max(lengths) + 1)
    k, v = fill(cache, table, 0, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
    qh, batch = kv_heads * group, len(lengths)
    idx = torch.randint(-2, max(lengths) + 3, (batch, qh, selected), generator=gen)
    for b, n in enumerate(lengths):
        idx[b, 0, ::5] = n
        idx[b, -1] = -1
        idx[b, -1, : selected // 2] = n + 1
    mask = torch.rand(idx.shape, generator=gen) < 0.8
    head_to_kv = torch.randint(0, kv_heads, (qh,), generator=gen)
    q = (torch.randn(batch, qh, 128, generator=gen) * 2).to(dtype).to(DEV)
    ck, cv = (torch.randn(batch, kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    ws = popkv.LayerStepWorkspace()
    for m in (None, mask):
        pick = [[[int(t) for e, t in enumerate(idx[b, h]) if 0 <= t <= n and (m is None or m[b, h, e])]
                 for h in range(qh)] for b, n in enumerate(lengths)]
        want = attend(q, k, v, ck, cv, lengths, pick, head_to_kv)
        args = (q, cache, 0, table, ck, cv, idx.to(index).to(DEV), head_to_kv.to(DEV), None if m is None else m.to(DEV))
        got = paged.paged_indexed_attention(*args, workspace=ws)
        err = (got.cpu().double() - want).abs()
        assert (err <= ULP[dtype] * want.abs() + FP32).all(), float(err.max())
        assert not got[:, -1].any()
        assert torch.equal(paged.paged_indexed_attention(*args, workspace=ws), got)


def test_indexed_attention_skips_missing_pages_and_keeps_nan():
    gen = torch.Generator().manual_seed(8)
    cache, table = make([256], 1, group=16)
    k = torch.randn(1, 1, 256, 128, generator=gen)
    v = torch.randn(1, 1, 256, 128, generator=gen)
    k[0, 0, 200, 7] = float("nan")
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(256)
    table.table[0, 1] = -1
    q, ck, cv = (torch.randn(1, n, 128, generator=gen).to(DEV) for n in (2, 1, 1))
    idx = torch.tensor([[[3, 64, 127, 10], [3, 200, 1, 256]]], device=DEV)
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.zeros(2, dtype=torch.int64, device=DEV))
    want = attend(q, dequantised(k, 16), dequantised(v, 16), ck, cv, [256], [[[3, 10], [3]]])
    assert ((got[0, 0].cpu().double() - want[0, 0]).abs() <= ULP[torch.float32] * want[0, 0].abs() + FP32).all()
    assert got[0, 1].isnan().all()


@pytest.mark.parametrize("group", (1, 4))
def test_one_workspace_for_both_attentions(group):
    """Dense and indexed calls of different sizes in turn on one workspace, the
    counts of their rows equal (one query head per KV head) or not."""
    gen = torch.Generator().manual_seed(20 + group)
    ws = popkv.LayerStepWorkspace()
    work = []
    for lengths in ([9000], [700, 40], [3, 0], [20000]):
        kv_heads, batch = 4 // len(lengths), len(lengths)  # batch * KVH is the same
        cache, table = make(lengths, kv_heads, max_tokens=max(lengths) + 1)
        k, v = fill(cache, table, 0, lengths, gen)
        table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
        q = torch.randn(batch, kv_heads * group, 128, generator=gen).to(DEV)
        ck, cv = (torch.randn(batch, kv_heads, 128, generator=gen).to(DEV) for _ in range(2))
        idx = torch.arange(max(lengths) + 1, device=DEV).expand(batch, kv_heads * group, -1).contiguous()
        work.append((q, cache, table, ck, cv, idx, torch.arange(kv_heads * group, device=DEV) // group,
                     attend(q, k, v, ck, cv, lengths)))
    for _ in range(3):
        for q, cache, table, ck, cv, idx, mapping, want in work:
            for got in (paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws),
                        paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, mapping, workspace=ws),
                        paged.paged_attention_step(q.half(), cache, 0, table, ck.half(), cv.half(), workspace=ws)):
                scale = 1 if got.dtype == torch.float32 else 200  # fp16 inputs: 2^-11 of queries, keys and values
                assert ((got.cpu().double() - want).abs() <= scale * FP32).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,group,lengths", [(1, 16, [8200]), (1, 8, [66000]), (2, 3, [33000]), (4, 1, [20000, 9000]),
                                                    (1, 4, [256 * 8 * 32 - 1]), (1, 1, [256 * 8 * 32 + 33])])
def test_dense_attention_merge_levels(dtype, kv_heads, group, lengths):
    """33 and more parts merge in two levels (sets of 16, the last one short),
    up to the 256 of one KV head; equal bits from the same workspace again,
    tickets back at zero."""
    gen = torch.Generator().manual_seed(group)
    cache, table = make(lengths, kv_heads, page=128)
    k, v = fill(cache, table, 0, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
    batch = len(lengths)
    q = (torch.randn(batch, kv_heads * group, 128, generator=gen) * 2).to(dtype).to(DEV)
    ck, cv = (torch.randn(batch, kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    ws = popkv.LayerStepWorkspace()
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws)
    want = attend(q, k, v, ck, cv, lengths)
    assert ((got.cpu().double() - want).abs() <= allowed(want, dtype, q, k, v, ck, cv)).all()
    assert torch.equal(paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws), got)
    assert not ws.buffer[:batch * kv_heads * 128].any()


# ---------------------------------------------------------------- pages

class Book:
    """The page table's rules in plain Python."""

    def __init__(self, table, counts, refs, page):
        self.table, self.counts, self.refs, self.page = [list(r) for r in table], list(counts), list(refs), page
        self.status = 0

    def free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def reserve(self, tokens):
        free, at = self.free(), 0
        for b, row in enumerate(self.table):
            n, more = self.counts[b], max(tokens[b], 0)
            if n + more > len(row) * self.page:
                self.status |= 1
                continue
            holes = [i for i in range(n // self.page, -(-(n + more) // self.page)) if row[i] < 0]
            if at + len(holes) > len(free):
                self.status |= 4 if holes else 0
            else:
                for i, p in zip(holes, free[at:]):
                    row[i] = p
                    self.refs[p] = 1
            at += len(holes)

    def fork(self, parents):
        old, counts = [list(r) for r in self.table], list(self.counts)
        moves, need = [], []
        for b, p in enumerate(parents):
            if not 0 <= p < len(old):
                self.status |= 8 if p != -1 else 0
                row, n = [-1] * len(old[b]), 0
            else:
                n, full = counts[p], counts[p] // self.page
                row = list(old[p])
                if p in parents[:b]:
                    row = row[:full] + [-1] * (len(row) - full)
                    if n % self.page and old[p][full] >= 0:
                        need.append((b, full, old[p][full]))
            for page, by in [(x, -1) for x in old[b]] + [(x, 1) for x in row]:
                if page >= 0:
                    self.refs[page] += by
            self.table[b], self.counts[b] = row, n
        free = self.free()
        for i, (b, full, source) in enumerate(need):
            if i < len(free):
                self.table[b][full] = free[i]
                self.refs[free[i]] = 1
                moves.append((source, free[i]))
            else:
                for page in self.table[b]:
                    if page >= 0:
                        self.refs[page] -= 1
                self.table[b], self.counts[b] = [-1] * len(old[b]), 0
                self.status |= 4
        return moves

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] == 0]
        moves = list(zip([p for p in live if p >= n], holes))
        where = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        for source, target in moves:
            where[source] = target
            self.refs[target], self.refs[source] = self.refs[source], 0
        self.table = [[where[p] if p >= 0 else p for p in row] for row in self.table]
        return moves, where


def random_pages(seed, batch, width, page, spare, layers=2, kv_heads=2, group=32):
    """A pool of random bytes and a table with shared full pages and pages
    reserved ahead."""
    rng = np.random.default_rng(seed)
    counts = [int(rng.integers(0, max(1, (width - 1) * page))) if rng.random() < 0.8 else 0 for _ in range(batch)]
    held = [-(-n // page) + (int(rng.integers(0, 2)) if n else 0) for n in counts]
    pages = max(1, sum(held) + spare)  # a pool holds one page at least
    order = [int(p) for p in rng.permutation(pages)]
    table, refs, at = [], [0] * pages, 0
    for b, n in enumerate(held):
        row = order[at:at + n] + [-1] * (width - n)
        if b and rng.random() < 0.4:  # shares the first full pages of an earlier one
            other = int(rng.integers(0, b))
            for i in range(min(counts[b], counts[other]) // page):
                row[i] = table[other][i]
        at += n
        table.append(row)
        for p in row:
            if p >= 0:
                refs[p] += 1
    cache = paged.allocate_paged_cache(layers, pages, kv_heads, page_tokens=page, dim_group_size=group, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cache.codes.random_(0, 256, generator=gen)
    cache.scales.copy_(torch.rand(cache.scales.shape, generator=gen, device=DEV))
    dev = paged.PageTable(torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(counts, device=DEV),
                          torch.tensor(refs, dtype=torch.int32, device=DEV), page, max(counts))
    return cache, dev, Book(table, counts, refs, page)


def same_book(pages, book):
    assert pages.table.tolist() == book.table
    assert pages.counts.tolist() == book.counts
    assert pages.refs.tolist() == book.refs


def moved(pool, moves):
    want = pool.clone()
    for source, target in moves:
        want[:, target] = pool[:, source]
    return want


SHAPES = [(0, 1, 1, 32, 0), (1, 1, 4, 64, 2), (2, 5, 6, 32, 40), (3, 33, 9, 64, 7), (4, 130, 20, 128, 300),
          (5, 7, 70, 32, 2000), (6, 1100, 2, 32, 500), (7, 40, 500, 32, 9000)]


@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("seed,batch,width,page,spare", SHAPES)
def test_reserve(seed, batch, width, page, spare, in_place):
    """One token, prompts, none at all, more than the table or the pool
    holds; counts unchanged, the input untouched unless it is the output."""
    cache, pages, book = random_pages(seed, batch, width, page, spare)
    rng = np.random.default_rng(seed)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    many = [int(x) for x in rng.integers(-1, width * page, batch)]
    for tokens in (1, 0, many, [3 * page] * batch, [2 ** 40] * batch):
        book.reserve(tokens if isinstance(tokens, list) else [tokens] * batch)
        was = [t.clone() for t in (pages.table, pages.counts, pages.refs)]
        arg = torch.tensor(tokens, device=DEV) if isinstance(tokens, list) else tokens
        new = paged.reserve_pages(pages, arg, status=status, out=pages if in_place else None)
        assert (new is pages) == in_place
        if not in_place:
            assert all(torch.equal(a, b) for a, b in zip(was, (pages.table, pages.counts, pages.refs)))
        pages = new
        same_book(pages, book)
        assert int(status) == book.status


@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("seed,batch,width,page,spare", SHAPES)
def test_fork(seed, batch, width, page, spare, in_place):
    """Kept, permuted, forked and freed sequences, several times over, and
    parents outside the batch; every page of every layer."""
    cache, pages, book = random_pages(seed, batch, width, page, spare)
    rng = np.random.default_rng(seed + 1)
    pages.refs[-1:] += 1  # a page that the program holds by itself
    book.refs[-1] += 1
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for parents in (list(range(batch)), [int(x) for x in rng.permutation(batch)],
                    [int(x) for x in rng.integers(-1, batch, batch)], [0] * batch,
                    [int(x) for x in rng.integers(-3, batch + 3, batch)], [-1] * batch):
        codes, scales = cache.codes.clone(), cache.scales.clone()
        moves = book.fork(parents)
        pages = paged.fork_sequences(cache, pages, torch.tensor(parents, device=DEV), status=status,
                                     out=pages if in_place else None)
        same_book(pages, book)
        assert int(status) == book.status
        assert torch.equal(cache.codes, moved(codes, moves)) and torch.equal(cache.scales, moved(scales, moves))


@pytest.mark.parametrize("free", (0, 1, 2))
def test_fork_with_few_free_pages(free):
    """Children that find no page are left empty; the others are whole."""
    table = [[0, 1, 2, 3, -1], [-1] * 5, [-1] * 5, [4, -1, -1, -1, -1], [-1] * 5, [5, -1, -1, -1, -1]]
    counts, refs = [101, 0, 0, 20, 0, 32], [1] * 6 + [0] * free
    cache, _, _ = random_pages(9, 6, 5, 32, 0)
    cache = paged.PagedKVCache(cache.codes[:, :6 + free].contiguous(), cache.scales[:, :6 + free].contiguous(), 32)
    pages = paged.PageTable(torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(counts, device=DEV),
                            torch.tensor(refs, dtype=torch.int32, device=DEV), 32, 101)
    book = Book(table, counts, refs, 32)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    codes = cache.codes.clone()
    keep = [0, 0, 0, 3, 0, 5]
    moves = book.fork(keep)
    new = paged.fork_sequences(cache, pages, torch.tensor(keep, device=DEV), status=status)
    same_book(new, book)
    assert new.counts.tolist() == [101] * (1 + free) + [0] * (2 - free) + [20, 0, 32]
    assert int(status) == book.status == 4
    assert torch.equal(cache.codes, moved(codes, moves))


@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("seed,batch,width,page,spare", SHAPES)
def test_compact(seed, batch, width, page, spare, in_place):
    cache, pages, book = random_pages(seed, batch, width, page, spare, layers=3, kv_heads=1, group=16)
    codes, scales = cache.codes.clone(), cache.scales.clone()
    moves, where = book.compact()
    new, page_map = paged.compact_pages(cache, pages, out=pages if in_place else None)
    same_book(new, book)
    assert page_map.tolist() == where
    assert torch.equal(cache.codes, moved(codes, moves)) and torch.equal(cache.scales, moved(scales, moves))
    # nothing is left to move
    again, page_map = paged.compact_pages(cache, new)
    same_book(again, book)
    assert torch.equal(cache.codes, moved(codes, moves))


@pytest.mark.parametrize("spare", (65530, 70001, 140000))
def test_pools_of_several_parts(spare):
    """Pools past the 65536 pages that a plan maps at once: pages reserved,
    forked and compacted across the parts."""
    cache, pages, book = random_pages(21, 12, 9, 32, spare, layers=1, kv_heads=1, group=64)
    rng = np.random.default_rng(spare)
    used = rng.random(cache.pages) < 0.5
    extra = torch.from_numpy(used.astype(np.int32)).to(DEV)  # pages that others hold
    pages.refs += extra
    book.refs = pages.refs.tolist()
    tokens = [int(x) for x in rng.integers(0, 100, 12)]
    book.reserve(tokens)
    pages = paged.reserve_pages(pages, torch.tensor(tokens, device=DEV))
    same_book(pages, book)
    # the lowest free pages lie past the first part
    pages.refs[:66000] += 1
    book.refs = pages.refs.tolist()
    codes = cache.codes.clone()
    parents = [0, 0, 0, 3, 3, -1, 6, 7, 8, 8, 8, 11]
    codes = moved(codes, book.fork(parents))
    pages = paged.fork_sequences(cache, pages, torch.tensor(parents, device=DEV))
    same_book(pages, book)
    assert torch.equal(cache.codes, codes)
    pages.refs[:66000] -= 1
    book.refs = pages.refs.tolist()
    moves, where = book.compact()
    pages, page_map = paged.compact_pages(cache, pages)
    same_book(pages, book)
    assert page_map.tolist() == where and torch.equal(cache.codes, moved(codes, moves))


def test_compact_of_empty_and_full_pools():
    cache, pages, book = random_pages(11, 3, 4, 64, 5)
    for value in (0, 1):
        pages.refs.fill_(value)
        pages.table.fill_(-1)
        codes = cache.codes.clone()
        new, page_map = paged.compact_pages(cache, pages)
        assert torch.equal(cache.codes, codes) and torch.equal(new.refs, pages.refs)
        assert page_map.tolist() == (list(range(cache.pages)) if value else [-1] * cache.pages)


# ---------------------------------------------------------------- together

class Plain:
    """The sequences of a batch as float64 rows of every layer."""

    def __init__(self, batch, layers, kv_heads, group):
        self.group = group
        self.rows = [[torch.zeros(2, kv_heads, 0, 128, dtype=torch.float64) for _ in range(layers)] for _ in range(batch)]

    def write(self, layer, k, v, tokens):
        for b, n in enumerate(tokens):
            new = torch.stack((dequantised(k[b, :, :n], self.group), dequantised(v[b, :, :n], self.group)))
            self.rows[b][layer] = torch.cat((self.rows[b][layer], new), 2)

    def fork(self, parents):
        empty = [r[:, :, :0] for r in self.rows[0]]
        self.rows = [[r.clone() for r in self.rows[p]] if p >= 0 else list(empty) for p in parents]

    def attend(self, layer, q, ck, cv):
        out = []
        for b in range(len(self.rows)):
            k, v = self.rows[b][layer]
            out.append(attend(q[b:b + 1], k[None], v[None], ck[b:b + 1], cv[b:b + 1], [k.shape[1]])[0])
        return torch.stack(out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_decode_loop_of_all_of_them(dtype):
    """Prompts of different lengths, decode steps across page borders, beams
    forked and ended, the pool compacted, a new prompt in a freed place, and
    the sequences read back: against float64 rows at every step."""
    layers, kv_heads, group, batch = 2, 2, 4, 4
    gen = torch.Generator().manual_seed(12)
    cache = paged.allocate_paged_cache(layers, 40, kv_heads, page_tokens=32, dim_group_size=32, device=DEV)
    pages = paged.PageTable.create(batch, 256, cache)
    plain = Plain(batch, layers, kv_heads, 32)
    ws = popkv.LayerStepWorkspace()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    counts = [0] * batch

    def admit(tokens):
        t = torch.tensor(tokens, device=DEV)
        paged.reserve_pages(pages, t, status=status, out=pages)
        for layer in range(layers):
            k, v = (torch.randn(batch, kv_heads, max(tokens), 128, generator=gen).to(dtype) for _ in range(2))
            paged.write_tokens(cache, layer, pages, k.to(DEV), v.to(DEV), tokens=t, status=status)
            plain.write(layer, k, v, tokens)
        for b, n in enumerate(tokens):
            counts[b] += n
        pages.advance(t, bound=max(counts))

    def step():
        paged.reserve_pages(pages, 1, status=status, out=pages)
        for layer in range(layers):
            q = torch.randn(batch, kv_heads * group, 128, generator=gen).to(dtype).to(DEV)
            k, v = (torch.randn(batch, kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
            got = paged.paged_attention_step(q, cache, layer, pages, k, v, workspace=ws)
            every = torch.arange(pages.bound + 1, device=DEV).expand(batch, kv_heads * group, -1).contiguous()
            picked = paged.paged_indexed_attention(q, cache, layer, pages, k, v, every,
                                                   torch.arange(kv_heads * group, device=DEV) // group)
            want = plain.attend(layer, q, k, v)
            # values up to 5, logits a few: fp16 roundings of K, V and weights (2^-11 each) and the type's
            bound = ULP[dtype] * want.abs() + (FP32 if dtype == torch.float32 else 5 * 8 * 2.0 ** -11)
            assert ((got.cpu().double() - want).abs() <= bound).all()
            assert ((picked.cpu().double() - want).abs() <= ULP[dtype] * want.abs() + FP32).all()
            paged.write_tokens(cache, layer, pages, k, v, status=status)
            plain.write(layer, k.cpu()[:, :, None], v.cpu()[:, :, None], [1] * batch)
        pages.advance()
        for b in range(batch):
            counts[b] += 1

    def fork(parents):
        paged.fork_sequences(cache, pages, torch.tensor(parents, device=DEV), status=status, out=pages)
        plain.fork(parents)
        counts[:] = [counts[p] if p >= 0 else 0 for p in parents]
        assert pages.counts.tolist() == counts

    admit([70, 0, 31, 64])
    for _ in range(3):
        step()
    fork([0, 0, 2, 0])
    step()
    fork([3, 1, 1, -1])
    for _ in range(2):
        step()
    paged.compact_pages(cache, pages, out=pages)
    live = int((pages.refs > 0).sum())
    assert (pages.refs[:live] > 0).all() and not pages.refs[live:].any()
    admit([0, 33, 0, 40])
    for _ in range(30):
        step()
    assert int(status) == 0
    held = pages.table[pages.table >= 0].long()
    assert torch.equal(torch.bincount(held, minlength=cache.pages).int(), pages.refs)
    for layer in range(layers):
        k, v = paged.read_tokens(cache, layer, pages, dtype=torch.float32)
        for b, n in enumerate(counts):
            assert torch.equal(k[b, :, :n].cpu(), plain.rows[b][layer][0].float())
            assert torch.equal(v[b, :, :n].cpu(), plain.rows[b][layer][1].float())
    fork([-1] * batch)
    assert not pages.refs.any() and (pages.table == -1).all()


def test_a_captured_decode_step():
    """Reserve, attend, select, write and advance captured once and replayed
    across page borders, with eager work on other tensors in between; a fork
    and a compaction replayed as well."""
    batch, kv_heads, group = 3, 2, 4
    gen = torch.Generator().manual_seed(13)
    mapping = torch.arange(kv_heads * group, device=DEV) // group

    def start():
        cache, table = make([60, 31, 0], kv_heads, page=32, spare=30, max_tokens=160, poison=False)
        fill(cache, table, 0, [60, 31, 0], torch.Generator().manual_seed(14), dtype=torch.bfloat16)
        table.advance(torch.tensor([60, 31, 0], device=DEV), bound=60)
        return cache, table

    cache, table = start()
    other, plain = start()
    q = torch.zeros(batch, kv_heads * group, 128, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(batch, kv_heads, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    idx = torch.zeros(batch, kv_heads * group, 20, dtype=torch.int64, device=DEV)
    parents = torch.arange(batch, device=DEV)
    dense, picked = torch.zeros_like(q), torch.zeros_like(q)
    ws, ws2 = popkv.LayerStepWorkspace(), popkv.LayerStepWorkspace()

    def step(cache, table, ws, ws2):
        paged.reserve_pages(table, 1, out=table)
        paged.paged_attention_step(q, cache, 0, table, k, v, max_tokens=120, workspace=ws, out=dense)
        paged.paged_indexed_attention(q, cache, 0, table, k, v, idx, mapping, workspace=ws2, out=picked)
        paged.write_tokens(cache, 0, table, k, v)
        table.counts.add_(1)
        paged.fork_sequences(cache, table, parents, out=table)
        paged.compact_pages(cache, table, out=table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spare_cache, spare = start()
        step(spare_cache, spare, ws, ws2)  # the workspaces take their size outside the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, table, ws, ws2)
    for i in range(40):
        q.copy_(torch.randn(q.shape, generator=gen))
        k.copy_(torch.randn(k.shape, generator=gen))
        v.copy_(torch.randn(v.shape, generator=gen))
        idx.copy_(torch.randint(-1, 32, idx.shape, generator=gen))
        parents.copy_(torch.tensor([0, 1, 2] if i % 7 else [1, 1, 0]))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (dense, picked)]
        step(other, plain, popkv.LayerStepWorkspace(), popkv.LayerStepWorkspace())
        assert torch.equal(dense, got[0]) and torch.equal(picked, got[1])
        assert torch.equal(table.table, plain.table) and torch.equal(table.counts, plain.counts)
        assert torch.equal(table.refs, plain.refs)
    assert torch.equal(cache.codes, other.codes)


def test_captured_calls_of_different_rows_share_a_workspace():
    """Graphs of dense and indexed calls with 2, 8 and 24 rows, captured on one
    workspace one after the other and replayed in turns: each finds its tickets
    zero whatever states the others left.  Equal bits with a workspace alone."""
    gen = torch.Generator().manual_seed(41)
    calls = []
    for lengths, kv_heads, group in (([20000], 2, 4), ([9000, 700, 5000], 2, 4)):
        cache, table = make(lengths, kv_heads, max_tokens=max(lengths) + 1)
        fill(cache, table, 0, lengths, gen)
        table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
        batch, qh = len(lengths), kv_heads * group
        q, ck, cv = (torch.randn(batch, n, 128, generator=gen).to(DEV) for n in (qh, kv_heads, kv_heads))
        idx = torch.randint(0, 700, (batch, qh, 3000), generator=gen).to(DEV)
        mapping = torch.arange(qh, device=DEV) // group
        calls.append(lambda out, ws, a=(q, cache, 0, table, ck, cv): paged.paged_attention_step(*a, workspace=ws, out=out))
        calls.append(lambda out, ws, a=(q, cache, 0, table, ck, cv, idx, mapping):
                     paged.paged_indexed_attention(*a, workspace=ws, out=out))
    shapes = [(1, 8, 128)] * 2 + [(3, 8, 128)] * 2
    want = [torch.empty(s, device=DEV) for s in shapes]
    out = [torch.empty(s, device=DEV) for s in shapes]
    ws = popkv.LayerStepWorkspace()
    for call, x, y in zip(calls, want, out):
        call(x, popkv.LayerStepWorkspace())
    for call, y in list(zip(calls, out)) * 2:  # the workspace takes its size
        call(y, ws)
    buffer = ws.buffer
    graphs = []
    for call, y in zip(calls, out):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(y, ws)
    assert ws.buffer is buffer
    for i in (0, 3, 1, 2, 0, 1, 3, 2, 2, 0, 3, 1, 0):
        out[i].fill_(float("nan"))
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(out[i], want[i]), i
        j = (i + 1) % 4
        out[j].fill_(float("nan"))
        calls[j](out[j], ws)  # and eager calls between the replays
        assert torch.equal(out[j], want[j]), j


def test_two_streams_at_once():
    """Two batches on two streams, each with its own workspace."""
    gen = torch.Generator().manual_seed(15)
    work = []
    for i in range(2):
        cache, table = make([900 + i, 400], 2)
        k, v = fill(cache, table, 0, [900 + i, 400], gen)
        table.advance(torch.tensor([900 + i, 400], device=DEV), bound=900 + i)
        q, ck, cv = (torch.randn(2, n, 128, generator=gen).to(DEV) for n in (8, 2, 2))
        work.append((cache, table, q, ck, cv, attend(q, k, v, ck, cv, [900 + i, 400]), popkv.LayerStepWorkspace()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for s, (cache, table, q, ck, cv, _, ws), out in zip(streams, work, outs):
            with torch.cuda.stream(s):
                out.append(paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws))
    torch.cuda.synchronize()
    for out, w in zip(outs, work):
        for x in out:
            assert ((x.cpu().double() - w[5]).abs() <= ULP[torch.float32] * w[5].abs() + FP32).all()


def test_a_retrieval_step_over_the_pages():
    """The sparse layer's operations -- encode, score, select -- with the
    attention over the 4-bit pages in the place of the 16-bit prefix."""
    gen = torch.Generator().manual_seed(16)
    kv_heads, group, tokens, budget = 2, 4, 1500, 257
    keys = torch.randn(kv_heads, tokens, 128, generator=gen).to(torch.bfloat16).to(DEV)
    vals = torch.randn(kv_heads, tokens, 128, generator=gen).to(torch.bfloat16).to(DEV)
    meta = popkv.build_popkv_cache(keys, group_size=64, dim_group_size=64, reserve_tokens=1)
    cache, table = make([tokens], kv_heads, group=32)
    paged.write_tokens(cache, 0, table, keys[None], vals[None])
    table.advance(tokens)
    q = torch.randn(kv_heads * group, 128, generator=gen).to(torch.bfloat16).to(DEV)
    ck, cv = (torch.randn(kv_heads, 128, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    mapping = torch.arange(kv_heads * group, device=DEV) // group
    enc = popkv_cuda.query_encode(q[None], dim_group_size=64)
    scores = popkv_cuda.score_encoded(enc, meta.packed, head_to_kv=mapping, tokens=tokens, dim_group_size=64)
    idx = topk.select_with_current(scores, budget - 1, tokens + 1)
    got = paged.paged_indexed_attention(q[None], cache, 0, table, ck[None], cv[None], idx[None], mapping)
    want = attend(q[None], dequantised(keys, 32)[None], dequantised(vals, 32)[None], ck[None], cv[None], [tokens],
                  [[row.tolist() for row in idx.cpu()]])
    assert ((got.cpu().double() - want).abs() <= ULP[torch.bfloat16] * want.abs() + FP32).all()


# ---------------------------------------------------------------- wide value groups

def wide_values(limit, dtype, gen, tokens, every):
    """V rows [1, 2, tokens, 128]; every `every`-th token's groups span +-limit."""
    v = torch.randn(1, 2, tokens, 128, generator=gen)
    wide = (torch.rand(1, 2, tokens, 128, generator=gen) * 2 - 1) * limit
    wide[..., 0::16], wide[..., 1::16] = -limit, limit
    far = torch.arange(tokens) % every == every - 1
    return torch.where(far[:, None], wide, v).to(dtype), far


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("limit", (34000.0, 57344.0))
@pytest.mark.parametrize("weights", ("all", "none"))
def test_attention_over_wide_value_groups(dtype, group, limit, weights):
    """Value groups up to the format's whole range (15 delta past fp16's largest
    number), in tokens that count like any other and in tokens whose weight is
    2^-40 and less, which change nothing."""
    gen = torch.Generator().manual_seed(50 + group)
    cache, table = make([300], 2, group=group)
    v, far = wide_values(limit, dtype, gen, 300, 1 if weights == "all" else 9)
    base = torch.randn(128, generator=gen)
    k = torch.randn(1, 2, 300, 128, generator=gen)
    if weights == "none":  # logits below -30
        k[:, :, far] = -4 * base
    k = k.to(dtype)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(300)
    k, v = dequantised(k, group), dequantised(v, group)
    q = (base + 0.1 * torch.randn(1, 8, 128, generator=gen)).to(dtype).to(DEV)
    ck, cv = (torch.randn(1, 2, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want = attend(q, k, v, ck, cv, [300])
    # the output's rounding; the fp32 work (FP32 is that of values up to about
    # 5); the wide tokens' own weights, below 2^-40 of 57344 each; and for the
    # dense bf16 form V and the weights in fp16, half a step of the largest each
    top = v.abs().max() if weights == "all" else v[:, :, ~far].abs().max()
    bound = ULP[dtype] * want.abs() + FP32 * top / 5 + 300 * 57344 * 2.0 ** -40
    half = bound + (2 * 2.0 ** -11 * top if dtype == torch.bfloat16 else 0)
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double()
    assert ((got - want).abs() <= half).all(), float((got - want).abs().max())
    idx = torch.arange(301, device=DEV).expand(1, 8, 301).contiguous()
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(8, device=DEV) // 4)
    assert ((got.cpu().double() - want).abs() <= bound).all(), float((got.cpu().double() - want).abs().max())


# ---------------------------------------------------------------- what the logits may lose

def outlier_rows(shape, gen):
    """K rows with four channels per KV head ten times as large."""
    x = torch.randn(shape, generator=gen)
    for h in range(shape[1]):
        x[:, h, :, torch.randperm(128, generator=gen)[:4]] *= 10
    return x


def logit_steps(q, k, group, kv_heads, n):
    """Of the dense kernel's sums for a logit, over the magnitudes that pass
    through them: [B, QH, n], in logits.  S = sum_g (low + 8 delta) qsum + sum_g
    delta (q . (c - 8))."""
    code, low, delta = (torch.from_numpy(t.astype(np.float64)) for t in quantise(k[:, :, :n].double().numpy(), group))
    per = q.shape[1] // kv_heads
    q = q.cpu().double()
    out = torch.zeros(q.shape[0], q.shape[1], n, dtype=torch.float64)
    for h in range(q.shape[1]):
        g = h // per
        part = q[:, h].unflatten(-1, (-1, group))  # [B, R, G]
        apart = torch.einsum("brg,bnrg->bnr", part.abs(), (code[:, g].unflatten(-1, (-1, group)) - 8).abs())
        first = ((low[:, g].abs() + 8 * delta[:, g]) * part.sum(-1).abs()[:, None]).sum(-1)
        out[:, h] = first + (delta[:, g] * apart).sum(-1)
    return out / math.sqrt(128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("kind", ("mean", "sign"))
def test_dense_logits_keep_what_fp32_sums_keep(dtype, group, kind):
    """Queries that do not average out over keys with outlier channels: the
    results' distance from float64 is that of the type's own rounding and of a
    few fp32 roundings of what the sums hold, in the norm."""
    gen = torch.Generator().manual_seed(60 + group)
    tokens = 3001
    cache, table = make([tokens], 2, group=group)
    k, v = outlier_rows((1, 2, tokens, 128), gen), torch.randn(1, 2, tokens, 128, generator=gen)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(tokens)
    q = torch.randn(1, 32, 128, generator=gen) * 1.5
    q = (q + 1.5 if kind == "mean" else q.abs()).to(dtype).to(DEV)
    ck, cv = (torch.randn(1, 2, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    keys, vals = dequantised(k, group), dequantised(v, group)
    want = attend(q, keys, vals, ck, cv, [tokens])
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double()
    # a logit's error: a step of fp32 (2^-23) of all that its sums hold, and of
    # the logit itself for its scaling and its exponential
    steps = logit_steps(q, k, group, 2, tokens)
    work = torch.zeros_like(want)
    for h in range(32):
        g = h // 16
        rows = torch.cat([keys[0, g], ck[0, g, None].cpu().double()])
        logit = rows @ q[0, h].cpu().double() / math.sqrt(128)
        p = torch.softmax(logit, 0)[:tokens]
        e = 2.0 ** -23 * (steps[0, h] + 2 * logit[:tokens].abs() + 8)
        if dtype == torch.bfloat16:  # V and the weights in fp16: half a step each, uniform
            e = torch.sqrt(e * e + 2 * (2.0 ** -11) ** 2 / 3)
        # errors of different tokens are independent: they add in the square
        work[0, h] = torch.sqrt(((p * e) ** 2) @ (vals[0, g].abs() + want[0, h].abs()) ** 2)
    rounding = (want.to(dtype).double() - want).norm()
    allowed_norm = torch.sqrt(rounding ** 2 + work.norm() ** 2)
    # (of 4096 elements, the cross term of rounding and work is within four of
    # its deviations, 4 / sqrt(4096))
    assert (got - want).norm() <= (1 + 4 / 64) * allowed_norm, float((got - want).norm() / allowed_norm)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    """No rows to write, and the rows of a table that holds none yet."""
    cache, table = make([64, 64], 3)
    before = cache.codes.clone()
    none = torch.empty(2, 3, 0, 128, dtype=dtype, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged.write_tokens(cache, 0, table, none, none, status=status)
    paged.write_tokens(cache, 0, table, none, none, tokens=torch.tensor([3, 0], device=DEV), status=status)
    assert int(status) == 0 and torch.equal(cache.codes, before)
    for k, v in (paged.read_tokens(cache, 0, table, dtype=dtype), paged.read_tokens(cache, 0, table, dtype=dtype, rows=0),
                 paged.read_tokens(cache, 0, table, out=(none, none.clone()))):
        assert tuple(k.shape) == tuple(v.shape) == (2, 3, 0, 128) and k.dtype == v.dtype == dtype


@pytest.mark.parametrize("batch", (256, 257, 264))
def test_captured_calls_of_many_rows_share_a_workspace(batch):
    """2048 rows (sequences times KV heads), 2056 and 2112, the last sequences in
    several parts, captured once; a call of few rows leaves its states in the
    workspace between the replays."""
    gen = torch.Generator().manual_seed(70)
    lengths = [i % 3 for i in range(batch - 3)] + [20000, 0, 30000]

    def case(lengths, kv_heads):
        cache, table = make(lengths, kv_heads, page=32, max_tokens=max(lengths) + 1, poison=False)
        cache.codes.random_(0, 256)
        cache.scales.uniform_(-1, 1)
        table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
        q, ck, cv = (torch.randn(len(lengths), kv_heads, 128, generator=gen).to(DEV) for _ in range(3))
        return lambda out, ws: paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws, out=out)

    many, few = case(lengths, 8), case([20000], 8)
    want, out, small = (torch.empty(n, 8, 128, device=DEV) for n in (batch, batch, 1))
    many(want, popkv.LayerStepWorkspace())
    ws = popkv.LayerStepWorkspace()
    many(out, ws)
    buffer = ws.buffer
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        many(out, ws)
    for _ in range(3):
        few(small, ws)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert ws.buffer is buffer and torch.equal(out, want)
    few(small, ws)
    many(out, ws)  # and without a graph
    assert torch.equal(out, want)


@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("seed,batch,width,page,spare", SHAPES)
def test_reserve_where_an_entry_is_no_page(seed, batch, width, page, spare, in_place):
    """An entry outside the pool is no page, as -1 is: a reservation fills it."""
    cache, pages, book = random_pages(seed, batch, width, page, spare)
    rng = np.random.default_rng(seed + 3)
    outside = [cache.pages, cache.pages + 7, 2 ** 31 - 1, -1, -5, -2 ** 31]
    for b in range(batch):  # from the next token's page on: nothing holds what lies there but the row itself
        for i in range(book.counts[b] // page, width):
            if book.table[b][i] < 0 or rng.random() < 0.3:
                if book.table[b][i] >= 0:
                    book.refs[book.table[b][i]] -= 1
                pages.table[b, i] = outside[int(rng.integers(len(outside)))]
                book.table[b][i] = -1
    pages.refs.copy_(torch.tensor(book.refs, dtype=torch.int32))
    left = pages.table.cpu()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    many = [int(x) for x in rng.integers(0, width * page, batch)]
    for tokens in ([1] * batch, many):
        book.reserve(tokens)
        pages = paged.reserve_pages(pages, torch.tensor(tokens, device=DEV), status=status,
                                    out=pages if in_place else None)
        got, want = pages.table.cpu(), torch.tensor(book.table)
        # what no token asked for is left as it was
        assert torch.equal(got, torch.where(want < 0, left, want.int()))
        assert pages.refs.tolist() == book.refs and pages.counts.tolist() == book.counts
        assert int(status) == book.status


def test_the_bound_is_the_programs():
    """Replays move the counts and not the host's bound: eager calls see the
    new tokens once the program has set it, and it may lower it as well."""
    gen = torch.Generator().manual_seed(80)
    cache, table = make([64, 30], 2, page=32, max_tokens=96)
    rows = torch.randn(2, 2, 64, 128, generator=gen).to(DEV)
    step = torch.zeros(2, 2, 1, 128, device=DEV)

    def call():
        paged.write_tokens(cache, 0, table, step, step)
        table.advance()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (compiles nothing: the first use of the kernels outside the capture)
        paged.write_tokens(cache, 0, table, step, step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    table.bound = 0
    for t in range(30):
        step.copy_(rows[:, :, t:t + 1])
        graph.replay()
    assert table.counts.tolist() == [30, 30] and table.bound == 0
    table.bound = 30
    want = dequantised(rows[:, :, :30], 32)
    for x in paged.read_tokens(cache, 0, table, dtype=torch.float32):
        assert torch.equal(x.cpu(), want.float())
    q, ck, cv = (torch.randn(2, 2, 128, generator=gen).to(DEV) for _ in range(3))
    for most, lengths in ((30, [30, 30]), (12, [12, 12])):
        table.bound = most
        want = attend(q, dequantised(rows, 32), dequantised(rows, 32), ck, cv, lengths)
        got = paged.paged_attention_step(q, cache, 0, table, ck, cv)
        assert ((got.cpu().double() - want).abs() <= ULP[torch.float32] * want.abs() + FP32).all()


# ---------------------------------------------------------------- bounds that a wrong sum breaks

def near(want, dtype, q, k, v, ck, cv, group, lengths):
    """Largest error per element of the dense kernel on K, V rows (as written):
    a logit's sums pass at most sixteen fp32 steps (2^-23) of the magnitudes they
    hold, its scaling and exponential four of itself and sixteen of one; the sums
    over the tokens 64 steps of what they hold (|low| + 16 delta); bf16 V and
    weights half an fp16 step each, and no weight is off by more than 2^-33 of the
    largest; then the result's own rounding."""
    kv_heads = ck.shape[1]
    per = q.shape[1] // kv_heads
    bound = torch.zeros_like(want)
    for b, n in enumerate(lengths):
        steps = logit_steps(q[b:b + 1], k[b:b + 1], group, kv_heads, n)[0]
        for g in range(kv_heads):
            keys = torch.cat([dequantised(k[b, g, :n], group), ck[b, g, None].cpu().double()])
            vals = torch.cat([dequantised(v[b, g, :n], group), cv[b, g, None].cpu().double()]).abs()
            _, low, delta = quantise(v[b, g, :n].double().numpy(), group)
            held = np.repeat(np.abs(low.astype(np.float64)) + 16 * delta.astype(np.float64), group, -1)
            held = torch.cat([torch.from_numpy(held.reshape(n, 128)), vals[n:]])
            for h in range(g * per, g * per + per):
                logit = keys @ q[b, h].cpu().double() / math.sqrt(128)
                p = torch.softmax(logit, 0)
                e = 2.0 ** -23 * (16 * torch.cat([steps[h], logit[n:].abs()]) + 4 * logit.abs() + 16)
                bound[b, h] = (p * e) @ (vals + want[b, h].abs()) + 64 * 2.0 ** -23 * (p @ held)
                if dtype == torch.bfloat16:
                    bound[b, h] += 2 * 2.0 ** -11 * (p @ vals) + n * 2.0 ** -33 * vals.max()
    half = torch.finfo(dtype).eps / 2
    return half * (want.abs() + bound) + bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("kv_heads,per,lengths", [(1, 16, [8200]), (2, 3, [20011]), (1, 8, [66000]), (1, 1, [65569]),
                                                  (4, 1, [4097, 33, 1, 1500]), (3, 2, [300] * 9)])
def test_dense_attention_to_its_bound(dtype, group, kv_heads, per, lengths):
    """Long sequences, merges in two levels and ragged batches against bounds
    that neither zeros nor half of the tokens would pass."""
    gen = torch.Generator().manual_seed(90 + group + per)
    cache, table = make(lengths, kv_heads, group=group, max_tokens=max(lengths) + 1)
    batch = len(lengths)
    k, v = (torch.randn(batch, kv_heads, max(lengths), 128, generator=gen) for _ in range(2))
    count = torch.tensor(lengths, device=DEV)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV), tokens=count)
    table.advance(count, bound=max(lengths))
    q = (torch.randn(batch, kv_heads * per, 128, generator=gen) * 2).to(dtype).to(DEV)
    ck, cv = (torch.randn(batch, kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    keys, vals = dequantised(k, group), dequantised(v, group)
    want = attend(q, keys, vals, ck, cv, lengths)
    bound = near(want, dtype, q, k, v, ck, cv, group, lengths)
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
    half = attend(q, keys, vals, ck, cv, [n // 2 for n in lengths])
    for wrong in (torch.zeros_like(want), half):
        assert ((wrong - want).abs() > bound).double().mean() > 0.9


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("first,last", [(0, 1), (96, 700), (0, 700)])
def test_attention_keeps_nan_values(dtype, group, first, last):
    """NaN values in live rows of one KV head: NaN in the dims of their scale
    group for that KV head's queries, none elsewhere."""
    gen = torch.Generator().manual_seed(first + last + group)
    cache, table = make([700], 2, group=group)
    k, v = (torch.randn(1, 2, 700, 128, generator=gen) for _ in range(2))
    v[0, 1, first:last, 70] = float("nan")
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(700)
    q = torch.randn(1, 8, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = (torch.randn(1, 2, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    idx = torch.arange(701, device=DEV).expand(1, 8, 701).contiguous()
    want = torch.zeros(8, 128, dtype=torch.bool)
    want[4:, 70 // group * group:(70 // group + 1) * group] = True
    for got in (paged.paged_attention_step(q, cache, 0, table, ck, cv),
                paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(8, device=DEV) // 4)):
        assert torch.equal(got[0].isnan().cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_queries_beside_a_large_one(dtype):
    """A head's largest query element is 2^14 times the others, and the keys
    make up for it: no query element loses bits to the largest."""
    gen = torch.Generator().manual_seed(95)
    group, tokens = 16, 400
    cache, table = make([tokens], 2, group=group)
    k, v = torch.randn(1, 2, tokens, 128, generator=gen) * 6e3, torch.randn(1, 2, tokens, 128, generator=gen)
    k[..., :group] = 0  # (the large element's group)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(tokens)
    q = torch.randn(1, 8, 128, generator=gen) * 1e-3
    q[..., 0] = 16.0
    q = q.to(dtype).to(DEV)
    ck = torch.zeros(1, 2, 128, dtype=dtype, device=DEV)
    cv = torch.randn(1, 2, 128, generator=gen).to(dtype).to(DEV)
    keys, vals = dequantised(k, group), dequantised(v, group)
    want = attend(q, keys, vals, ck, cv, [tokens])
    bound = near(want, dtype, q, k, v, ck, cv, group, [tokens])
    # and each element off by at most 2^-29 of the largest, in the products with c - 8
    code, _, delta = quantise(k.double().numpy(), group)
    size = torch.from_numpy(np.abs(code.astype(np.float64) - 8) * np.repeat(delta.astype(np.float64), group, -1)).sum(-1)
    for h in range(8):
        p = torch.softmax(torch.cat([keys[0, h // 4] @ q[0, h].cpu().double() / math.sqrt(128), torch.zeros(1)]), 0)
        e = 2.0 ** -29 * 16 * size[0, h // 4] / math.sqrt(128)
        bound[0, h] += (p[:tokens] * e) @ (vals[0, h // 4].abs() + want[0, h].abs())
    got = paged.paged_attention_step(q, cache, 0, table, ck, cv).cpu().double()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,per", [(64, 2), (100, 1), (129, 1), (300, 2)])
def test_attention_of_many_kv_heads(dtype, kv_heads, per):
    """As many KV heads as leave each four workgroups, two, or one, and more of
    them than the card has places for at once; 256-token pages, int32 indices."""
    lengths = [2100, 0, 300]
    gen = torch.Generator().manual_seed(kv_heads)
    cache, table = make(lengths, kv_heads, group=64, page=256, max_tokens=2101)
    k, v = (torch.randn(3, kv_heads, 2100, 128, generator=torch.Generator(device=DEV).manual_seed(kv_heads + i),
                        device=DEV) for i in range(2))
    count = torch.tensor(lengths, device=DEV)
    paged.write_tokens(cache, 0, table, k, v, tokens=count)
    table.advance(count, bound=2100)
    rows, vals = paged.read_tokens(cache, 0, table, dtype=torch.float32)  # (bit for bit the format's: tested above)
    q = torch.randn(3, kv_heads * per, 128, generator=gen).to(dtype).to(DEV)
    ck, cv = (torch.randn(3, kv_heads, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    rows = torch.cat([rows, torch.zeros_like(rows[:, :, :1])], 2).double()
    vals = torch.cat([vals, torch.zeros_like(vals[:, :, :1])], 2).double()
    for b, n in enumerate(lengths):
        rows[b, :, n], vals[b, :, n] = ck[b].double(), cv[b].double()
    want = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lengths):
        for h in range(kv_heads):
            s = torch.softmax(q[b, h * per:(h + 1) * per].double() @ rows[b, h, :n + 1].t().contiguous() / math.sqrt(128), 1)
            want[b, h * per:(h + 1) * per] = s @ vals[b, h, :n + 1]
    # fp32 work, and for the dense bf16 form V and the weights in fp16 of the largest value
    bound = torch.finfo(dtype).eps / 2 * (want.abs() + FP32) + FP32
    half = bound + (2 * 2.0 ** -11 * float(vals.abs().max()) if dtype == torch.bfloat16 else 0)
    ws = popkv.LayerStepWorkspace()
    for _ in range(2):
        got = paged.paged_attention_step(q, cache, 0, table, ck, cv, workspace=ws)
        assert ((got.double() - want).abs() <= half).all(), float((got.double() - want).abs().max())
    idx = torch.arange(2101, device=DEV, dtype=torch.int32).expand(3, kv_heads * per, 2101).contiguous()
    got = paged.paged_indexed_attention(q, cache, 0, table, ck, cv, idx, torch.arange(kv_heads * per, device=DEV) // per,
                                        workspace=ws)
    assert ((got.double() - want).abs() <= bound).all(), float((got.double() - want).abs().max())
