"""Chunks of new tokens over the paged 4-bit cache against plain float64: their
attention, the weights that tokens gather, eviction by them, and a serving loop
of all of them together."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from popkv_amd import paged, popkv

from test_gpu_paged import dequantised, fill, make, unpack

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# fp32 sums and exponentials of logits up to about 30 in magnitude: relative
# error about 30 * 2^-23 of values up to about 5 (as for the dense layer)
FP32 = 4e-5


def attend(q, k, v, nk, nv, lengths, new):
    """float64 [B, QH, rows, 128] and the weights [B, KVH, longest + rows] that every
    token (cached, then new at its place) gathers; rows past new[b] are zero."""
    q, nk, nv = (t.cpu().double() for t in (q, nk, nv))
    batch, qh, rows, _ = q.shape
    kvh = nk.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    w = torch.zeros((batch, kvh, max(lengths) + rows), dtype=torch.float64)
    for b, (n, m) in enumerate(zip(lengths, new)):
        ahead = torch.arange(n + m)[None] > n + torch.arange(m)[:, None]
        for h in range(qh if m else 0):
            g = h // (qh // kvh)
            keys, vals = torch.cat([k[b, g, :n], nk[b, g, :m]]), torch.cat([v[b, g, :n], nv[b, g, :m]])
            logits = (q[b, h, :m] @ keys.T / math.sqrt(128)).masked_fill(ahead, -math.inf)
            p = torch.softmax(logits, 1)
            out[b, h, :m] = torch.where(p[..., None] > 0, p[..., None] * vals, 0.0).sum(1) if not vals.isfinite().all() \
                else p @ vals
            w[b, g, :n + m] += p.sum(0)
    return out, w


def allowed(want, dtype, v, nv):
    """Largest error per element: the output's rounding (half a step) and the fp32 work;
    for 16-bit tensors the rounding of cached values to fp16, half a step (2^-11) of at
    most the largest value; for bf16 ones those of the weights too, fp16 on cached tokens
    and bf16 (2^-8) on new ones, twice as the sum that they are divided by is the rounded
    ones'."""
    bound = torch.finfo(dtype).eps / 2 * want.abs() + FP32
    if dtype == torch.float32:
        return bound
    group = want.shape[1] // nv.shape[1]
    top = torch.cat([v, nv.cpu().double()], 2).abs().amax((2, 3)).repeat_interleave(group, 1)[..., None, None]
    return bound + top * (2.0 ** -11 if dtype == torch.float16 else 3 * 2.0 ** -11 + 2 * 2.0 ** -8)


def setup(lengths, new, kv_heads, group, dtype, *, dims=32, page=64, seed=0, spread=2.0, layers=1):
    gen = torch.Generator().manual_seed(seed)
    rows = max(max(new), 1)
    cache, table = make([max(n, 1) for n in lengths], kv_heads, group=dims, page=page, layers=layers,
                        max_tokens=max(lengths) + rows, seed=seed)
    k, v = fill(cache, table, layers - 1, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=max(lengths))
    batch = len(lengths)
    q = (torch.randn(batch, rows, kv_heads * group, 128, generator=gen) * spread).to(dtype).to(DEV).transpose(1, 2)
    nk, nv = (torch.randn(batch, rows, kv_heads, 128, generator=gen).to(dtype).to(DEV).transpose(1, 2) for _ in range(2))
    return cache, table, k, v, q, nk, nv


CHUNKS = [([0], [1]), ([0], [33]), ([1], [1]), ([63, 64, 65], [1, 2, 3]), ([31, 0, 200, 5], [64, 65, 0, 7]),
          ([129], [300]), ([1000, 3, 517], [130, 257, 1]), ([5000], [6]), ([0, 0], [700, 511])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (2, 2), (3, 2), (4, 2), (7, 1), (8, 2), (20, 1)])
@pytest.mark.parametrize("lengths,new", CHUNKS, ids=str)
def test_chunk_attention(dtype, group, kv_heads, lengths, new):
    """Nothing cached, one token, tile and page edges, ragged chunks with an empty one,
    groups that no tile of rows is a multiple of; the same with weights gathered."""
    dims, page = (16, 32, 64)[(len(lengths) + group) % 3], (32, 64, 128, 256)[(group + max(new)) % 4]
    cache, table, k, v, q, nk, nv = setup(lengths, new, kv_heads, group, dtype, dims=dims, page=page, seed=sum(lengths) + group)
    want, gathered = attend(q, k, v, nk, nv, lengths, new)
    bound = allowed(want, dtype, v, nv)
    tokens = torch.tensor(new, device=DEV)
    ws = popkv.LayerStepWorkspace()
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens, workspace=ws)
    assert got.shape == q.shape and got.stride() == q.stride()
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    for b, n in enumerate(new):
        assert not got[b, :, n:].any()
    w = torch.full((len(lengths), kv_heads, table.capacity), 0.25, device=DEV)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    back = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens, weights=w, workspace=ws, out=out)
    assert back is out
    for b, n in enumerate(new):
        assert (out[b, :, n:] == 7.0).all()
        err = (out[b, :, :n].cpu().double() - want[b, :, :n]).abs()
        assert (err <= bound[b, :, :n]).all()
        total = lengths[b] + n
        err = (w[b, :, :total].cpu().double() - 0.25 - gathered[b, :, :total]).abs()
        # the sum's own rounding, and every weight's relative error
        assert (err <= 2.0 ** -23 * (gathered[b, :, :total] + 0.25) + FP32 * gathered[b, :, :total] + 1e-7).all()
        assert (w[b, :, total:] == 0.25).all()
    # equal bits from call to call
    again = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens, workspace=ws)
    assert torch.equal(again, got)
    w2 = torch.full_like(w, 0.25)
    paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens, weights=w2, workspace=ws)
    assert torch.equal(w2, w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_of_none_are_all_rows(dtype):
    lengths, new = [70, 9], [37, 37]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, dtype, seed=5)
    want, _ = attend(q, k, v, nk, nv, lengths, new)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv)
    assert ((got.cpu().double() - want).abs() <= allowed(want, dtype, v, nv)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_is_a_decode_step(dtype):
    """A chunk of one token and the decode step's attention agree."""
    lengths = [300, 0, 1029]
    cache, table, k, v, q, nk, nv = setup(lengths, [1, 1, 1], 2, 4, dtype, seed=6)
    want, _ = attend(q, k, v, nk, nv, lengths, [1, 1, 1])
    bound = allowed(want, dtype, v, nv)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv)
    step = paged.paged_attention_step(q[:, :, 0].contiguous(), cache, 0, table, nk[:, :, 0].contiguous(),
                                      nv[:, :, 0].contiguous())
    assert ((got[:, :, 0].cpu().double() - step.cpu().double()).abs() <= 2 * bound[:, :, 0]).all()


@pytest.mark.parametrize("dims", (16, 32, 64))
@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_with_outlier_channels(dtype, dims):
    """Channels ten times as large, queries of one sign: logits up to a hundred, where
    keys rounded to fp16 would show."""
    lengths, new, gen = [900, 200], [40, 3], torch.Generator().manual_seed(dims)
    cache, table, _, _, q, nk, nv = setup(lengths, new, 2, 4, dtype, dims=dims, seed=7)
    scale = torch.ones(128)
    scale[torch.randperm(128, generator=gen)[:4]] = 10.0
    k, v = torch.randn(2, 2, 900, 128, generator=gen) * scale, torch.randn(2, 2, 900, 128, generator=gen)
    table.counts.zero_()
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV), tokens=torch.tensor(lengths, device=DEV))
    table.counts.copy_(torch.tensor(lengths))
    k, v = dequantised(k, dims), dequantised(v, dims)
    q = (q.float().abs() * 0.5).to(dtype)
    want, gathered = attend(q, k, v, nk, nv, lengths, new)
    w = torch.zeros((2, 2, table.capacity), device=DEV)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=torch.tensor(new, device=DEV), weights=w)
    err = (got.cpu().double() - want).abs()
    # fp32's own: a logit is a sum of 128 terms with partial sums up to a few hundred
    bound = allowed(want, dtype, v, nv) + 1e-3 * (dtype == torch.bfloat16) + 2e-4
    assert (err <= bound).all(), float((err / bound).max())
    for b, n in enumerate(lengths):
        total = n + new[b]
        assert ((w[b, :, :total].cpu().double() - gathered[b, :, :total]).abs() <= 2e-4 * gathered[b, :, :total] + 1e-6).all()


def test_operand_strides_and_alignment():
    """Slices of wider tensors, odd alignments (read through copies), a strided out."""
    lengths, new = [100, 33], [20, 20]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, torch.bfloat16, seed=8)
    want = paged.paged_chunk_attention(q, cache, 0, table, nk, nv)
    fused = torch.cat((q, nk, nv), 1).transpose(1, 2).contiguous().transpose(1, 2)  # [B, QH + 2 KVH, rows, 128]
    got = paged.paged_chunk_attention(fused[:, :8], cache, 0, table, fused[:, 8:10], fused[:, 10:])
    assert torch.equal(got, want)
    odd = lambda x: torch.cat((torch.zeros(1, dtype=x.dtype, device=DEV), x.reshape(-1)))[1:].view(x.shape)  # noqa: E731
    assert torch.equal(paged.paged_chunk_attention(odd(q), cache, 0, table, odd(nk), odd(nv)), want)
    wide = torch.full((2, 20, 8, 192), 3.0, dtype=torch.bfloat16, device=DEV)
    out = wide[..., :128].transpose(1, 2)
    paged.paged_chunk_attention(q, cache, 0, table, nk, nv, out=out)
    assert torch.equal(out, want) and (wide[..., 128:] == 3.0).all()
    flat = torch.empty(2, 8, 20, 128, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(paged.paged_chunk_attention(q, cache, 0, table, nk, nv, out=flat), want)


def test_layers_bounds_and_negative_counts():
    """Another layer than the first; a bound that cuts; counts and tokens outside their
    ranges are held in them."""
    lengths, new = [70, 9], [5, 5]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, torch.float32, seed=9, layers=3)
    want, _ = attend(q, k, v, nk, nv, lengths, new)
    got = paged.paged_chunk_attention(q, cache, 2, table, nk, nv, tokens=torch.tensor([500, 5], device=DEV), max_tokens=9999)
    assert ((got.cpu().double() - want).abs() <= allowed(want, torch.float32, v, nv)).all()
    table.bound = 40
    want, _ = attend(q, k, v, nk, nv, [40, 9], new)
    got = paged.paged_chunk_attention(q, cache, 2, table, nk, nv)
    assert ((got.cpu().double() - want).abs() <= allowed(want, torch.float32, v, nv)).all()
    table.counts.fill_(-3)
    want, gathered = attend(q, k, v, nk, nv, [0, 0], [5, 0])
    w = torch.zeros((2, 2, table.capacity), device=DEV)
    got = paged.paged_chunk_attention(q, cache, 2, table, nk, nv, tokens=torch.tensor([5, -1], device=DEV), weights=w)
    assert ((got.cpu().double() - want).abs() <= allowed(want, torch.float32, v, nv)).all()
    assert ((w[:, :, :5].cpu().double() - gathered[:, :, :5]).abs() <= FP32).all() and not w[:, :, 5:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_missing_pages_are_left_out(dtype):
    lengths, new = [160, 70], [9, 9]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 2, dtype, page=32, seed=10)
    table.table[0, 1], table.table[0, 4], table.table[1, 0] = -1, cache.pages, cache.pages + 5
    keep = [torch.tensor([t for t in range(n) if t // 32 not in gone]) for n, gone in zip(lengths, ((1, 4), (0,)))]
    w = torch.zeros((2, 2, table.capacity), device=DEV)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=w)
    for b in range(2):
        want, gathered = attend(q[b:b + 1], k[b:b + 1, :, keep[b]], v[b:b + 1, :, keep[b]], nk[b:b + 1], nv[b:b + 1],
                                [len(keep[b])], [9])
        assert ((got[b:b + 1].cpu().double() - want).abs() <= allowed(want, dtype, v[b:b + 1], nv[b:b + 1])).all()
        at = torch.cat((keep[b], lengths[b] + torch.arange(9)))
        assert ((w[b, :, at.to(DEV)].cpu().double() - gathered[0]).abs() <= FP32 * (1 + gathered[0])).all()
        rest = torch.ones(table.capacity, dtype=torch.bool)
        rest[at] = False
        assert not w[b, :, rest.to(DEV)].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_masked_may_be_anything(dtype):
    """Rows of new K/V and q behind tokens[b], and tokens ahead of a row, hold NaN and
    infinities: rows that do not see them are finite and the same."""
    lengths, new = [50, 0], [9, 40]
    cache, table, k, v, q, nk, nv = setup(lengths, [40, 40], 2, 4, dtype, seed=11)
    tokens = torch.tensor(new, device=DEV)
    want, gathered = attend(q, k, v, nk, nv, lengths, new)
    nk, nv, q = nk.clone(), nv.clone(), q.clone()
    nk[0, :, 9:], nv[0, :, 9:], q[0, :, 9:] = float("nan"), float("inf"), float("nan")
    nk[1, 0, 30], nv[1, 0, 30, 5] = float("nan"), float("nan")
    nv[1, 1, 20, 100], nv[1, 1, 35, 100] = float("inf"), float("-inf")
    w = torch.zeros((2, 2, table.capacity), device=DEV)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens, weights=w).cpu().double()
    bound = allowed(want, dtype, v, nv.nan_to_num(0, 0, 0))
    ok = (got - want).abs() <= bound
    assert ok[0].all()
    # the first KV head's query heads see a NaN key from row 30 on
    assert ok[1, :4, :30].all() and got[1, :4, 30:].isnan().all()
    # the others infinite values at one dim, plus from row 20 on, both from row 35 on
    rest = torch.arange(128) != 100
    assert ok[1, 4:][..., rest].all() and ok[1, 4:, :20].all()
    assert (got[1, 4:, 20:35, 100] == math.inf).all() and got[1, 4:, 35:, 100].isnan().all()
    assert ((w[0, :, :59].cpu().double() - gathered[0, :, :59]).abs() <= FP32 * (1 + gathered[0, :, :59])).all()


def test_infinite_and_nan_logits():
    """Logits of plus infinity or NaN make their rows NaN, as a softmax does; minus
    infinity is no weight."""
    lengths, new = [40], [6]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 1, 2, torch.float32, seed=12)
    nk, q = nk.clone(), q.clone()
    q[..., 0] = 1.0
    nk[0, 0, 2, 0] = float("-inf")
    want, _ = attend(q, k, v, torch.where(nk.isinf(), -1e30, nk), nv, lengths, new)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv).cpu().double()
    assert ((got - want).abs() <= FP32 + 2.0 ** -24 * want.abs()).all()
    nk[0, 0, 3, 0] = float("inf")
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv).cpu().double()
    assert ((got - want).abs()[:, :, :3] <= FP32 + 2.0 ** -24 * want.abs()[:, :, :3]).all() and got[:, :, 3:].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_and_large_elements(dtype):
    """Queries of all sizes, tiny beside large elements, values up to the type's reach."""
    lengths, new = [130, 64], [17, 17]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, dtype, seed=13)
    q = q.clone()
    q[:, :, ::3] *= 2.0 ** -12
    q[:, :, 1::3, 64:] *= 2.0 ** -10
    q[:, 1] = 0
    nv = (nv * 4096).to(dtype)
    want, _ = attend(q, k, v, nk, nv, lengths, new)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv).cpu().double()
    bound = allowed(want, dtype, v, nv) + FP32 * 4096
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


def test_large_batches():
    """More sequences than a wave has lanes, most of them empty or short."""
    lengths, new = [(i * 37) % 90 if i % 3 else 0 for i in range(150)], [(i * 11) % 7 for i in range(150)]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 1, 2, torch.bfloat16, page=32, seed=14)
    want, _ = attend(q, k, v, nk, nv, lengths, new)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=torch.tensor(new, device=DEV))
    assert ((got.cpu().double() - want).abs() <= allowed(want, torch.bfloat16, v, nv)).all()


@pytest.mark.parametrize("kv_heads", (1, 300))
def test_many_heads_and_long_chunks(kv_heads):
    """More KV heads than CUs; a chunk of many tiles of rows in one group."""
    lengths, new = ([90], [3]) if kv_heads == 300 else ([700], [1100])
    cache, table, k, v, q, nk, nv = setup(lengths, new, kv_heads, 2, torch.bfloat16, page=32, seed=15)
    want, gathered = attend(q, k, v, nk, nv, lengths, new)
    w = torch.zeros((1, kv_heads, table.capacity), device=DEV)
    for weights in (None, w):
        got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=weights)
        assert ((got.cpu().double() - want).abs() <= allowed(want, torch.bfloat16, v, nv)).all()
    total = lengths[0] + new[0]
    assert ((w[:, :, :total].cpu().double() - gathered).abs() <= FP32 * (gathered + 0.01)).all()


def test_weights_on_average_as_exact_as_float32():
    """The norm of the weights' error beside that of plain float32 sums of dequantised
    rows: one rounding more of each logit, and of each sum, at most."""
    lengths, new = [2000], [64]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, torch.bfloat16, seed=16)
    _, gathered = attend(q, k, v, nk, nv, lengths, new)
    w = torch.zeros((1, 2, table.capacity), device=DEV)
    paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=w)
    keys = torch.cat((k[0, :, :2000], nk[0].cpu().double()), 1).float()
    logits = q[0].cpu().float().reshape(2, 4 * 64, 128) @ keys.transpose(1, 2) / math.sqrt(128)
    ahead = torch.arange(2064)[None] > 2000 + torch.arange(64)[:, None]
    p = torch.softmax(logits.unflatten(1, (4, 64)).masked_fill(ahead, -math.inf), 3).sum((1, 2))
    plain = (p.double() - gathered[0]).norm()
    assert (w[0, :, :2064].cpu().double() - gathered[0]).norm() <= 2 * plain


def test_no_rows():
    cache, table, _, _, q, nk, nv = setup([5], [1], 1, 1, torch.bfloat16)
    got = paged.paged_chunk_attention(q[:, :, :0], cache, 0, table, nk[:, :, :0], nv[:, :, :0])
    assert got.shape == (1, 1, 0, 128)


def test_a_pool_past_32_bit_offsets():
    """Pages whose bytes lie beyond 2^32 of the layer's pool, read, chosen and moved."""
    pages = 17_000  # 256 KiB of codes each: 4.4 GB
    cache = paged.allocate_paged_cache(1, pages, 8, page_tokens=256, dim_group_size=64, device=DEV)
    table = paged.PageTable.create(1, 768, cache)
    table.table[0, :2] = torch.tensor([pages - 1, pages - 300])
    table.refs[pages - 1] = table.refs[pages - 300] = 1
    gen = torch.Generator().manual_seed(2)
    k, v = fill(cache, table, 0, [300], gen)
    table.advance(300)
    q, nk, nv = (torch.randn(1, 8, 20, 128, generator=gen).to(DEV) for _ in range(3))
    w = paged.allocate_token_weights(cache, table)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=w[0])
    want, gathered = attend(q, k, v, nk, nv, [300], [20])
    assert ((got.cpu().double() - want).abs() <= allowed(want, torch.float32, v, nv)).all()
    new, moved, kept = paged.evict_tokens(cache, table, w, 200, recent=10)
    rows = [x[0].cpu() for x in paged.read_tokens(cache, 0, new, dtype=torch.float32)]
    for h in range(8):
        at = kept[0, 0, h].long().cpu()
        assert torch.equal(rows[0][h, :200], k[0, h, at].float()) and torch.equal(rows[1][h, :200], v[0, h, at].float())
    assert new.table.tolist() == [[pages - 1, -1, -1]] and int(new.refs[pages - 300]) == 0


# ---------------------------------------------------------------- eviction

def choose(w: np.ndarray, n: int, keep: int, recent: int) -> np.ndarray:
    """The kept places of a row of weights, ascending."""
    recent = min(recent, keep)
    m = n - recent
    key = np.where(np.isnan(w[:m]), np.inf, w[:m].astype(np.float64))
    order = sorted(range(m), key=lambda i: (not np.isnan(w[i]), -key[i], i))
    return np.sort(np.array(order[:keep - recent] + list(range(m, n)), dtype=np.int64))


def check_evict(cache, table, w, keep, recent, *, keeps=None, cut=None, **kw):
    """Runs an eviction and checks everything that it may and may not change, for
    sequences `cut` (default: all that are longer than their share)."""
    codes, scales = cache.codes.cpu().numpy().copy(), cache.scales.cpu().view(torch.int16).numpy().copy()
    tab, counts, refs = (x.cpu().numpy().copy() for x in (table.table, table.counts, table.refs))
    weights = w.cpu().numpy().copy()
    page, (layers, batch, kvh, capacity) = cache.page_tokens, weights.shape
    share = [keep] * batch if keeps is None else [min(max(int(x), 0), keep) for x in keeps.tolist()]
    new, moved, kept = paged.evict_tokens(cache, table, w, keep, recent=recent, keeps=keeps, **kw)
    got_codes, got_scales = cache.codes.cpu().numpy(), cache.scales.cpu().view(torch.int16).numpy()
    got_tab, got_counts, got_refs = (x.cpu().numpy() for x in (new.table, new.counts, new.refs))
    moved, kept = moved.cpu().numpy(), kept.cpu().numpy()
    want_tab, want_refs, want_kept, want_moved = tab.copy(), refs.copy(), np.full(kept.shape, -1, np.int32), weights.copy()
    free = iter(np.flatnonzero(refs == 0))
    want_codes, want_scales = codes.copy(), scales.copy()
    for b in range(batch):
        n, k = min(max(int(counts[b]), 0), capacity), share[b]
        if n <= k or (cut is not None and b not in cut):
            continue
        stay = -(-k // page)
        for i in range(tab.shape[1]):
            was = tab[b, i]
            now = was if i < stay and refs[was] == 1 else next(free) if i < stay else -1
            want_tab[b, i] = now
            if now != was:
                if was >= 0:
                    want_refs[was] -= 1
                if now >= 0:
                    want_refs[now] = 1
        for layer in range(layers):
            for h in range(kvh):
                at = choose(weights[layer, b, h], n, k, recent)
                want_kept[layer, b, h, :k] = at
                j = np.arange(k)
                src, dst = (tab[b, at // page], at % page), (want_tab[b, j // page], j % page)
                want_codes[layer, dst[0], h, dst[1]] = codes[layer, src[0], h, src[1]]
                want_scales[layer, dst[0], h, dst[1]] = scales[layer, src[0], h, src[1]]
                want_moved[layer, b, h] = 0
                want_moved[layer, b, h, :k] = weights[layer, b, h, at]
        counts[b] = k
    assert np.array_equal(kept, want_kept)
    assert np.array_equal(got_tab, want_tab) and np.array_equal(got_counts, counts) and np.array_equal(got_refs, want_refs)
    assert np.array_equal(moved, want_moved, equal_nan=True)
    assert np.array_equal(got_codes, want_codes) and np.array_equal(got_scales, want_scales)
    return new


def filled_pool(lengths, kv_heads, *, page=32, group=32, layers=2, spare=3, room=0, seed=0):
    cache, table = make(lengths, kv_heads, group=group, page=page, layers=layers, spare=spare,
                        max_tokens=max(lengths) + room, seed=seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cache.codes.random_(0, 256, generator=gen)
    cache.scales.copy_(torch.randn(cache.scales.shape, generator=gen, device=DEV))
    table.counts.copy_(torch.tensor(lengths))
    table.bound = max(lengths)
    w = torch.randn((layers, len(lengths), kv_heads, table.capacity), generator=gen, device=DEV).mul_(2).exp_()
    return cache, table, w


@pytest.mark.parametrize("group", (16, 32, 64))
@pytest.mark.parametrize("lengths,keep,recent,page", [([100], 40, 8, 32), ([65, 64, 63, 1, 0, 300], 64, 0, 64),
                                                     ([200, 150], 1, 1, 32), ([200, 31], 0, 0, 32), ([90], 89, 100, 128),
                                                     ([1500, 1300], 1100, 64, 256), ([40, 41, 42], 37, 5, 32)])
def test_evict(group, lengths, keep, recent, page):
    cache, table, w = filled_pool(lengths, 3, page=page, group=group, room=70, seed=keep + len(lengths))
    check_evict(cache, table, w, keep, recent)


def test_evict_in_place_and_twice():
    """The table and the weights in place; then again, and again."""
    cache, table, w = filled_pool([700, 340, 20], 2, seed=3)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for keep in (500, 300, 299, 12):
        new = check_evict(cache, table, w, keep, 9, out=table, weights_out=w, status=status)
        assert new is table
    assert int(status) == 0 and table.counts.tolist() == [12, 12, 12]


def test_evict_shares_of_their_own():
    """keeps: a share for each sequence, held in [0, keep]."""
    cache, table, w = filled_pool([100, 100, 100, 100], 2, seed=4)
    check_evict(cache, table, w, 70, 10, keeps=torch.tensor([-5, 30, 99, 70], device=DEV))


def test_evict_ties_and_odd_weights():
    """Equal weights keep the first; -0 is 0; NaN is above infinity; negative ones."""
    cache, table, w = filled_pool([500, 400], 2, seed=5)
    w[0] = 1.0
    w[1, 0, 0] = 0.0
    w[1, 0, 0, ::2] = -0.0
    w[1, 0, 1] = (torch.arange(w.shape[-1], device=DEV) % 5).float() - 2
    w[1, 1, 0, 7], w[1, 1, 0, 20], w[1, 1, 0, 300] = float("nan"), float("inf"), float("nan")
    w[1, 1, 0, 50:60] = float("-inf")
    w[1, 1, 1] = -w[1, 1, 1]
    for keep in (450, 120, 2):
        check_evict(cache, table, w.clone(), keep, 1, out=table)


def test_evict_long_rows():
    """A row of weights past what registers would hold, of few and of many values."""
    n = 70_001
    cache, table, w = filled_pool([n], 1, page=256, layers=2, seed=6)
    w[1] = torch.randint(0, 3, w[1].shape, device=DEV).float()
    check_evict(cache, table, w, 65_000, 100)


def test_evict_pages_that_forks_share():
    """Pages of the front with further holders stay theirs; without free ones the
    sequence is left whole, and the next that needs none is still cut."""
    cache, table, w = filled_pool([320, 320, 320, 320], 2, page=32, spare=12, seed=7)
    for b in (1, 2):
        held = table.table[b, :6].long()
        table.refs[held] -= 1
        table.table[b, :6] = table.table[0, :6]
        table.refs[table.table[0, :6].long()] += 1
    w[:, 1:] = w[:, 1:].flip(-1)
    new = check_evict(cache, table, w, 150, 20)
    assert new.table.unique().numel() == 4 * 5 + 1
    cache, table, w = filled_pool([320, 320, 320], 2, page=32, spare=0, seed=8)
    shared = table.table[0, :3].long()
    table.refs[table.table[1, :3].long()] = 5  # held elsewhere, for good
    table.table[1, :3] = table.table[0, :3]
    table.refs[shared] += 1
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check_evict(cache, table, w, 150, 20, cut=(2,), status=status)
    assert int(status) == 4


def test_evict_from_a_large_pool():
    """Pools and tables past what one workgroup plans."""
    cache, table, w = filled_pool([200 + i % 90 for i in range(40)], 1, page=32, layers=1, spare=17_000, seed=11)
    for b in range(1, 40, 3):
        held = table.table[b, :2].long()
        table.refs[held] -= 1
        table.table[b, :2] = table.table[b - 1, :2]
        table.refs[table.table[b - 1, :2].long()] += 1
    check_evict(cache, table, w.clone(), 230, 16)
    check_evict(cache, table, w.clone(), 100, 16, out=table)


def test_evict_to_nothing_and_reuse():
    """Everything given back, and the pages taken again."""
    cache, table, w = filled_pool([100, 40], 2, page=32, spare=0, seed=12)
    new = check_evict(cache, table, w, 0, 5, out=table, weights_out=w)
    assert not new.refs.any() and (new.table == -1).all() and not w.any()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged.reserve_pages(new, 40, status=status, out=new)
    assert int(status) == 0 and (new.table >= 0).sum() == 4


def test_evict_missing_pages_and_counts_outside():
    cache, table, w = filled_pool([320, 320, 320], 2, page=32, seed=9)
    table.table[0, 4], table.table[1, 0] = -1, cache.pages
    table.counts.copy_(torch.tensor([320, 320, 9999]))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check_evict(cache, table, w, 100, 20, cut=(2,), status=status)
    assert int(status) == 4


def test_evict_gives_reserved_pages_back():
    cache, table, w = filled_pool([100, 64], 2, page=32, spare=8, room=200, seed=10)
    paged.reserve_pages(table, 100, out=table)
    new = check_evict(cache, table, w, 64, 5)
    # the second sequence, not cut, keeps the pages reserved for it
    assert (new.table[0] >= 0).sum() == 2 and (new.table[1] >= 0).sum() == 6


# ---------------------------------------------------------------- together

def test_a_bounded_cache_serves_prompts_and_decodes():
    """Prompts in chunks of different lengths, then decode, the cache cut back whenever
    it has grown past its budget: every layer and head against float64 over the rows
    that it should hold."""
    layers, kvh, group, batch, keep, recent = 2, 2, 2, 3, 96, 16
    cache = paged.allocate_paged_cache(layers, 24, kvh, page_tokens=32, dim_group_size=32, device=DEV)
    table = paged.PageTable.create(batch, 256, cache)
    w = paged.allocate_token_weights(cache, table)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ws = popkv.LayerStepWorkspace()
    gen = torch.Generator().manual_seed(20)
    rows = [[[(torch.zeros(0, 128, dtype=torch.float64),) * 2 for _ in range(kvh)] for _ in range(batch)]
            for _ in range(layers)]
    gathered = [[[torch.zeros(0, dtype=torch.float64) for _ in range(kvh)] for _ in range(batch)] for _ in range(layers)]
    steps = [[40, 7, 64], [30, 64, 1]] + [[1, 1, 1]] * 3 + [[20, 0, 33], [5, 5, 5]] + [[1, 1, 1]] * 4
    for new in steps:
        most = max(new)
        tokens = torch.tensor(new, device=DEV)
        paged.reserve_pages(table, tokens, status=status, out=table)
        for layer in range(layers):
            q, k, v = (torch.randn(batch, h, most, 128, generator=gen) for h in (kvh * group, kvh, kvh))
            out = paged.paged_chunk_attention(q.to(DEV), cache, layer, table, k.to(DEV), v.to(DEV), tokens=tokens,
                                              weights=w[layer], workspace=ws).cpu().double()
            paged.write_tokens(cache, layer, table, k.to(DEV), v.to(DEV), tokens=tokens, status=status)
            kq, vq = dequantised(k, 32), dequantised(v, 32)
            for b in range(batch):
                for g in range(kvh):
                    ck, cv = rows[layer][b][g]
                    n, m = len(ck), new[b]
                    want, add = attend(q[b:b + 1, g * group:g * group + group], ck[None, None], cv[None, None],
                                       k[b:b + 1, g:g + 1], v[b:b + 1, g:g + 1], [n], [m])
                    err = (out[b, g * group:g * group + group] - want[0]).abs()
                    assert (err <= FP32 + 2.0 ** -24 * want[0].abs()).all()
                    gathered[layer][b][g] = torch.cat((gathered[layer][b][g], torch.zeros(m))) + add[0, 0, :n + m]
                    rows[layer][b][g] = (torch.cat((ck, kq[b, g, :m])), torch.cat((cv, vq[b, g, :m])))
        table.advance(tokens, bound=min(table.bound + most, 256))
        if max(len(rows[0][b][0][0]) for b in range(batch)) > keep + 8:
            held = w.cpu().numpy().copy()
            _, _, kept = paged.evict_tokens(cache, table, w, keep, recent=recent, status=status, out=table, weights_out=w)
            table.bound = keep
            kept = kept.cpu()
            for layer in range(layers):
                for b in range(batch):
                    for g in range(kvh):
                        n = len(rows[layer][b][g][0])
                        sums = gathered[layer][b][g]
                        assert np.abs(held[layer, b, g, :n] - sums.numpy()).max() <= 1e-3
                        if n <= keep:
                            assert (kept[layer, b, g] == -1).all()
                            continue
                        at = kept[layer, b, g].long()
                        assert np.array_equal(at.numpy(), choose(held[layer, b, g], n, keep, recent))
                        rows[layer][b][g] = tuple(x[at] for x in rows[layer][b][g])
                        gathered[layer][b][g] = sums[at]
    assert int(status) == 0
    assert table.counts.tolist() == [len(rows[0][b][0][0]) for b in range(batch)]


def test_captured_steps_replay():
    """A decode step with its weights, and an eviction, captured once and replayed while
    the sequences grow, with eager work between the replays."""
    lengths, layers = [40, 100], 1
    cache, table = make([400, 400], 2, page=32, spare=4, max_tokens=400, seed=21)
    gen = torch.Generator().manual_seed(21)
    fill(cache, table, 0, lengths, gen)
    table.advance(torch.tensor(lengths, device=DEV), bound=100)
    w = paged.allocate_token_weights(cache, table)
    q, k, v = (torch.randn(2, h, 3, 128, generator=gen).bfloat16().to(DEV) for h in (8, 2, 2))
    tokens = torch.tensor([3, 2], device=DEV)
    ws, keeps = popkv.LayerStepWorkspace(), torch.tensor([400, 400], device=DEV)

    def step(cache, table, w):
        paged.reserve_pages(table, tokens, out=table)
        out = paged.paged_chunk_attention(q, cache, 0, table, k, v, tokens=tokens, weights=w[0], max_tokens=400,
                                          workspace=ws)
        paged.write_tokens(cache, 0, table, k, v, tokens=tokens)
        table.counts.add_(tokens)
        paged.evict_tokens(cache, table, w, 400, recent=4, keeps=keeps, out=table, weights_out=w)
        return out

    def clone():
        return (paged.PagedKVCache(cache.codes.clone(), cache.scales.clone(), 32),
                paged.PageTable(table.table.clone(), table.counts.clone(), table.refs.clone(), 32, 100), w.clone())

    mirror = clone()
    first = clone()
    step(*first)  # the workspace grown and everything loaded
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(cache, table, w)
    for i in range(6):
        keeps.fill_(90 if i % 3 == 2 else 400)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step(*mirror)
        assert torch.equal(out, want)
        assert torch.equal(w, mirror[2]) and torch.equal(table.table, mirror[1].table)
        assert torch.equal(table.counts, mirror[1].counts) and torch.equal(cache.codes, mirror[0].codes)


def test_on_another_stream():
    lengths, new = [300, 20], [10, 40]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, torch.bfloat16, seed=22)
    tokens = torch.tensor(new, device=DEV)
    want = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=tokens)
    stream.synchronize()
    assert torch.equal(got, want)


def test_a_workspace_shared_with_decode_steps():
    """The merge tickets of the decode steps, at the workspace's front, stay zero."""
    lengths = [3000, 20]
    cache, table, k, v, q, nk, nv = setup(lengths, [2, 2], 2, 4, torch.bfloat16, seed=23)
    ws = popkv.LayerStepWorkspace()
    step = lambda: paged.paged_attention_step(q[:, :, 0].contiguous(), cache, 0, table, nk[:, :, 0].contiguous(),  # noqa: E731
                                              nv[:, :, 0].contiguous(), workspace=ws)
    w = torch.zeros((2, 2, table.capacity), device=DEV)
    want = step()
    for _ in range(3):
        paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=w, workspace=ws)
        assert torch.equal(step(), want)
        assert not ws.buffer[:1 << 18].any()
