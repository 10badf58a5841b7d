"""Chunks over the paged 4-bit cache and its eviction where they can go wrong: a bound
behind the counts, elements at the end of a type's range, the norm of the errors, one
token both ways, shares of free pages that do not fit, proposals that are rejected."""
from __future__ import annotations

import math

import pytest
import torch

from popkv_amd import paged, popkv

from test_gpu_paged import dequantised, make, wide_values
from test_gpu_paged_chunk import DEV, DTYPES, FP32, allowed, attend, check_evict, filled_pool, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_of_new_tokens_behind_a_bound_that_cuts(dtype):
    """Replays move the counts and not the bound: cached tokens past it are left out, and
    a chunk's tokens still gather at the places where they are written, ``counts[b] + t``,
    up to the table's end."""
    lengths, new = [70, 9], [5, 3]
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, dtype, seed=30)
    table.bound = 40
    want, gathered = attend(q, k, v, nk, nv, [40, 9], new)
    w = torch.full((2, 2, table.capacity), 0.25, device=DEV)
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=torch.tensor(new, device=DEV), weights=w)
    assert ((got.cpu().double() - want).abs() <= allowed(want, dtype, v, nv)).all()
    for b, seen in enumerate((40, 9)):
        at = torch.cat((torch.arange(seen), lengths[b] + torch.arange(new[b])))
        add = gathered[b, :, :seen + new[b]]
        assert ((w[b, :, at.to(DEV)].cpu().double() - 0.25 - add).abs() <= 2.0 ** -23 * (add + 0.25) + FP32 * add + 1e-7).all()
        rest = torch.ones(table.capacity, dtype=torch.bool)
        rest[at] = False
        assert (w[b, :, rest.to(DEV)] == 0.25).all()
    # a count at and past the table's end: new tokens have no place
    table.counts.copy_(torch.tensor([table.capacity, table.capacity + 100]))
    w.fill_(0.25)
    paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=torch.tensor(new, device=DEV), weights=w)
    assert (w[:, :, 40:] == 0.25).all()


def test_float32_elements_near_the_largest():
    """Finite elements that bf16 would round to infinity: a value that a row does not see
    does not reach it, one of small weight adds what it is worth, and a key's product with
    a small query element is a logit like any other."""
    gen = torch.Generator().manual_seed(31)
    big = torch.finfo(torch.float32).max
    base = torch.randn(128, generator=gen)
    cache, table = make([0], 1, max_tokens=64)
    for rows, group in ((40, 1), (9, 2), (90, 4)):  # waves that share tokens, and that do not
        q = base + 0.1 * torch.randn(1, group, rows, 128, generator=gen)
        nk, nv = (torch.randn(1, 1, rows, 128, generator=gen) for _ in range(2))
        nk[0, 0, 5] = -4 * base  # weights of e^-40 and less
        nv[0, 0, 5, 3], nv[0, 0, 5, 70], nv[0, 0, 5, 100] = big, -big, 3.397e38
        want, _ = attend(q, torch.zeros(1, 1, 0, 128, dtype=torch.float64), torch.zeros(1, 1, 0, 128, dtype=torch.float64),
                         nk, nv, [0], [rows])
        got = paged.paged_chunk_attention(q.to(DEV), cache, 0, table, nk.to(DEV), nv.to(DEV)).cpu().double()
        # a weight's own error: 24 steps of sums up to 512, times 1 / sqrt(128)
        assert ((got - want).abs() <= FP32 + 24 * 2.0 ** -14 / math.sqrt(128) * want.abs()).all()
        assert got[:, :, :5].abs().max() < 10
        nv = torch.randn(1, 1, rows, 128, generator=gen)
        q[..., 0], nk[0, 0, 2, 0], nk[0, 0, 3, 0] = 2.0 ** -126, big, -big
        want, _ = attend(q, torch.zeros(1, 1, 0, 128, dtype=torch.float64), torch.zeros(1, 1, 0, 128, dtype=torch.float64),
                         nk, nv, [0], [rows])
        w = torch.zeros(1, 1, table.capacity, device=DEV)
        got = paged.paged_chunk_attention(q.to(DEV), cache, 0, table, nk.to(DEV), nv.to(DEV), weights=w).cpu().double()
        assert ((got - want).abs() <= FP32 * 4).all()
        assert w.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dims", (16, 32, 64))
@pytest.mark.parametrize("rows", (1, 6, 40, 100))
@pytest.mark.parametrize("weights", ("all", "none"))
def test_chunks_over_wide_value_groups(dtype, dims, rows, weights):
    """Cached value groups up to the format's whole range, in tokens that count like any
    other and in tokens whose weight is 2^-40 and less, which change nothing."""
    gen = torch.Generator().manual_seed(50 + dims)
    cache, table = make([300], 2, group=dims, max_tokens=300 + rows)
    v, far = wide_values(57344.0, dtype, gen, 300, 1 if weights == "all" else 9)
    base = torch.randn(128, generator=gen)
    k = torch.randn(1, 2, 300, 128, generator=gen)
    if weights == "none":  # logits below -30
        k[:, :, far] = -4 * base
    k = k.to(dtype)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(300)
    k, v = dequantised(k, dims), dequantised(v, dims)
    q = (base + 0.1 * torch.randn(1, 8, rows, 128, generator=gen)).to(dtype).to(DEV)
    nk, nv = (torch.randn(1, 2, rows, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want, _ = attend(q, k, v, nk, nv, [300], [rows])
    top = v.abs().max() if weights == "all" else max(v[:, :, ~far].abs().max(), nv.abs().max().cpu().double())
    # as `allowed`, with FP32 for values up to 5, and the wide tokens' own weights, below 2^-40 of 57344 each
    bound = torch.finfo(dtype).eps / 2 * want.abs() + FP32 * top / 5 + 300 * 57344 * 2.0 ** -40
    bound = bound + top * {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 3 * 2.0 ** -11 + 2 * 2.0 ** -8}[dtype]
    tokens = torch.tensor([rows], device=DEV)
    w = torch.zeros(1, 2, table.capacity, device=DEV)
    for kw in (dict(tokens=tokens), dict(tokens=tokens, weights=w)):
        got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, **kw).cpu().double()
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dims", (16, 32, 64))
@pytest.mark.parametrize("dtype", DTYPES)
def test_chunks_over_wide_key_groups(dtype, dims):
    """Cached key groups up to the format's whole range under small queries."""
    gen = torch.Generator().manual_seed(60 + dims)
    cache, table = make([300], 2, group=dims, max_tokens=340)
    k, _ = wide_values(57344.0, torch.float32, gen, 300, 1)
    v = torch.randn(1, 2, 300, 128, generator=gen)
    paged.write_tokens(cache, 0, table, k.to(DEV), v.to(DEV))
    table.advance(300)
    k, v = dequantised(k, dims), dequantised(v, dims)
    q = (torch.randn(1, 8, 40, 128, generator=gen) * 2e-5).to(dtype).to(DEV)
    nk, nv = (torch.randn(1, 2, 40, 128, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want, gathered = attend(q, k, v, nk, nv, [300], [40])
    # a logit's error: bf16 rows without weights have keys in fp16, half a step (2^-11) each; else the fp32 sums',
    # some 36 steps (2^-23) of partial sums up to that of the products' magnitudes; weights that are off by e each move a
    # mean by 2 e of the largest value
    size = float((q.cpu().double().abs() @ k.abs().amax(2).amax(1)[0][:, None]).max()) / math.sqrt(128)
    for weights in (None, torch.zeros(1, 2, table.capacity, device=DEV)):
        e = size * (2.0 ** -11 if dtype == torch.bfloat16 and weights is None else 80 * 2.0 ** -24)
        got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, weights=weights).cpu().double()
        bound = allowed(want, dtype, v, nv) + 2 * e * float(v.abs().max())
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
    total = (weights[:, :, :340].cpu().double() - gathered).abs()
    assert (total <= (2 * e + FP32) * gathered + 1e-7).all()


# Norm of the error over the norm of the result, of independent roundings: the result's own,
# half a step of numbers whose mantissas spread evenly over their logarithm, 0.735 step / sqrt(12)
# (1.66e-3 in bf16, 2.07e-4 in fp16); as much again where each weight (bf16 rows on new tokens) or
# each cached value (fp16 rows) is rounded to the same type; for bf16 rows on cached tokens fp16
# weights (truncated: 0.735 2^-10 / sqrt(12) = 2.07e-4 about their mean, which the sum has too),
# values (2.07e-4) and, without gathered weights, keys, 2.07e-4 of each product of a logit of up to
# 3 in magnitude: 4e-4 at most in all.  fp32: some 40 roundings of partial sums of logits about 4, half a step of 8
# (2^-22 / sqrt(3) each), 9e-7, and the exponent's, 3e-7.  A fifth of that on top.
def error_norm(dtype, cached, new):
    own = {torch.bfloat16: 1.66e-3, torch.float16: 2.07e-4, torch.float32: 0.0}[dtype]
    parts = [own, 1e-6]
    if dtype == torch.bfloat16:
        parts += [own if new else 0.0, 4e-4 if cached else 0.0]
    if dtype == torch.float16:
        parts += [own if cached else 0.0]
    return 1.2 * math.hypot(*parts)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gather", (False, True))
@pytest.mark.parametrize("lengths,new", [([5000], [6]), ([3000], [13]), ([2000], [30]), ([4000], [70]), ([0], [40]),
                                         ([0], [700]), ([3000, 2500, 2200, 2800], [1, 1, 1, 90])], ids=str)
def test_error_norms(dtype, gather, lengths, new):
    """The norm of the error of each sequence's rows, which one token left out (a norm of about
    one over the root of the tokens) or a rounding to fewer bits breaks; a mixed batch of decoding
    sequences and a prompt's piece among them."""
    cache, table, k, v, q, nk, nv = setup(lengths, new, 2, 4, dtype, spread=1.0, seed=sum(lengths) + 31)
    want, _ = attend(q, k, v, nk, nv, lengths, new)
    w = torch.zeros(len(lengths), 2, table.capacity, device=DEV) if gather else None
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, tokens=torch.tensor(new, device=DEV), weights=w)
    got = got.cpu().double()
    for b, n in enumerate(new):
        err = float((got[b, :, :n] - want[b, :, :n]).norm() / want[b, :, :n].norm())
        assert err <= error_norm(dtype, lengths[b] > 0, lengths[b] == 0), (b, err)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_both_ways(dtype):
    """One token a sequence laid out as a decode step's is the decode step, to the bit; with
    ``tokens``, more query heads than that has or other strides it is a chunk.  Both are
    the formula's."""
    lengths = [300, 0, 1029]
    cache, table, k, v, q, nk, nv = setup(lengths, [1, 1, 1], 2, 4, dtype, spread=1.0, seed=6)
    want, _ = attend(q, k, v, nk, nv, lengths, [1, 1, 1])
    bound = allowed(want, dtype, v, nv)
    step = paged.paged_attention_step(q[:, :, 0].contiguous(), cache, 0, table, nk[:, :, 0].contiguous(),
                                      nv[:, :, 0].contiguous())
    assert torch.equal(paged.paged_chunk_attention(q, cache, 0, table, nk, nv)[:, :, 0], step)
    out = torch.empty(3, 8, 1, 256, dtype=dtype, device=DEV)[..., :128]
    for kw in (dict(tokens=torch.ones(3, dtype=torch.int64, device=DEV)), dict(out=out)):
        got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv, **kw)
        assert ((got.cpu().double() - want).abs() <= bound).all()
        for b in (0, 2):
            assert (got[b].cpu().double() - want[b]).norm() <= error_norm(dtype, True, False) * want[b].norm()
    cache, table, k, v, q, nk, nv = setup(lengths, [1, 1, 1], 1, 20, dtype, seed=7)
    want, _ = attend(q, k, v, nk, nv, lengths, [1, 1, 1])
    got = paged.paged_chunk_attention(q, cache, 0, table, nk, nv).cpu().double()
    assert ((got - want).abs() <= allowed(want, dtype, v, nv)).all()


@pytest.mark.parametrize("batch,large", [(5, False), (5, True), (150, False), (150, True)])
def test_evict_passes_over_shares_that_do_not_fit(batch, large):
    """A sequence that needs more free pages than are left stays whole, and those behind it
    still take theirs; in one workgroup's plan and in several launches'."""
    left, cut = 4 if batch == 5 else 151, []  # (the last of 151 fits past the first 64 sequences)
    cache, table, w = filled_pool([320 if batch == 5 else 130] * batch, 1, page=32, layers=1,
                                  spare=17_000 if large else left, seed=32)
    table.refs[torch.nonzero(table.refs == 0)[left:, 0]] = 3  # held elsewhere
    shared = [5, 2, 0, 4, 1] if batch == 5 else [(7 * b) % 5 for b in range(batch)]
    for b, n in enumerate(shared):
        table.refs[table.table[b, :n].long()] = 2  # held elsewhere too
    keep = 150 if batch == 5 else 100
    stay = -(-keep // 32)
    for b, n in enumerate(shared):
        if min(n, stay) <= left:
            left -= min(n, stay)
            cut.append(b)
    assert 0 < len(cut) < batch
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check_evict(cache, table, w, keep, 20, cut=cut, status=status)
    assert int(status) == 4


def test_pages_given_back_serve_the_next_call():
    """Free pages are those that were free before the call: what it gives back itself
    lets a second call cut the sequences that the first had to leave."""
    cache, table, w = filled_pool([320, 320], 2, page=32, spare=0, seed=33)
    table.refs[table.table[0, :2].long()] = 2
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check_evict(cache, table, w, 150, 20, cut=(1,), out=table, weights_out=w, status=status)
    assert int(status) == 4
    status.zero_()
    check_evict(cache, table, w, 150, 20, cut=(0,), out=table, weights_out=w, status=status)
    assert int(status) == 0 and table.counts.tolist() == [150, 150]


@pytest.mark.parametrize("dtype", DTYPES)
def test_proposed_tokens_of_which_some_are_accepted(dtype):
    """Proposals verified without gathering, then the accepted ones' weights gathered before
    they are advanced over: the sums are those of the rows that stay, whatever was
    proposed beside them, and the next proposals' places begin at zero."""
    kvh, group, page = 2, 2, 32
    cache = paged.allocate_paged_cache(1, 40, kvh, page_tokens=page, dim_group_size=32, device=DEV)
    table = paged.PageTable.create(2, 256, cache)
    w = paged.allocate_token_weights(cache, table)
    ws, status = popkv.LayerStepWorkspace(), torch.zeros(1, dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(34)
    held = [[torch.zeros(kvh, 0, 128, dtype=torch.float64) for _ in range(2)] for _ in range(2)]  # [b][k, v]
    sums = [torch.zeros(kvh, 0, dtype=torch.float64) for _ in range(2)]
    for proposed, accepted in (([40, 33], [40, 33]), ([6, 6], [2, 6]), ([6, 4], [1, 1]), ([6, 6], [6, 3])):
        most = max(proposed)
        bound = table.bound + most
        piece = torch.tensor(proposed, device=DEV)
        q, k, v = (torch.randn(2, h, most, 128, generator=gen).to(dtype).to(DEV) for h in (kvh * group, kvh, kvh))
        paged.reserve_pages(table, piece, bound=bound, status=status, out=table)
        out = paged.paged_chunk_attention(q, cache, 0, table, k, v, tokens=piece, workspace=ws)
        paged.write_tokens(cache, 0, table, k, v, tokens=piece, status=status)
        took = torch.tensor(accepted, device=DEV)
        paged.paged_chunk_attention(q, cache, 0, table, k, v, tokens=took, weights=w[0], workspace=ws)
        table.advance(took, bound=bound)
        kq, vq = dequantised(k, 32), dequantised(v, 32)
        for b, m in enumerate(accepted):
            ck, cv = held[b]
            n = ck.shape[1]
            want, _ = attend(q[b:b + 1], ck[None], cv[None], k[b:b + 1], v[b:b + 1], [n], [proposed[b]])
            _, add = attend(q[b:b + 1], ck[None], cv[None], k[b:b + 1], v[b:b + 1], [n], [m])
            bound_b = allowed(want, dtype, cv[None], v[b:b + 1])
            assert ((out[b:b + 1].cpu().double() - want).abs() <= bound_b).all()
            sums[b] = torch.cat((sums[b], torch.zeros(kvh, m)), 1) + add[0, :, :n + m]
            held[b] = [torch.cat((ck, kq[b, :, :m]), 1), torch.cat((cv, vq[b, :, :m]), 1)]
            have = w[0, b].cpu().double()
            assert ((have[:, :n + m] - sums[b]).abs() <= 2 * FP32 * (1 + sums[b])).all()
            assert not have[:, n + m:].any()
    assert int(status) == 0 and table.counts.tolist() == [x[0].shape[1] for x in held]
