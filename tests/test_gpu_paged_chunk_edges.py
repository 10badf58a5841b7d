"""Chunks over the paged 4-bit cache and its eviction where they can go wrong: a bound
behind the counts, elements at the end of a type's range, the norm of the errors, one
token both ways, shares of free pages that do not fit, proposals that are rejected."""
from __future__ import annotations

import math

import pytest
import torch

from popkv_amd import paged, popkv

from test_gpu_paged import dequantised, make
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
    proposed beside them, and the next round's tokens begin at zero."""
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
