"""Chunks over the paged 4-bit cache and its eviction where they can go wrong: a bound
behind the counts, elements at the end of a type's range, the norm of the errors, one
token both ways, shares of free pages that do not fit, proposals that are rejected."""
from __future__ import annotations

import pytest
import torch

from popkv_amd import paged

from test_gpu_paged_chunk import DEV, DTYPES, FP32, allowed, attend, setup

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
