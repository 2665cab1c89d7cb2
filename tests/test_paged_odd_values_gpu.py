"""Values that are not finite, of seen keys whose weight is far below what fp32 holds."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import DEV, Cache, check_attention, gen, ints, randn, starts_of

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,length,at", [(5, 70, 64), (5, 70, 66), (5, 1500, 1496), (40, 300, 258), (150, 400, 250), (150, 400, 399),
                                          (64, 64, 0), (130, 130, 127)])
def test_a_seen_value_counts_whatever_its_weight(nq, length, at, d, causal):
    """A key with a score 160 below the others', so that its weight, e^-160, is 0 in fp32: the rows that see it have its
    infinities and NaN all the same, the others and the other columns do not.  (Its 32 keys hold one that some row does not see,
    or the last of all.)"""
    cache = Cache([length], 2, d, 16, seed=nq)
    q = randn(gen(3), nq, 4, d)
    q[..., 5] = 8.0
    p, s = (t[at] for t in cache.where(0, length))
    cache.k[..., 5] = torch.where(torch.isnan(cache.k[..., 5]), cache.k[..., 5], 0.0)
    cache.k[p, :, s] = 0
    cache.k[p, :, s, 5] = -200.0
    o, m, l = P.paged_attention(q, cache.k, cache.v, cache.table, ints([length]), starts_of([nq]), 0.1, causal=causal,
                                return_ml=True)
    check_attention(cache, q, [nq], [length], o, scale=0.1, causal=causal, m=m, l=l)
    odd = {1: INF, 2: -INF, d - 1: float("nan")}
    for col, x in odd.items():
        cache.v[p, :, s, col] = x
    o2, m2, l2 = P.paged_attention(q, cache.k, cache.v, cache.table, ints([length]), starts_of([nq]), 0.1, causal=causal,
                                   return_ml=True)
    assert torch.equal(m2, m) and torch.equal(l2, l)
    sees = torch.ones(nq, dtype=torch.bool, device=DEV) if not causal else torch.arange(nq, device=DEV) + length - nq >= at
    hit = torch.zeros(o.shape, dtype=torch.bool, device=DEV)
    hit[:, :, list(odd)] = sees[:, None, None]
    assert torch.equal(o2[~hit], o[~hit])
    assert not torch.isfinite(o2[hit]).any()
