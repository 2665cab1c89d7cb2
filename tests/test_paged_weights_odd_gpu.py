"""Keys' attention weights where scores are not finite: a row adds to the keys that it sees and to no other, in the form
of stored products (few rows) as in that of products formed again."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import BF16, DEV, Cache, check_attention, gen, ints, randn, starts_of

pytestmark = pytest.mark.gpu

INF = float("inf")


def _call(cache, q, nq, lens, before, causal=True):
    w = torch.full_like(before, 77.0)
    o, m, l = P.paged_attention(q, cache.k, cache.v, cache.table, ints(lens), starts_of(nq), 0.1, causal=causal,
                                return_ml=True, weights=before, weights_out=w)
    return o, m, l, w


def _sums(cache, seed):
    return torch.rand((len(cache.lens), cache.Hkv, cache.table.shape[1] * cache.page), generator=gen(seed), device=DEV)


# new tokens, key heads, query heads: 32 rows a key head or fewer (stored), more, and no multiple of 32 of either
ROWS = [([5], [70], 2, 2), ([1, 3], [300, 700], 2, 8), ([37], [400], 1, 3), ([150, 7], [400, 90], 2, 4),
        ([2050], [2300], 1, 1)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,lens,Hkv,Hq", ROWS)
def test_keys_whose_scores_are_all_minus_infinity_get_nothing(nq, lens, Hkv, Hq, d, causal):
    """One infinity in a key, against queries that are positive there: its weight is exp(-inf) = 0, as if it were masked.
    One of the keys lies before the new tokens and one among them."""
    cache = Cache(lens, Hkv, d, 16, seed=sum(nq) + d)
    q = randn(gen(1), sum(nq), Hq, d)
    q[..., 3] = q[..., 3].abs() + 0.5
    keep = []
    for b, (n, length) in enumerate(zip(nq, lens)):
        keep.append(torch.ones(length, dtype=torch.bool, device=DEV))
        for j in ((length - n) // 2, length - (n + 1) // 2):
            p, s = (t[j] for t in cache.where(b, length))
            cache.k[p, :, s] = 0
            cache.k[p, :, s, 3] = -INF
            keep[b][j] = False
    before = _sums(cache, 5)
    o, m, l, w = _call(cache, q, nq, lens, before, causal)
    check_attention(cache, q, nq, lens, o, scale=0.1, causal=causal, m=m, l=l, weights=w, before=before, keep=keep)
