"""Keys' attention weights where scores are not finite: a row adds to the keys that it sees and to no other, in the form
of stored products (few rows) as in that of products formed again."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import DEV, Cache, check_attention, gen, ints, randn, starts_of

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


# new tokens, keys, key and query heads, the token whose query is not finite
@pytest.mark.parametrize("x", [float("nan"), INF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,length,Hkv,Hq,token", [(5, 70, 2, 4, 2), (12, 900, 2, 4, 0), (150, 400, 2, 2, 70),
                                                    (150, 150, 1, 3, 40), (64, 1000, 2, 4, 33), (90, 91, 1, 1, 0)])
def test_a_query_that_is_not_finite_reaches_only_the_keys_it_sees(nq, length, Hkv, Hq, token, d, x):
    """The sums of later tokens' keys, and of the other key heads, are the same bits as without it."""
    cache = Cache([length], Hkv, d, 16, seed=nq + d)
    q = randn(gen(2), nq, Hq, d)
    before = _sums(cache, 5)
    o, m, l, w = _call(cache, q, [nq], [length], before)
    check_attention(cache, q, [nq], [length], o, scale=0.1, m=m, l=l, weights=w, before=before)
    q[token, Hq // Hkv - 1] = x  # the last query head of the first key head: every score is NaN or infinite
    o2, m2, l2, w2 = _call(cache, q, [nq], [length], before)
    seen = length - nq + token + 1
    assert torch.isnan(o2[token, Hq // Hkv - 1]).all() and torch.isnan(w2[0, 0, :seen]).all()
    assert torch.equal(w2[0, 0, seen:], w[0, 0, seen:]) and torch.equal(w2[0, 1:], w[0, 1:])
    rest = torch.ones((nq, Hq), dtype=torch.bool, device=DEV)
    rest[token, Hq // Hkv - 1] = False
    for a, b in ((o2, o), (m2, m), (l2, l)):
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1])
@pytest.mark.parametrize("nq,length", [(1, 200), (2, 3000), (90, 200)])
def test_keys_of_an_invalid_page_get_nothing_from_any_row(nq, length, bad):
    """Also from a row whose query is NaN: such keys count as masked."""
    cache = Cache([length], 2, 128, 16, seed=4)
    good = ints([0, 5, 6])  # pages, none of a new token's key
    q = randn(gen(1), nq, 4, 128)
    q[nq // 2, 1] = float("nan")
    before = _sums(cache, 5)
    keys = (16 * good[:, None] + torch.arange(16, device=DEV)).flatten()
    keys = keys[keys < length - nq]
    cache.table[0, good.long()] = bad
    *_, w = _call(cache, q, [nq], [length], before)
    assert torch.equal(w[0][:, keys], before[0][:, keys])
    rest = torch.ones(length - nq, dtype=torch.bool, device=DEV)
    rest[keys] = False
    assert torch.isnan(w[0, 0, :length - nq][rest]).all() and torch.isfinite(w[0, 1, :length]).all()
