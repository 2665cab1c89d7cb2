"""The om carriers of paged attention, combined over two caches by ``om_compose``, against float64 over all keys."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import kernels as K
from catopt_amd import paged as P
from paged_ref import BF16, DEV, HALF_STEP, Cache, attention, gen, ints, randn, starts_of

pytestmark = pytest.mark.gpu

SCALE = 0.1


def _carrier(cache, q, nq, causal):
    o, m, l = P.paged_attention(q, cache.k, cache.v, cache.table, ints(cache.lens), starts_of(nq), SCALE, causal=causal,
                                return_ml=True)
    return m, l, o.float() * l[..., None]


# the new tokens of each sequence, its keys in a cache of prefixes, and in one of its own (new tokens included)
CASES = [([1, 1, 1], [300, 0, 7], [1, 20, 900]), ([5, 2], [0, 1], [70, 2]), ([150, 40], [200, 0], [150, 300]),
         ([1], [5000], [3000])]


@pytest.mark.parametrize("d,Hq,Hkv", [(64, 4, 4), (128, 8, 2)])
@pytest.mark.parametrize("nq,prefix,own", CASES)
def test_two_caches_compose(nq, prefix, own, d, Hq, Hkv):
    """A prefix that every new token sees whole, and the sequence's own keys behind it.  Each part's result is rounded to
    bf16 (half a step of its own size), its terms as in one call; the statistics are fp32."""
    a, b = Cache(prefix, Hkv, d, 16, seed=1), Cache(own, Hkv, d, 32, seed=2)
    q = randn(gen(3), sum(nq), Hq, d)
    fa, fb = _carrier(a, q, nq, False), _carrier(b, q, nq, True)
    m, l, num = K.om_compose(fa, fb)
    o = num / l[..., None]
    at = 0
    for i, n in enumerate(nq):
        rows = slice(at, at + n)
        at += n
        ka, va, kb, vb = a.rows(a.k, i), a.rows(a.v, i), b.rows(b.k, i), b.rows(b.v, i)
        r = attention(q[rows], torch.cat([ka, kb], 1), torch.cat([va, vb], 1), SCALE)
        parts = [attention(q[rows], ka, va, SCALE, False), attention(q[rows], kb, vb, SCALE)]
        # the parts' shares of the row's sum, and their results' sizes
        share = [torch.where(p["l"] > 0, p["l"] * torch.exp(p["m"] - r["m"]) / r["l"], 0.0) for p in parts]
        sizes = sum(s[..., None] * torch.where(p["l"][..., None] > 0, p["o"], 0.0).abs() for s, p in zip(share, parts))
        # exp of a difference of maxima: their own errors es, and steps of fp32 of their size
        es = torch.expm1(4 * r["es"] + 2.0 ** -21 * (1 + r["m"].abs())) + (prefix[i] + own[i] + 64) * 2.0 ** -24
        gm, gl, go = m[rows].double().t(), l[rows].double().t(), o[rows].double().transpose(0, 1)
        assert ((gm - r["m"]).abs() <= r["es"] + 1e-37).all()
        assert ((gl - r["l"]).abs() <= es * r["l"] * 1.01).all()
        tol = ((HALF_STEP[BF16] + es)[..., None] * r["mag"] + (HALF_STEP[BF16] + es[..., None]) * sizes) * 1.01 + 1e-37
        err = (go - r["o"]).abs()
        assert (err <= tol).all(), (i, float((err / tol).max()))


@pytest.mark.parametrize("nq,prefix,own", [([3], [1], [40]), ([70], [1], [300]), ([3], [600], [1500])])
def test_a_score_that_is_nan_stays_in_the_carrier(nq, prefix, own):
    """The maximum of a row that sees a NaN is NaN, as everywhere in the om algebra, which leaves out a part whose maximum
    is -inf: a part whose only scores are NaN is not an empty one."""
    a, b = Cache(prefix, 2, 64, 16, seed=1), Cache(own, 2, 64, 16, seed=2)
    q = randn(gen(3), sum(nq), 4, 64)
    p, s = (t[prefix[0] // 2] for t in a.where(0, prefix[0]))
    a.k[p, 0, s, 9] = float("nan")  # a key of the first key head: its two query heads see it
    q[1, 3, 0] = float("nan")  # and one query of the second
    fa, fb = _carrier(a, q, nq, False), _carrier(b, q, nq, True)
    nan = torch.zeros((sum(nq), 4), dtype=torch.bool, device=DEV)
    nan[1, 3] = True
    assert torch.equal(torch.isnan(fb[0]), nan) and torch.equal(torch.isnan(fb[1]), nan)
    nan[:, :2] = True
    assert torch.equal(torch.isnan(fa[0]), nan) and torch.equal(torch.isnan(fa[1]), nan)
    m, l, num = K.om_compose(fa, fb)
    o = num / l[..., None]
    assert torch.isnan(o[nan]).all() and torch.isfinite(o[~nan]).all()
    assert torch.isnan(m[nan]).all() and torch.isfinite(m[~nan]).all()


def test_empty_and_infinite_rows():
    """No key: (-inf, 0).  A score of +inf is the maximum, and its row's result NaN."""
    b = Cache([20, 0], 2, 64, 16, seed=2)
    q = randn(gen(3), 3, 2, 64)
    q[..., 0] = q[..., 0].abs() + 0.5
    p, s = (t[4] for t in b.where(0, 20))
    b.k[p, 0, s] = 0
    b.k[p, 0, s, 0] = float("inf")
    m, l, num = _carrier(b, q, [2, 1], True)
    assert torch.isposinf(m[:2, 0]).all() and torch.isnan(l[:2, 0]).all() and torch.isnan(num[:2, 0]).all()
    assert torch.isfinite(m[:2, 1]).all() and torch.isfinite(l[:2, 1]).all()
    assert torch.isneginf(m[2]).all() and (l[2] == 0).all()
