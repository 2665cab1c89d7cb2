"""Eviction by accumulated attention weight: the kept keys by their definition, the moved rows bit for bit."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import BF16, DEV, Cache, evict, gen, ints, randn, starts_of, check_attention

pytestmark = pytest.mark.gpu


def _weights(cache, seed, ties=True):
    w = torch.rand((len(cache.lens), cache.Hkv, cache.table.shape[1] * cache.page), generator=gen(seed), device=DEV)
    return torch.floor(w * 16) / 4 if ties else w


def _check(cache, w, budget, recent, kept, lens, w_to, out):
    for b, n in enumerate(cache.lens):
        m = min(n, budget)
        assert int(lens[b]) == m
        for h in range(cache.Hkv):
            want = evict(w[b, h], n, budget, recent)
            assert kept[b, h, :m].tolist() == want, (b, h)
            assert (kept[b, h, m:] == -1).all()
            idx = ints(want, torch.int64)
            assert torch.equal(torch.nan_to_num(w_to[b, h, :m], 5.0), torch.nan_to_num(w[b, h][idx], 5.0))
            for src, dst in ((cache.k, out.k), (cache.v, out.v)):
                assert torch.equal(out.rows(dst, b, m)[h], cache.rows(src, b)[h][idx]), (b, h)


# lengths, key heads, head dim, page, page of the output, budget, recent
CASES = [([100], 2, 64, 16, 16, 40, 8), ([1], 1, 8, 8, 8, 1, 0), ([5, 0, 17], 3, 128, 16, 8, 16, 16),
         ([2100, 40, 1024, 1025], 2, 128, 16, 64, 300, 33), ([3000], 1, 64, 5, 7, 1023, 0),
         ([700, 699], 2, 96, 32, 16, 2000, 50), ([4097], 2, 64, 64, 16, 4096, 1), ([333], 4, 16, 8, 16, 1, 1)]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("lens,Hkv,d,page,page_out,budget,recent", CASES)
def test_kept_keys_and_rows(lens, Hkv, d, page, page_out, budget, recent, dtype):
    cache = Cache(lens, Hkv, d, page, seed=budget, dtype=dtype, slot_major=page % 16 == 5)
    out = Cache([budget] * len(lens), Hkv, d, page_out, seed=1, dtype=dtype)
    spare = out.k[out.free.long()].clone()
    for ties in (True, False):
        w = _weights(cache, budget, ties)
        kept, new, w_to = P.paged_evict(cache.k, cache.v, cache.table, ints(lens), w, out.table, budget, recent,
                                        k_out=out.k, v_out=out.v)
        _check(cache, w, budget, recent, kept, new, w_to, out)
        for b, n in enumerate(lens):
            assert (w_to[b, :, min(n, budget):] == 0).all()
    assert torch.equal(torch.nan_to_num(out.k[out.free.long()], 3.0), torch.nan_to_num(spare, 3.0))


def test_rows_behind_the_last_kept_key_stay():
    cache, out = Cache([30], 2, 64, 16), Cache([64], 2, 64, 16, seed=2)
    before = out.rows(out.k, 0)
    w, w_to = _weights(cache, 0), torch.full((1, 2, 70), 8.0, device=DEV)
    P.paged_evict(cache.k, cache.v, cache.table, ints([30]), w, out.table, 64, 4, k_out=out.k, v_out=out.v,
                  weights_out=w_to)
    assert torch.equal(out.rows(out.k, 0)[:, 30:], before[:, 30:])
    assert (w_to[..., 30:] == 8).all()


def test_odd_weights():
    """NaN ranks above every number, zeros of both signs tie, infinities and negative numbers take their places."""
    n = 200
    cache, out = Cache([n], 2, 64, 16), Cache([64], 2, 64, 16, seed=2)
    w = torch.zeros((1, 2, cache.table.shape[1] * 16), device=DEV)
    w[0, 0, ::3] = -0.0
    w[0, 0, 150] = float("nan")
    w[0, 0, 60], w[0, 0, 61] = float("inf"), float("-inf")
    w[0, 1] = -torch.rand(w.shape[2], generator=gen(1), device=DEV)
    w[0, 1, 7] = float("-inf")
    w[0, 1, 9], w[0, 1, 199] = 1e-42, float("nan")  # a denormal above the negative ones
    for budget, recent in ((1, 0), (3, 1), (40, 4), (64, 64)):
        kept, new, w_to = P.paged_evict(cache.k, cache.v, cache.table, ints([n]), w, out.table, budget, recent,
                                        k_out=out.k, v_out=out.v)
        _check(cache, w, budget, recent, kept, new, w_to, out)


def test_weights_in_place_and_the_same_pool():
    n, budget = 3000, 500
    cache = Cache([n, 600], 2, 64, 16, seed=5)
    extra = 2 * -(-budget // 16)
    k, v = (torch.cat([t, torch.zeros((extra, *t.shape[1:]), dtype=t.dtype, device=DEV)]) for t in (cache.k, cache.v))
    to = torch.arange(cache.n_pages, cache.n_pages + extra, device=DEV, dtype=torch.int32).view(2, -1)
    w = _weights(cache, 3)
    same = w.clone()
    kept, new, w_to = P.paged_evict(k, v, cache.table, ints([n, 600]), same, to, budget, 64, weights_out=same)
    assert w_to is same
    out = Cache([budget, budget], 2, 64, 16)
    out.k, out.v, out.table = k, v, to
    _check(cache, w, budget, 64, kept, new, same, out)
    assert torch.equal(same[:, :, budget:], w[:, :, budget:])


def test_invalid_pages_and_lengths():
    cache, out = Cache([64, 64], 1, 64, 16), Cache([32, 32], 1, 64, 16, seed=2)
    w = torch.arange(cache.table.shape[1] * 16, device=DEV).float().expand(2, 1, -1).contiguous()
    for bad in (-1, cache.n_pages, 2 ** 31 - 1, -2 ** 31):
        table, to = cache.table.clone(), out.table.clone()
        table[0, 3], to[1, 1] = bad, bad
        ko, vo = out.k.clone(), out.v.clone()
        P.paged_evict(cache.k, cache.v, table, ints([64, 64]), w, to, 32, 0, k_out=ko, v_out=vo)
        assert (ko[out.table[0, 1].long()] == 0).all()  # its keys' rows move as zeros
        assert torch.equal(ko[out.table[0, 0].long(), :, :], cache.k[cache.table[0, 2].long()])
        assert torch.equal(ko[out.table[1, 1].long()], out.k[out.table[1, 1].long()])  # the write is dropped
    kept, new, _ = P.paged_evict(cache.k, cache.v, cache.table, ints([2 ** 31 - 1, -4]), w, out.table, 32, 0,
                                 k_out=out.k, v_out=out.v)
    cap = cache.table.shape[1] * 16
    assert new.tolist() == [32, 0] and kept[0, 0].tolist() == list(range(cap - 32, cap)) and (kept[1] == -1).all()


def test_keys_past_the_registers_of_a_workgroup():
    """Tables of more than 16384 keys read their weights again in every sweep; in place too."""
    lens, budget = [20000, 16385, 300], 3000
    cache, out = Cache(lens, 1, 8, 16, seed=4), Cache([budget] * 3, 1, 8, 16, seed=2)
    for ties in (True, False):
        w = _weights(cache, 7, ties)
        same = w.clone()
        kept, new, w_to = P.paged_evict(cache.k, cache.v, cache.table, ints(lens), w, out.table, budget, 100, k_out=out.k,
                                        v_out=out.v)
        _check(cache, w, budget, 100, kept, new, w_to, out)
        kept2, _, _ = P.paged_evict(cache.k, cache.v, cache.table, ints(lens), same, out.table, budget, 100, k_out=out.k,
                                    v_out=out.v, weights_out=same)
        assert torch.equal(kept, kept2)
        for b, n in enumerate(lens):
            m = min(n, budget)
            assert torch.equal(same[b, :, :m], w_to[b, :, :m]) and torch.equal(same[b, :, m:], w[b, :, m:])


@pytest.mark.parametrize("lens,Hkv,budget", [([900], 1, 64), ([900], 1, 65), ([3000, 20], 3, 1000), ([600] * 200, 2, 130),
                                             ([17000], 2, 4000)])
def test_parts_of_a_head(lens, Hkv, budget):
    """Heads whose kept rows one workgroup moves, and several; the weights apart and in place."""
    cache, out = Cache(lens, Hkv, 16, 16, seed=budget), Cache([budget] * len(lens), Hkv, 16, 16, seed=2)
    w = _weights(cache, 5)
    same = w.clone()
    args = (cache.k, cache.v, cache.table, ints(lens))
    kept, new, w_to = P.paged_evict(*args, w, out.table, budget, 7, k_out=out.k, v_out=out.v)
    _check(cache, w, budget, 7, kept, new, w_to, out)
    ko, vo = torch.zeros_like(out.k), torch.zeros_like(out.v)
    P.paged_evict(*args, same, out.table, budget, 7, k_out=ko, v_out=vo, weights_out=same)
    for b, n in enumerate(lens):
        m = min(n, budget)
        assert torch.equal(same[b, :, :m], w_to[b, :, :m])
        assert torch.equal(out.rows(ko, b, m), out.rows(out.k, b, m)) and torch.equal(out.rows(vo, b, m), out.rows(out.v, b, m))


def test_captured():
    lens = [500, 260]
    cache, out = Cache(lens, 2, 64, 16), Cache([128, 128], 2, 64, 16, seed=2)
    w, kv = _weights(cache, 1), ints(lens)
    w_to = torch.zeros((2, 2, 128), device=DEV)
    call = lambda: P.paged_evict(cache.k, cache.v, cache.table, kv, w, out.table, 128, 16, k_out=out.k,  # noqa: E731
                                 v_out=out.v, weights_out=w_to)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, new, _ = call()
    for step in range(4):
        w.copy_(_weights(cache, 20 + step))
        cache.lens = [500 - 100 * step, 260 - 60 * step]
        kv.copy_(ints(cache.lens))
        g.replay()
        torch.cuda.synchronize()
        _check(cache, w, 128, 16, kept, new, w_to, out)


def test_refusals():
    cache, out = Cache([64], 2, 64, 16), Cache([32], 2, 64, 16, seed=2)
    w = _weights(cache, 0)

    def bad(exc, k=cache.k, v=cache.v, table=cache.table, kv=ints([64]), w=w, to=out.table, budget=32, recent=0, ko=out.k,
            vo=out.v, wo=None):
        with pytest.raises(exc):
            P.paged_evict(k, v, table, kv, w, to, budget, recent, k_out=ko, v_out=vo, weights_out=wo)

    bad(ValueError, k=cache.k.cpu())
    bad(NotImplementedError, k=cache.k.half(), v=cache.v.half())
    bad(ValueError, vo=None)
    bad(ValueError, budget=0)
    bad(ValueError, recent=33)
    bad(ValueError, recent=-1)
    bad(ValueError, budget=out.table.shape[1] * 16 + 1)
    bad(ValueError, w=w[..., :32])
    bad(ValueError, w=w.double())
    bad(ValueError, kv=ints([64], torch.int64))
    bad(ValueError, to=out.table.long())
    bad(ValueError, ko=out.k.float(), vo=out.v.float())
    bad(ValueError, ko=out.k[:, :1], vo=out.v[:, :1])
    bad(ValueError, vo=out.k)
    bad(ValueError, ko=cache.v, vo=cache.k)
    bad(ValueError, to=cache.table, ko=None, vo=None)
    bad(ValueError, wo=torch.zeros((1, 2, 31), device=DEV))
    bad(ValueError, wo=w[..., 8:])
    c12 = Cache([64], 2, 12, 16)
    bad(NotImplementedError, k=c12.k, v=c12.v, ko=c12.k, vo=c12.v)
    torch.cuda.synchronize()


@pytest.mark.parametrize("Hq,Hkv,d,page", [(8, 2, 128, 16), (4, 4, 64, 32)])
def test_a_prompt_steps_an_eviction_and_more_steps(Hq, Hkv, d, page):
    """The operators as a layer runs them: prompts enter the cache and are attended to with their keys' weights, tokens
    follow, the cache is cut, and tokens follow again.  Each stage is checked against float64 of the state before it."""
    lens, budget, room = [150, 61], 48, 16
    g = gen(7)
    cache = Cache([n + room for n in lens], Hkv, d, page, seed=3)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    ang = torch.arange(512, dtype=torch.float64, device=DEV)[:, None] * inv
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(BF16) for _ in range(2))
    w = torch.full((2, Hkv, cache.table.shape[1] * page), float("nan"), device=DEV)

    def step(cache, w, nq, have, seen):
        """``nq`` new tokens of each sequence behind ``have`` cached ones, ``seen`` tokens into the text."""
        n = sum(nq)
        rows = randn(g, n, (Hq + 2 * Hkv) * d)
        q, k, v = (t.unflatten(1, (-1, d)) for t in rows.split([Hq * d, Hkv * d, Hkv * d], 1))
        pos = torch.cat([torch.arange(s, s + x, device=DEV) for s, x in zip(seen, nq)])
        at = [torch.arange(h, h + x, device=DEV) for h, x in zip(have, nq)]
        slots = torch.cat([cache.table[b].long()[a // page] * page + a % page for b, a in enumerate(at)])
        qr = P.qk_norm_rope_append(q, k, v, cos, sin, pos, cache.k, cache.v, slots, qw, kw)
        qe, ke = P.qk_norm_rope(q, k, cos, sin, pos, qw, kw)
        assert torch.equal(qr, qe)
        assert torch.equal(cache.k[slots // page, :, slots % page], ke)
        assert torch.equal(cache.v[slots // page, :, slots % page], v)
        now = [h + x for h, x in zip(have, nq)]
        before = w.clone()
        o, m, l = P.paged_attention(qr, cache.k, cache.v, cache.table, ints(now), starts_of(nq), d ** -0.5, weights=w,
                                    weights_out=w, return_ml=True)
        check_attention(cache, qr, nq, now, o, scale=d ** -0.5, m=m, l=l, weights=w, before=before)
        return now, [s + x for s, x in zip(seen, nq)]

    have, seen = step(cache, w, lens, [0, 0], [0, 0])
    for _ in range(3):
        have, seen = step(cache, w, [1, 1], have, seen)
    small = Cache([budget + room] * 2, Hkv, d, page, seed=9)
    small.k.fill_(float("nan"))
    small.v.fill_(float("nan"))
    w2 = torch.full((2, Hkv, small.table.shape[1] * page), float("nan"), device=DEV)
    cache.lens = have
    kept, new, _ = P.paged_evict(cache.k, cache.v, cache.table, ints(have), w, small.table, budget, 8, k_out=small.k,
                                 v_out=small.v, weights_out=w2)
    _check(cache, w, budget, 8, kept, new, w2, small)
    have = new.tolist()
    for nq in ([1, 1], [5, 2], [1, 1]):
        have, seen = step(small, w2, nq, have, seen)
