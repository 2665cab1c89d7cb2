"""Attention of new tokens over a paged cache, and the keys' attention weights, against float64."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import BF16, DEV, Cache, check_attention, gen, ints, randn, starts_of

pytestmark = pytest.mark.gpu


def _run(nq, lens, Hq, Hkv, d, page, seed=0, q_scale=1.0, causal=True, slot_major=False, empty="nan", weights=True,
         ml=True):
    cache = Cache(lens, Hkv, d, page, seed, slot_major=slot_major)
    g = gen(seed)
    q = randn(g, sum(nq), Hq, d, scale=q_scale)
    scale = d ** -0.5
    before = torch.rand((len(lens), Hkv, cache.table.shape[1] * page + 5), generator=g, device=DEV)
    w = torch.full_like(before, 77.0)
    kw = {"weights": before, "weights_out": w} if weights else {}
    r = P.paged_attention(q, cache.k, cache.v, cache.table, ints(lens), starts_of(nq), scale, causal=causal,
                          return_ml=ml, empty_rows=empty, **kw)
    o, m, l = r if ml else (r, None, None)
    check_attention(cache, q, nq, lens, o, scale=scale, causal=causal, m=m, l=l, weights=w if weights else None,
                    before=before, empty=empty)
    if weights:
        for b, n in enumerate(lens):
            assert (w[b, :, n:] == 77).all(), b
    return o


# sequences' new tokens, their keys, query and key heads, head dim, page
CASES = [
    ([1], [1], 1, 1, 8, 8),
    ([1], [33], 2, 1, 128, 16),
    ([2], [64], 4, 4, 64, 16),
    ([1, 1, 1], [1, 700, 129], 8, 2, 128, 16),
    ([1] * 9, [5, 64, 65, 2000, 31, 32, 1, 511, 1025], 12, 4, 64, 32),
    ([7, 0, 40], [40, 50, 41], 6, 2, 96, 24),
    ([33, 64, 5], [33, 64, 300], 8, 8, 128, 64),
    ([130], [130], 5, 1, 128, 16),
    ([200, 77], [513, 1000], 14, 2, 64, 8),
    ([300], [1300], 4, 2, 80, 128),
    ([257, 1, 129], [900, 1500, 129], 8, 1, 128, 16),
    ([1], [5000], 32, 1, 128, 48),
    ([31], [3000], 1, 1, 40, 16),
]


@pytest.mark.parametrize("nq,lens,Hq,Hkv,d,page", CASES)
def test_causal(nq, lens, Hq, Hkv, d, page):
    _run(nq, lens, Hq, Hkv, d, page, seed=sum(lens) + d)


@pytest.mark.parametrize("nq,lens,Hq,Hkv,d,page", CASES[1::3])
def test_all_keys_seen(nq, lens, Hq, Hkv, d, page):
    _run(nq, lens, Hq, Hkv, d, page, seed=d, causal=False, slot_major=True)


@pytest.mark.parametrize("weights,ml", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("nq,lens", [([1, 1], [900, 40]), ([150], [700])])
def test_without_the_optional_outputs(nq, lens, weights, ml):
    _run(nq, lens, 8, 2, 128, 16, weights=weights, ml=ml)


@pytest.mark.parametrize("empty", ["nan", "zero"])
@pytest.mark.parametrize("nq,lens", [([3, 5], [0, 2]), ([1, 1, 2], [0, 9, 1]), ([140, 200], [3, 0]), ([0, 4], [0, 4])])
def test_rows_that_see_no_key(nq, lens, empty):
    # more new tokens than keys: the first of them see none
    _run(nq, lens, 4, 2, 64, 16, empty=empty)
    _run(nq, lens, 4, 4, 128, 16, empty=empty)


@pytest.mark.parametrize("nq,lens", [([1, 3], [900, 64]), ([160], [500])])
def test_large_scores(nq, lens):
    _run(nq, lens, 8, 2, 128, 16, q_scale=30.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,length", [(5, 70), (5, 700), (150, 400), (64, 64)])
def test_what_lies_in_keys_not_seen_does_not_matter(nq, length, d):
    """Infinities and NaN in the values and keys of later tokens reach only the rows that see them."""
    cache = Cache([length], 2, d, 16, seed=nq)
    off = length - nq
    for j, x in ((off + nq - 1, float("nan")), (off + nq // 2, float("inf")), (off + nq // 2 + 1, float("-inf"))):
        p, s = (t[j] for t in cache.where(0, length))
        cache.v[p, 0, s, 3], cache.v[p, 1, s, d - 1] = x, x
    q = randn(gen(3), nq, 4, d)
    o, m, l = P.paged_attention(q, cache.k, cache.v, cache.table, ints([length]), starts_of([nq]), 0.1, return_ml=True)
    check_attention(cache, q, [nq], [length], o, scale=0.1, m=m, l=l)
    # a key of NaN: rows before it are as without it
    p, s = (t[length - 1] for t in cache.where(0, length))
    cache.k[p, :, s] = float("nan")
    o2 = P.paged_attention(q, cache.k, cache.v, cache.table, ints([length]), starts_of([nq]), 0.1)
    assert torch.equal(torch.nan_to_num(o2[:nq - 1]), torch.nan_to_num(o[:nq - 1]))
    assert torch.isnan(o2[nq - 1]).all()


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "n_pages"])
@pytest.mark.parametrize("nq", [1, 90])
def test_keys_of_an_invalid_page_count_as_masked(nq, bad):
    length, page = 200, 16
    cache = Cache([length, 40], 2, 128, page, seed=4)
    good = cache.table.clone()
    keep = torch.ones(length, dtype=torch.bool, device=DEV)
    for i in (0, 5, 6):
        cache.table[0, i] = cache.n_pages if bad == "n_pages" else bad
        keep[16 * i:16 * i + 16] = False
    q = randn(gen(1), nq + 1, 4, 128)
    w = torch.zeros((2, 2, cache.table.shape[1] * page), device=DEV)
    o, m, l = P.paged_attention(q, cache.k, cache.v, cache.table, ints([length, 40]), starts_of([nq, 1]), 0.1,
                                return_ml=True, weights_out=w)
    cache.table = good
    check_attention(cache, q, [nq, 1], [length, 40], o, scale=0.1, m=m, l=l, weights=w,
                    keep=[keep, torch.ones(40, dtype=torch.bool, device=DEV)])


@pytest.mark.parametrize("nq", [1, 70])
def test_lengths_are_cut_to_the_table(nq):
    cache = Cache([320], 2, 64, 16, seed=8, table_extra=0)
    q = randn(gen(1), nq, 2, 64)
    args = (q, cache.k, cache.v, cache.table)
    want = P.paged_attention(*args, ints([320]), starts_of([nq]), 0.1)
    assert torch.equal(P.paged_attention(*args, ints([2 ** 31 - 1]), starts_of([nq]), 0.1), want)
    assert torch.isnan(P.paged_attention(*args, ints([-5]), starts_of([nq]), 0.1)).all()
    assert torch.isnan(P.paged_attention(q, cache.k, cache.v, cache.table[:, :0], ints([9]), starts_of([nq]), 0.1)).all()


@pytest.mark.parametrize("nq,lens", [([1, 1], [300, 70]), ([100, 37], [300, 70])])
def test_padded_rows_and_strided_operands(nq, lens):
    """Queries out of a packed projection, pages by slot, an output inside a wider one; idle sequences and their rows."""
    cache = Cache(lens + [0, 0], 2, 128, 16, seed=6, slot_major=True)
    n = sum(nq)
    packed = randn(gen(2), n + 3, 8 * 128)
    q = packed[:, 128:5 * 128].unflatten(1, (4, 128))
    wide = torch.full((n + 3, 6, 128), 5.0, dtype=BF16, device=DEV)
    out = wide[:, 1:5]
    r = P.paged_attention(q, cache.k, cache.v, cache.table, ints(lens + [0, 0]), starts_of(nq + [0, 0]), 0.1, out=out)
    assert r is out
    check_attention(cache, q, nq, lens, out, scale=0.1)
    assert (wide[n:] == 5).all() and (wide[:, 0] == 5).all() and (wide[:, 5] == 5).all()


def test_rows_before_the_first_sequence_and_bad_starts():
    cache = Cache([100, 50], 2, 64, 16, seed=6)
    q = randn(gen(2), 20, 4, 64)
    out = torch.full_like(q, 5.0)
    P.paged_attention(q, cache.k, cache.v, cache.table, ints([100, 50]), ints([4, 10, 15]), 0.1, out=out)
    check_attention(cache, q[4:15], [6, 5], [100, 50], out[4:15], scale=0.1)
    assert (out[:4] == 5).all() and (out[15:] == 5).all()
    # starts that leave the rows stay inside them
    for bad in ([0, 10, 2 ** 31 - 1], [-7, 10, 20], [15, 10, 3], [2 ** 31 - 1] * 3, [-2 ** 31] * 3):
        P.paged_attention(q, cache.k, cache.v, cache.table, ints([100, 50]), ints(bad), 0.1, out=out,
                          weights_out=torch.zeros((2, 2, 160), device=DEV))
    torch.cuda.synchronize()


@pytest.mark.parametrize("nq", [1, 120])
def test_weights_in_place_and_from_nothing(nq):
    cache = Cache([400], 2, 128, 16, seed=3)
    q = randn(gen(2), nq, 8, 128)
    args = (q, cache.k, cache.v, cache.table, ints([400]), starts_of([nq]), 0.1)
    before = torch.rand((1, 2, 416), generator=gen(5), device=DEV)
    fresh, apart, same = torch.zeros_like(before), torch.zeros_like(before), before.clone()
    o = P.paged_attention(*args, weights_out=fresh)
    check_attention(cache, q, [nq], [400], o, scale=0.1, weights=fresh)
    P.paged_attention(*args, weights=before, weights_out=apart)
    check_attention(cache, q, [nq], [400], o, scale=0.1, weights=apart, before=before)
    P.paged_attention(*args, weights=same, weights_out=same)
    assert torch.equal(same[..., :400], apart[..., :400]) and torch.equal(same[..., 400:], before[..., 400:])
    # sums behind the seen keys are not read: the new tokens' own may hold anything
    before[..., 400 - nq:] = float("nan")
    again = torch.zeros_like(before)
    P.paged_attention(*args, weights=before, weights_out=again)
    assert torch.equal(again, apart)


@pytest.mark.parametrize("nq,lens", [([1, 1, 1], [3000, 90, 800]), ([200, 3, 40], [900, 90, 800])])
def test_the_same_call_gives_the_same_bits(nq, lens):
    cache = Cache(lens, 2, 128, 16, seed=3)
    q = randn(gen(2), sum(nq), 8, 128)
    res = []
    for _ in range(3):
        w = torch.zeros((3, 2, cache.table.shape[1] * 16), device=DEV)
        res.append((*P.paged_attention(q, cache.k, cache.v, cache.table, ints(lens), starts_of(nq), 0.1, return_ml=True,
                                       weights_out=w), w))
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


@pytest.mark.parametrize("nq", [1, 80])
def test_captured_steps_replay_on_new_lengths(nq):
    """Two graphs of the same call share no workspace; lengths, tables and queries change between the replays."""
    lens = [700, 333]
    caches = [Cache(lens, 2, 128, 16, seed=s) for s in (1, 2)]
    q = [randn(gen(s), 2 * nq, 8, 128) for s in (1, 2)]
    kv = [ints(lens) for _ in range(2)]
    st = starts_of([nq, nq])
    out = [torch.zeros_like(x) for x in q]
    w = [torch.zeros((2, 2, c.table.shape[1] * 16), device=DEV) for c in caches]

    def call(i, o, ws):
        P.paged_attention(q[i], caches[i].k, caches[i].v, caches[i].table, kv[i], st, 0.1, out=o, weights_out=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            call(i, out[i], w[i])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, out[i], w[i])
        graphs.append(g)
    for step in range(4):
        for i in range(2):
            kv[i].copy_(ints([700 - 90 * step, nq + 17 * step]))
            q[i].copy_(randn(gen(10 * step + i), 2 * nq, 8, 128))
            out[i].zero_()
            w[i].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            o2, w2 = torch.zeros_like(out[i]), torch.zeros_like(w[i])
            call(i, o2, w2)
            assert torch.equal(o2, out[i]) and torch.equal(w2, w[i]), (step, i)
            check_attention(caches[i], q[i], [nq, nq], kv[i].tolist(), out[i], scale=0.1, weights=w[i])


@pytest.mark.parametrize("nq", [1, 80])
def test_on_a_side_stream(nq):
    cache = Cache([600], 2, 128, 16, seed=1)
    q = randn(gen(2), nq, 8, 128)
    args = (q, cache.k, cache.v, cache.table, ints([600]), starts_of([nq]), 0.1)
    want = P.paged_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [P.paged_attention(*args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("nq", [1, 100])
def test_pages_past_32_bit_offsets(nq):
    """The last pages of a cache of more than 2^31 elements (4 GiB of keys)."""
    page, Hkv, d, length = 64, 8, 128, 300
    n_pages = (1 << 31) // (page * Hkv * d) + 9
    k, v = (torch.empty((n_pages, Hkv, page, d), dtype=BF16, device=DEV) for _ in range(2))
    small = Cache([length], Hkv, d, page, seed=2)
    n = -(-length // page)
    table = torch.full((1, n + 1), -1, dtype=torch.int32, device=DEV)
    for i in range(n):
        table[0, i] = n_pages - 1 - i
        k[n_pages - 1 - i], v[n_pages - 1 - i] = small.k[small.table[0, i]], small.v[small.table[0, i]]
    q = randn(gen(2), nq, 16, d)
    kv, st = ints([length]), starts_of([nq])
    got = P.paged_attention(q, k, v, table, kv, st, 0.1)
    assert torch.equal(got, P.paged_attention(q, small.k, small.v, small.table[:, :n + 1].contiguous(), kv, st, 0.1))
    check_attention(small, q, [nq], [length], got, scale=0.1)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("cap,nq,lens,Hq,Hkv", [
    (1024, [1] * 3, [1024, 700, 1], 8, 2),        # the widest table of one range
    (1040, [1] * 3, [1040, 700, 1], 8, 2),        # one page more: ranges
    (512, [1] * 70, [(37 * i) % 500 + 1 for i in range(70)], 8, 4),  # more tiles than CUs
    (1600, [1] * 150, [(97 * i) % 1600 + 1 for i in range(150)], 2, 1),  # sequences past one look of a wave
    (1500, [1, 2, 1, 3] * 17, [(211 * i) % 1400 + 30 for i in range(68)], 32, 8),  # many rows to combine
    (6000, [2], [6000], 64, 2),                   # every range of a tile
])
def test_steps_at_the_borders_of_their_kernels(cap, nq, lens, Hq, Hkv, weights):
    cache = Cache(lens, Hkv, 128, 16, seed=cap)
    table = torch.full((len(lens), cap // 16), -1, dtype=torch.int32, device=DEV)
    table[:, :cache.table.shape[1]] = cache.table[:, :cap // 16]
    q = randn(gen(2), sum(nq), Hq, 128)
    w = torch.zeros((len(lens), Hkv, cap), device=DEV) if weights else None
    o, m, l = P.paged_attention(q, cache.k, cache.v, table, ints(lens), starts_of(nq), 0.1, return_ml=True, weights_out=w)
    check_attention(cache, q, nq, lens, o, scale=0.1, m=m, l=l, weights=w)


def test_weights_of_a_step_whose_products_are_not_stored():
    """Few rows and a table so wide that every product would take more than 1 GiB: they are formed again."""
    B, cap = 64, 1 << 17
    lens = [(131 * i) % 300 + 1 for i in range(B)]
    lens[5] = 9000
    cache = Cache(lens, 8, 64, 16, seed=3)
    table = torch.full((B, cap // 16 + 1), -1, dtype=torch.int32, device=DEV)
    table[:, :cache.table.shape[1]] = cache.table
    q = randn(gen(2), B, 32, 64)
    w = torch.zeros((B, 8, cap + 16), device=DEV)
    o = P.paged_attention(q, cache.k, cache.v, table, ints(lens), starts_of([1] * B), 0.1, weights_out=w)
    check_attention(cache, q, [1] * B, lens, o, scale=0.1, weights=w)


@pytest.mark.parametrize("groups", [1, 3, 5, 7, 8, 32, 33, 40, 130])
def test_query_heads_that_do_not_divide_a_tile(groups):
    _run([40, 3], [90, 300], groups * 2, 2, 64, 16, seed=groups)
    _run([1, 1], [90, 300], groups * 2, 2, 128, 16, seed=groups)


def test_no_new_tokens_keep_the_weights():
    cache = Cache([50, 9], 2, 64, 16)
    e = torch.empty((0, 4, 64), dtype=BF16, device=DEV)
    before = torch.rand((2, 2, 80), generator=gen(1), device=DEV)
    w = torch.full_like(before, 7.0)
    P.paged_attention(e, cache.k, cache.v, cache.table, ints([50, 9]), ints([0, 0, 0]), 0.1, weights=before, weights_out=w)
    for b, n in enumerate((50, 9)):
        assert torch.equal(w[b, :, :n], before[b, :, :n]) and (w[b, :, n:] == 7).all()


@pytest.mark.parametrize("nq", [1, 40])
def test_axes_of_one_entry_and_queries_off_alignment(nq):
    """The stride of an axis of one entry is no stride; queries that start between 16-byte pieces are copied."""
    cache = Cache([100], 1, 64, 128, seed=3)
    table, st = cache.table, ints([0, nq])
    q = randn(gen(2), nq, 4, 64)
    want = P.paged_attention(q, cache.k, cache.v, table, ints([100]), st, 0.1)
    w = torch.zeros((1, 1, table.shape[1] * 128), device=DEV)
    off = torch.empty((nq * 256 + 3,), dtype=BF16, device=DEV)[3:].view(nq, 4, 64)
    off.copy_(q)
    k, v = (t.as_strided(t.shape, (t.stride(0), 77, t.stride(2), 1)) for t in (cache.k, cache.v))  # one key head
    w1 = w.as_strided(w.shape, (5, 3, 1))
    assert torch.equal(P.paged_attention(off, k, v, table, ints([100]), st, 0.1, weights_out=w1), want)
    page = int(table[0, 0])
    k, v = (t[page:page + 1].as_strided((1, 1, 128, 64), (13, 77, 64, 1)) for t in (cache.k, cache.v))  # and one page
    assert torch.equal(P.paged_attention(q, k, v, torch.zeros_like(table), ints([100]), st, 0.1), want)
    if nq == 1:
        q1 = q.as_strided(q.shape, (101, 64, 1))
        out = torch.empty_like(q).as_strided(q.shape, (7, 64, 1))
        assert torch.equal(P.paged_attention(q1, k, v, torch.zeros_like(table), ints([100]), st, 0.1, out=out), want)


def test_nothing_to_do():
    cache = Cache([10], 2, 64, 16)
    e = torch.empty((0, 4, 64), dtype=BF16, device=DEV)
    assert P.paged_attention(e, cache.k, cache.v, cache.table, ints([10]), ints([0, 0]), 0.1).shape == (0, 4, 64)
    out = torch.ones((2, 4, 64), dtype=BF16, device=DEV)
    P.paged_attention(out.clone(), cache.k, cache.v, cache.table[:0], ints([]), ints([0]), 0.1, out=out)
    assert (out == 1).all()


def test_refusals():
    cache = Cache([100], 2, 64, 16)
    q, kv, st = randn(gen(0), 4, 4, 64), ints([100]), ints([0, 4])

    def bad(exc, q=q, k=cache.k, v=cache.v, table=cache.table, kv=kv, st=st, scale=0.1, **kw):
        with pytest.raises(exc):
            P.paged_attention(q, k, v, table, kv, st, scale, **kw)

    w = torch.zeros((1, 2, cache.table.shape[1] * 16), device=DEV)
    bad(ValueError, q=q.cpu())
    bad(TypeError, q=[1])
    bad(NotImplementedError, q=q.float())
    bad(NotImplementedError, k=cache.k.float(), v=cache.v.float())
    bad(ValueError, v=cache.v.float())
    bad(ValueError, q=q[0])
    bad(ValueError, q=randn(gen(0), 4, 3, 64))  # three query heads on two key heads
    bad(ValueError, q=randn(gen(0), 4, 4, 32))
    bad(ValueError, v=cache.v[:-1])
    bad(ValueError, k=cache.k.transpose(2, 3), v=cache.v.transpose(2, 3))
    c9 = Cache([100], 2, 64, 9)
    bad(NotImplementedError, k=c9.k, v=c9.v, table=c9.table)
    c136 = Cache([100], 2, 136, 16)
    bad(NotImplementedError, q=randn(gen(0), 4, 4, 136), k=c136.k, v=c136.v)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        bad(ValueError, scale=s)
    bad(ValueError, kv=kv.long())
    bad(ValueError, kv=kv[None])
    bad(ValueError, st=st.long())
    bad(ValueError, st=ints([0]))
    bad(ValueError, table=cache.table.long())
    bad(ValueError, table=cache.table.expand(2, -1))
    bad(ValueError, empty_rows="none")
    bad(ValueError, out=q)
    bad(ValueError, out=torch.empty_like(q)[:3])
    bad(ValueError, out=torch.empty((1, 4, 64), dtype=BF16, device=DEV).expand(4, 4, 64))
    bad(ValueError, out=cache.k.reshape(-1)[:4 * 256].view(4, 4, 64))
    bad(ValueError, weights=w)
    bad(ValueError, weights_out=w[..., :64])
    bad(ValueError, weights_out=w.double())
    bad(ValueError, weights_out=w.expand(2, 2, -1))
    big = torch.zeros((1, 2, w.shape[2] + 8), device=DEV)
    bad(ValueError, weights=big[..., 8:], weights_out=big[..., :-8])  # overlapping, not the same
    torch.cuda.synchronize()
