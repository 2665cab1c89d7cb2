"""Tables, slots and positions of a step from its requests' lengths, and pages given back, against plain Python."""

from __future__ import annotations

import random

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import DEV, ints

pytestmark = pytest.mark.gpu


def _ceil(a, b):
    return -(-a // b)


def extend_ref(table, lens, new, pool, count, n_tokens, page, offsets=None):
    table, reach = [list(r) for r in table], len(table[0]) * page if table else 0
    count = min(max(count, 0), len(pool))
    starts, positions, slots, lens_out, at = [0], [0] * n_tokens, [-1] * n_tokens, [], 0
    for b, (have, fresh) in enumerate(zip(lens, new)):
        have, fresh = min(max(have, 0), reach), min(max(fresh, 0), n_tokens - at)
        after = min(have + fresh, reach)
        for i in range(_ceil(have, page), _ceil(after, page)):
            count -= 1
            table[b][i] = pool[count] if count >= 0 else -1
        for i in range(fresh):
            key = have + i
            positions[at] = key + (offsets[b] if offsets else 0)
            if key < reach and table[b][key // page] >= 0:
                slots[at] = table[b][key // page] * page + key % page
            at += 1
        starts.append(at)
        lens_out.append(after)
    return table, starts, positions, slots, lens_out, max(count, 0)


def release_ref(table, lens, released, pool, count, page):
    pool, count, out = list(pool), min(max(count, 0), len(pool)), []
    for row, n, gone in zip(table, lens, released):
        if gone:
            for x in row[:min(_ceil(max(n, 0), page), len(row))]:
                if x >= 0:
                    if count < len(pool):
                        pool[count] = x
                    count += 1
        out.append(0 if gone else n)
    return pool, out, min(count, len(pool))


def _state(rng, B, ctx, width, page, free):
    lens = [rng.randint(0, ctx) for _ in range(B)]
    ids = list(range(sum(_ceil(n, page) for n in lens) + free))
    rng.shuffle(ids)
    table, at = [], 0
    for n in lens:
        k = _ceil(n, page)
        table.append(ids[at:at + k] + [-7] * (width - k))
        at += k
    return table, lens, ids[at:]


def _check_extend(table, lens, new, pool, count, n_tokens, page, offsets=None):
    t, p = ints(table).reshape(len(lens), -1), ints(pool)
    r = P.paged_extend(t, ints(lens), ints(new), p, ints([count]), n_tokens, page,
                       offsets=None if offsets is None else ints(offsets))
    want = extend_ref(table, lens, new, pool, count, n_tokens, page, offsets)
    assert r.q_starts.tolist() == want[1]
    assert r.positions.tolist() == want[2]
    assert r.slots.tolist() == want[3]
    assert r.kv_lens.tolist() == want[4] and r.free_count.tolist() == [want[5]]
    assert t.tolist() == want[0] and p.tolist() == pool
    assert r.q_starts.dtype == r.kv_lens.dtype == r.free_count.dtype == torch.int32
    assert r.positions.dtype == r.slots.dtype == torch.int64


@pytest.mark.parametrize("B,ctx,q,page,pad", [
    (1, 0, 1, 16, 0), (1, 0, 5000, 16, 0), (1, 77, 1, 1, 3), (3, 5, 0, 8, 0), (3, 5, 0, 8, 5), (8, 3000, 1, 16, 0),
    (64, 200, 70, 16, 9), (65, 100, 3, 24, 0), (511, 90, 2, 16, 0), (512, 90, 2, 16, 1), (513, 90, 4, 7, 0),
    (1300, 40, 3, 16, 2000), (5, 1000, 900, 128, 0)])
def test_extend(B, ctx, q, page, pad):
    rng = random.Random(B * 1000 + page)
    table, lens, pool = _state(rng, B, ctx, _ceil(ctx + q, page) + 1, page, B * (_ceil(q, page) + 1))
    new = [rng.randint(0, q) for _ in range(B)]
    offsets = [rng.randint(-50, 1 << 20) for _ in range(B)] if B % 2 else None
    _check_extend(table, lens, new, pool, len(pool), sum(new) + pad, page, offsets)


@pytest.mark.parametrize("free,count", [(3, 3), (0, 0), (9, -5), (6, 100), (40, 2)])
def test_a_pool_that_runs_out(free, count):
    rng = random.Random(free)
    table, lens, pool = _state(rng, 6, 40, 12, 8, free)
    _check_extend(table, lens, [9, 0, 17, 8, 1, 20], pool, count, 60, 8)


def test_more_tokens_than_rows():
    rng = random.Random(1)
    table, lens, pool = _state(rng, 5, 30, 16, 8, 60)
    for n in (0, 1, 20, 34, 35, 36):
        _check_extend(table, lens, [10, 0, 15, 10, 2 ** 31 - 1], pool, len(pool), n, 8)


def test_lengths_out_of_range():
    rng = random.Random(2)
    table, lens, pool = _state(rng, 5, 20, 4, 8, 20)
    lens[1], lens[3] = -9, 2 ** 31 - 1
    _check_extend(table, lens, [5, 12, -3, 6, 50], pool, len(pool), 80, 8)
    _check_extend([[], []], [0, 4], [3, 2], pool, len(pool), 6, 8)  # a table of no pages


def test_invalid_pages_give_no_slot():
    _check_extend([[-1, 5, 0], [3, -2, 0]], [16, 9], [3, 3], [-1, 4], 2, 6, 8)


def test_nothing_to_do():
    r = P.paged_extend(ints([]).reshape(0, 3), ints([]), ints([]), ints([4, 5]), ints([2]), 4, 16)
    assert r.q_starts.tolist() == [0] and r.slots.tolist() == [-1] * 4 and r.free_count.tolist() == [2]
    r = P.paged_extend(ints([[1]]), ints([3]), ints([0]), ints([]), ints([0]), 0, 16)
    assert r.q_starts.tolist() == [0, 0] and r.kv_lens.tolist() == [3] and r.slots.shape == (0,)


def test_extend_views_and_streams():
    rng = random.Random(3)
    table, lens, pool = _state(rng, 7, 50, 9, 8, 40)
    wide = torch.full((7, 20), 55, dtype=torch.int32, device=DEV)
    wide[:, 4:13] = ints(table)
    both = torch.stack([ints(lens), ints([3] * 7)], 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = P.paged_extend(wide[:, 4:13], both[:, 0], both[:, 1], ints(pool), ints([len(pool)]), 21, 8)
    side.synchronize()
    want = extend_ref(table, lens, [3] * 7, pool, len(pool), 21, 8)
    assert wide[:, 4:13].tolist() == want[0] and (wide[:, :4] == 55).all() and (wide[:, 13:] == 55).all()
    assert r.slots.tolist() == want[3] and r.kv_lens.tolist() == want[4]


@pytest.mark.parametrize("B,ctx,page", [(1, 100, 16), (1, 0, 8), (16, 300, 16), (17, 300, 16), (300, 2000, 16), (3, 9000, 1)])
@pytest.mark.parametrize("share", [0.0, 0.4, 1.0])
def test_release(B, ctx, page, share):
    rng = random.Random(B)
    table, lens, pool = _state(rng, B, ctx, _ceil(ctx, page) + 1, page, 20)
    gone = [rng.random() < share for _ in range(B)]
    for row in table[::3]:
        for i in range(0, len(row), 5):
            row[i] = -1  # a page that the pool did not have
    count = len(pool)
    pool = pool + [-3] * (sum(len(r) for r in table))
    t, p = ints(table).reshape(B, -1), ints(pool)
    new, c = P.paged_release(t, ints(lens), torch.tensor(gone, device=DEV), p, ints([count]), page)
    want = release_ref(table, lens, gone, pool, count, page)
    assert p.tolist() == want[0] and new.tolist() == want[1] and c.tolist() == [want[2]]
    assert t.tolist() == table


@pytest.mark.parametrize("B", [3, 40])
def test_release_out_of_range(B):
    table = [[10 * b + i for i in range(4)] for b in range(B)]
    for lens, count in (([2 ** 31 - 1] * B, 0), ([-5] * B, 1), ([20] * B, 99), ([20] * B, -4), ([32] * B, 3)):
        pool = [-1] * 7  # fewer places than pages
        t, p = ints(table), ints(pool)
        new, c = P.paged_release(t, ints(lens), torch.ones((B,), dtype=torch.bool, device=DEV), p, ints([count]), 8)
        want = release_ref(table, lens, [True] * B, pool, count, 8)
        assert p.tolist() == want[0] and new.tolist() == want[1] and c.tolist() == [want[2]]
    new, c = P.paged_release(ints([]).reshape(0, 2), ints([]), torch.zeros((0,), dtype=torch.bool, device=DEV), ints([1]), ints([1]), 8)
    assert new.shape == (0,) and c.tolist() == [1]


@pytest.mark.parametrize("B,q", [(3, 1), (30, 40), (600, 3)])
def test_a_captured_step_goes_on_in_place(B, q):
    """Lengths, pool and table as the state of a server: extended and released by the replays of two graphs."""
    rng = random.Random(B)
    page, width = 8, 60
    table, lens, pool = _state(rng, B, 30, width, page, B * 4)
    n = B * q
    t, kv, p, c = ints(table), ints(lens), ints(pool + [-1] * B * width), ints([len(pool)])
    new, gone = ints([0] * B), torch.zeros((B,), dtype=torch.bool, device=DEV)
    pool = pool + [-1] * B * width

    def extend():
        return P.paged_extend(t, kv, new, p, c, n, page, kv_lens_out=kv, free_count_out=c)

    def release():
        P.paged_release(t, kv, gone, p, c, page, kv_lens_out=kv, free_count_out=c)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        extend(), release()  # nothing new, nothing released
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (extend, release):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = f()
        graphs.append(g)
        if f is extend:
            out = r
    count = c.item()
    for step in range(6):
        fresh = [rng.randint(0, q) for _ in range(B)]
        ended = [rng.random() < 0.3 for _ in range(B)]
        new.copy_(ints(fresh))
        gone.copy_(torch.tensor(ended))
        graphs[0].replay()
        table, starts, positions, slots, lens, count = extend_ref(table, lens, fresh, pool, count, n, page)
        assert t.tolist() == table and kv.tolist() == lens and c.tolist() == [count]
        assert out.q_starts.tolist() == starts and out.slots.tolist() == slots and out.positions.tolist() == positions
        graphs[1].replay()
        pool, lens, count = release_ref(table, lens, ended, pool, count, page)
        assert p.tolist() == pool and kv.tolist() == lens and c.tolist() == [count]


def test_table_past_32_bit_offsets():
    """Rows of a table that lie more than 2^31 entries apart."""
    ld = (1 << 30) + 24
    wide = torch.empty((2 * ld + 16,), dtype=torch.int32, device=DEV)
    t = wide.as_strided((3, 16), (ld, 1))
    rng = random.Random(1)
    table, lens, pool = _state(rng, 3, 100, 16, 16, 40)
    t.copy_(ints(table))
    new = [20, 1, 37]
    r = P.paged_extend(t, ints(lens), ints(new), ints(pool), ints([len(pool)]), 60, 16)
    want = extend_ref(table, lens, new, pool, len(pool), 60, 16)
    assert t.tolist() == want[0] and r.slots.tolist() == want[3] and r.kv_lens.tolist() == want[4]
    back, p = r.kv_lens.tolist(), ints(pool)
    kv, c = P.paged_release(t, r.kv_lens, torch.tensor([True, False, True], device=DEV), p, r.free_count, 16)
    after = release_ref(want[0], back, [True, False, True], pool, r.free_count.item(), 16)
    assert p.tolist() == after[0] and kv.tolist() == after[1] and c.tolist() == [after[2]]
