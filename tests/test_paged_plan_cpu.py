"""What the entries for a step's tables and slots refuse on the host, before any launch (the addresses are never read)."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import _lib as L
from catopt_amd import paged as P

A = [1 << 20 | i << 32 for i in range(16)]  # far apart


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from catopt_amd import build

        build.build()
    return L.load()


def _extend(lib, B=4, N=32, page=16, table=A[0], ld=8, n_table=8, lens=A[1], new=A[2], pool=A[3], n_free=20, count=A[4],
            offsets=A[5], starts=A[6], positions=A[7], slots=A[8], lens_out=A[9], count_out=A[10]):
    return lib.catopt_hip_paged_extend(B, N, page, table, ld, n_table, lens, new, pool, n_free, count, offsets, starts,
                                       positions, slots, lens_out, count_out, None)


def test_extend_refuses(lib):
    for kw in ({"B": -1}, {"N": -1}, {"page": 0}, {"n_table": -1}, {"ld": -1}, {"n_free": -1}, {"lens": None}, {"new": None},
               {"pool": None}, {"count": None}, {"starts": None}, {"positions": None}, {"slots": None}, {"lens_out": None},
               {"count_out": None}, {"table": None}, {"ld": 7}, {"ld": 0}, {"lens_out": A[1] + 4}, {"count_out": A[1]},
               {"lens_out": A[4]}, {"starts": A[1]}, {"starts": A[0] + 4 * 31}, {"slots": A[7] + 8 * 31}, {"slots": A[3]},
               {"positions": A[2]}, {"table": A[3] - 4}, {"table": A[1]}, {"lens_out": A[2]}, {"lens_out": A[5] + 12},
               {"count_out": A[3] + 76}, {"starts": A[4]}):
        assert _extend(lib, **kw) == L.E_INVAL, kw
    for kw in ({"B": 1 << 21}, {"N": 1 << 30}, {"n_free": 1 << 30}, {"page": 1 << 30}, {"page": 1 << 20, "n_table": 1 << 10},
               {"n_table": 1 << 40}):
        assert _extend(lib, **kw) == L.E_UNSUPPORTED, kw


def _release(lib, B=20, page=16, table=A[0], ld=8, n_table=8, lens=A[1], out=A[2], pool=A[3], n_free=20, count=A[4],
             lens_out=A[5], count_out=A[6], ws=A[7], wsb=1 << 20):
    return lib.catopt_hip_paged_release(B, page, table, ld, n_table, lens, out, pool, n_free, count, lens_out, count_out, ws,
                                        wsb, None)


def test_release_refuses(lib):
    for kw in ({"B": -1}, {"page": 0}, {"n_table": -1}, {"ld": -1}, {"n_free": -1}, {"lens": None}, {"out": None}, {"pool": None},
               {"count": None}, {"lens_out": None}, {"count_out": None}, {"table": None}, {"lens_out": A[1] + 4},
               {"count_out": A[1]}, {"lens_out": A[4] - 8}, {"pool": A[1]}, {"pool": A[4] - 40}, {"lens_out": A[2]},
               {"pool": A[0] + 4}, {"count_out": A[3]}, {"lens_out": A[3]}, {"count_out": A[5] + 8}):
        assert _release(lib, **kw) == L.E_INVAL, kw
    for kw in ({"B": 1 << 21}, {"n_free": 1 << 30}, {"page": 1 << 30}, {"page": 1 << 20, "n_table": 1 << 10}):
        assert _release(lib, **kw) == L.E_UNSUPPORTED, kw
    f = lib.catopt_hip_paged_release_workspace_bytes
    assert f(-1) == -1 and f(1 << 21) == -1 and f(4) == 0 and f(20) == 84
    for kw in ({"ws": None}, {"wsb": 83}, {"ws": A[7] + 2}):
        assert _release(lib, **kw) == L.E_WORKSPACE, kw


def test_python_checks(monkeypatch):
    i = torch.zeros((4,), dtype=torch.int32)
    table, one = torch.zeros((4, 8), dtype=torch.int32), torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        P.paged_extend(table, i, i.clone(), i.clone(), one, 4, 16)
    with pytest.raises(ValueError, match="ROCm device"):
        P.paged_release(table, i, i.bool(), i.clone(), one, 16)
    monkeypatch.setattr(P, "_device", lambda ts: 0)  # the checks behind it, which end before the launch
    bad = [
        dict(n_tokens=-1), dict(page_size=0), dict(kv_lens=i.long()), dict(new_lens=i[:3]), dict(free_pages=i[::2]),
        dict(free_pages=table), dict(free_pages=i.long()), dict(free_count=i), dict(block_table=table[:3]),
        dict(block_table=torch.zeros((8, 4), dtype=torch.int32).t()), dict(offsets=i.long()), dict(kv_lens_out=i.long()),
        dict(kv_lens_out=torch.zeros((8,), dtype=torch.int32)[::2]), dict(free_count_out=i),
    ]
    for kw in bad:
        args = dict(block_table=table, kv_lens=i, new_lens=i, free_pages=i, free_count=one, n_tokens=4, page_size=16) | kw
        with pytest.raises(ValueError):
            P.paged_extend(**args)
    for kw in (dict(page_size=0), dict(released=i), dict(released=i[:3].bool()), dict(free_pages=i[::2]), dict(free_count=i),
               dict(kv_lens_out=i.long()), dict(free_count_out=i), dict(block_table=table[:3])):
        args = dict(block_table=table, kv_lens=i, released=i.bool(), free_pages=i, free_count=one, page_size=16) | kw
        with pytest.raises(ValueError):
            P.paged_release(**args)
