"""The paged cache's operators on the host: what the C ABI refuses before any launch (the operand addresses are never
read) and the checks of layouts and overlaps that the Python entry points make."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from catopt_amd import _lib as L
from catopt_amd import paged as P

FAKE = 1 << 12
Q, KP, VP, OUT, WIN, WOUT, KO, VO, QO = (FAKE + (i << 32) for i in range(1, 10))  # far apart, never read


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from catopt_amd import build

        build.build()
    return L.load()


def _attn(lib, dtype=L.BF16, B=1, N=4, Hq=4, Hkv=2, d=64, q=Q, k=KP, v=VP, n_pages=8, page=16, table=FAKE, ld=4,
          n_table=4, lens=FAKE, starts=FAKE, scale=1.0, causal=1, norm=1, o=OUT, w_in=None, w_out=None, strides=None,
          ws=FAKE, wsb=1 << 40):
    st = (C.c_int64 * 14)(*(strides or [256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64, 128, 64, 128, 64]))
    return lib.catopt_hip_paged_attn_fwd(dtype, B, N, Hq, Hkv, d, q, k, v, n_pages, page, table, ld, n_table, lens,
                                         starts, scale, causal, norm, o, None, None, w_in, w_out, st, ws, wsb, None)


def test_attention_refuses(lib):
    # nothing to do is no error, and touches nothing
    assert _attn(lib, B=0) == L.OK and _attn(lib, N=0, q=None, o=None) == L.OK
    for kw in ({"B": -1}, {"N": -1}, {"Hq": 3}, {"Hkv": 0}, {"n_pages": -1}, {"n_table": -1}, {"ld": -1}, {"norm": 0},
               {"norm": 3}, {"q": None}, {"o": None}, {"k": None}, {"v": None}, {"table": None}, {"lens": None},
               {"starts": None}, {"q": Q + 8}, {"o": OUT + 2}, {"k": KP + 4}, {"v": VP + 4}, {"w_in": WIN},
               {"strides": [-256] + [64] * 13}, {"strides": [4] + [64] * 13}, {"strides": [64] * 10 + [-1] * 4}):
        assert _attn(lib, **kw) == L.E_INVAL, kw
    for kw in ({"dtype": L.F32}, {"d": 60}, {"d": 136}, {"d": 0}, {"page": 12}, {"scale": 0.0}, {"scale": float("inf")},
               {"scale": float("nan")}, {"scale": 3e38}, {"N": 1 << 40}, {"B": 1 << 40}, {"n_table": 1 << 30}, {"page": 1 << 40}):
        assert _attn(lib, **kw) == L.E_UNSUPPORTED, kw
    need = lib.catopt_hip_paged_attn_workspace_bytes(1, 4, 4, 2, 64, 4, 16, 1)
    assert need > 0
    assert _attn(lib, w_out=WOUT, ws=None) == L.E_WORKSPACE
    assert _attn(lib, w_out=WOUT, wsb=need - 1) == L.E_WORKSPACE
    assert _attn(lib, w_out=WOUT, ws=FAKE + 8, wsb=need) == L.E_WORKSPACE


def test_attention_refuses_overlaps(lib):
    """Asked with a workspace too small, so that what is not refused as an overlap ends at that check."""
    def ask(**kw):
        return _attn(lib, **{"w_out": WOUT, "wsb": 0, **kw})

    ok = [256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64, 128, 64, 128, 64]

    def strides(at, *v):
        return ok[:at] + list(v) + ok[at + len(v):]

    # q: 4 x 256 elements; pages: 8 x 2048; weights: 1 x 2 x 64 of 4 bytes
    odd = [100, 1] + ok[2:8] + [3, 5, 7, 128, 9, 128]  # axes of one entry may have any stride
    for kw in ({}, {"N": 1, "Hq": 1, "Hkv": 1, "strides": odd}, {"o": Q + 2048},
               {"o": KP + 2 * 8 * 2048}, {"v": KP}, {"w_in": WIN}, {"w_in": WOUT}, {"w_out": Q + 2048}, {"w_in": WOUT + 512}, {"strides": strides(8, 512, 64)},
               {"strides": strides(8, 64, 256)}, {"N": 1, "strides": strides(8, 0, 64)}):
        assert ask(**kw) == L.E_WORKSPACE, kw
    for kw in ({"o": Q}, {"o": Q + 2032}, {"o": Q - 2032}, {"o": KP + 64}, {"o": VP + 2 * 8 * 2048 - 16}, {"w_out": Q + 2044},
               {"w_out": KP}, {"w_out": OUT + 4}, {"w_in": OUT}, {"w_in": WOUT + 4}, {"w_in": WOUT - 256},
               {"w_in": WOUT, "strides": strides(10, 128, 128)}, {"strides": strides(8, 0, 64)},
               {"strides": strides(8, 256, 0)}, {"strides": strides(8, 128, 64)}, {"strides": strides(8, 64, 64)},
               {"strides": strides(12, 128, 32)}):
        assert ask(**kw) == L.E_INVAL, kw


def test_workspace_query(lib):
    f = lib.catopt_hip_paged_attn_workspace_bytes
    ok = [1, 4, 4, 2, 64, 4, 16, 0]
    assert f(*ok) >= 0 and f(*ok[:-1], 1) > 0
    for i, x in ((0, -1), (1, -1), (2, 3), (3, 0), (4, 0), (4, 132), (4, 60), (5, -1), (6, 0), (6, 12), (1, 1 << 31),
                 (2, 1 << 20), (5, 1 << 31), (6, 1 << 31)):
        bad = list(ok)
        bad[i] = x
        assert f(*bad) == -1, bad


def _rope(lib, dtype=L.BF16, N=4, Hq=4, Hkv=2, d=64, rot=64, q=Q, k=WIN, v=WOUT, cos=FAKE, sin=FAKE, n_pos=8, ld=32,
          pos=FAKE, qo=QO, ko=KP, vo=VP, strides=None, slots=None, n_pages=4, page=16):
    st = (C.c_int64 * 12)(*(strides or [256, 64, 128, 64, 128, 64, 2048, 1024, 64, 2048, 1024, 64]))
    return lib.catopt_hip_qk_norm_rope(dtype, N, Hq, Hkv, d, rot, 0, q, k, v, None, None, 1e-6, cos, sin, n_pos, ld, pos,
                                       qo, ko, vo, st, slots, n_pages, page, None)


def test_norm_rope_refuses(lib):
    assert _rope(lib, N=0) == L.OK and _rope(lib, Hq=0, Hkv=0) == L.OK
    for kw in ({"N": -1}, {"Hq": -1}, {"d": 0}, {"rot": 66}, {"rot": 3}, {"rot": -2}, {"n_pos": -1}, {"pos": None},
               {"q": None}, {"qo": None}, {"k": None}, {"ko": None}, {"cos": None}, {"sin": None}, {"ld": 31},
               {"strides": [-1] * 12}, {"slots": FAKE, "v": None}, {"slots": FAKE, "vo": None},
               {"slots": FAKE, "page": 0}, {"slots": FAKE, "n_pages": -1}, {"slots": FAKE, "vo": KP},
               {"slots": FAKE, "k": KP}, {"slots": FAKE, "v": VP + 4096}, {"slots": FAKE, "q": VP},
               {"slots": FAKE, "strides": [256, 64, 128, 64, 128, 64, 0, 1024, 64, 2048, 1024, 64]}):
        assert _rope(lib, **kw) == L.E_INVAL, kw
    for kw in ({"dtype": 2}, {"d": 257}, {"N": 1 << 41}, {"N": 1 << 36}, {"Hq": 1 << 21},
               {"slots": FAKE, "n_pages": 1 << 27}, {"slots": FAKE, "n_pages": 1 << 40, "page": 1 << 40}):
        assert _rope(lib, **kw) == L.E_UNSUPPORTED, kw


def _evict(lib, dtype=L.BF16, B=1, H=2, d=64, k=KP, v=VP, n_pages=8, page=16, table=FAKE, ld=4, n_table=4, lens=FAKE,
           w=WIN, budget=8, recent=2, ko=KO, vo=VO, n_out=8, page_out=16, to=OUT, to_ld=4, n_to=4, kept=FAKE,
           new=FAKE, wo=None, strides=None):
    st = (C.c_int64 * 16)(*(strides or [2048, 1024, 64] * 4 + [128, 64] * 2))
    return lib.catopt_hip_paged_evict(dtype, B, H, d, k, v, n_pages, page, table, ld, n_table, lens, w, budget, recent,
                                      ko, vo, n_out, page_out, to, to_ld, n_to, kept, new, wo, 0, st, None)


def test_evict_refuses(lib):
    assert _evict(lib, B=0) == L.OK
    for kw in ({"B": -1}, {"H": 0}, {"d": 0}, {"n_pages": -1}, {"page": 0}, {"n_table": -1}, {"ld": -1}, {"n_out": -1},
               {"page_out": 0}, {"n_to": -1}, {"to_ld": -1}, {"budget": 0}, {"recent": -1}, {"recent": 9},
               {"budget": 65}, {"lens": None}, {"kept": None}, {"new": None}, {"to": None}, {"table": None}, {"w": None},
               {"k": None}, {"v": None}, {"ko": None}, {"vo": None}, {"k": KP + 8}, {"vo": VO + 8},
               {"strides": [4] * 16}, {"strides": [64] * 12 + [-1] * 4}, {"ko": VP, "vo": KP}, {"vo": KO}, {"ko": KP + 2048},
               {"vo": VP + 4096}, {"ko": KP, "vo": VP, "to": FAKE}, {"ko": KP, "vo": VP, "n_out": 9}, {"ko": KP}, {"vo": VP},
               {"w": KO}, {"w": VO}, {"wo": KO}, {"wo": KP}, {"wo": WIN + 4},
               {"strides": [2048, 1024, 64] * 2 + [0, 1024, 64] * 2 + [128, 64] * 2},
               {"strides": [2048, 1024, 64] * 4 + [128, 64, 0, 64], "wo": WOUT, "B": 2}):
        assert _evict(lib, **kw) == L.E_INVAL, kw
    for kw in ({"dtype": 2}, {"d": 4}, {"d": 1 << 14}, {"B": 1 << 21}, {"H": 1 << 21}, {"B": 1 << 11, "H": 1 << 11},
               {"n_table": 1 << 27}, {"budget": 1 << 31, "n_to": 1 << 28},
               {"d": 1 << 12, "page": 1 << 20, "n_table": 4, "budget": 1 << 22, "n_to": 1 << 18}):
        assert _evict(lib, **kw) == L.E_UNSUPPORTED, kw


def test_host_tensors_are_refused():
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    p = torch.zeros((2, 4, 16, 64), dtype=torch.bfloat16)
    i = torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        P.paged_attention(q, p, p.clone(), i[None], i, torch.zeros((2,), dtype=torch.int32), 1.0)
    with pytest.raises(ValueError, match="ROCm device"):
        P.qk_norm_rope(q, q, torch.ones((4, 32)), torch.ones((4, 32)), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="ROCm device"):
        P.paged_evict(p, p.clone(), i[None], i, torch.zeros((1, 4, 16)), i[None], 1)
    with pytest.raises(TypeError):
        P.qk_norm_rope_append(q, q, q, None, None, None, p, p, None)


def test_layout_checks():
    u = torch.zeros((3, 4, 12))
    assert P._heads("t", u[..., :7], 4)[3] == u.data_ptr()  # rows of 48 bytes: read in place
    t, shape, strides, at = P._heads("t", u[..., 1:8], 4)
    assert t.is_contiguous() and shape == (3, 4, 7) and strides == (28, 7, 1) and at == t.data_ptr()  # misaligned: copied
    with pytest.raises(ValueError):
        P._heads("t", u[0], 4)
    with pytest.raises(ValueError):
        P._pages(u, u)
