"""Head norm and rotation in one pass, with and without the write into the cache, against float64."""

from __future__ import annotations

import math

import pytest
import torch

from catopt_amd import paged as P
from paged_ref import BF16, DEV, gen, ints, randn, rope

pytestmark = pytest.mark.gpu
F32 = torch.float32


def _tables(rot, n=997):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / max(rot, 1))
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cos(a).float(), torch.sin(a).float()


def _case(N, Hq, Hkv, d, rot, dtype, norm, seed=0, packed=True):
    g = gen(seed)
    if packed:
        rows = randn(g, N, (Hq + 2 * Hkv) * d, dtype=dtype)
        q, k, v = (t.unflatten(1, (-1, d)) for t in rows.split([Hq * d, Hkv * d, Hkv * d], 1))
    else:
        q, k, v = (randn(g, h, N, d, dtype=dtype).transpose(0, 1) for h in (Hq, Hkv, Hkv))
    w = [1 + 0.2 * torch.randn(d, generator=g, device=DEV) for _ in range(2)] if norm else [None, None]
    w = [None if x is None else x.to(dtype) for x in w]
    cos, sin = _tables(rot)
    pos = torch.randint(0, cos.shape[0], (N,), generator=g, device=DEV)
    return q, k, v, w, cos, sin, pos


def _near(got, x, w, cos, sin, pos, pairs, eps=1e-6):
    want, tol = rope(x, w, cos, sin, pos, pairs, eps)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    err = (got.double() - want).abs()
    assert (err <= tol)[~nan].all(), float((err / tol)[~nan].max())


# tokens, query and key heads, head dim, rotated dims
SHAPES = [(1, 1, 1, 2, 2), (1, 4, 1, 128, 128), (3, 32, 8, 128, 128), (130, 12, 4, 64, 32), (17, 3, 3, 96, 96),
          (9, 5, 1, 80, 20), (33, 2, 1, 256, 64), (5, 7, 7, 112, 112), (4, 2, 2, 63, 62), (7, 1, 1, 72, 0),
          (600, 8, 2, 128, 64), (2, 64, 8, 192, 64), (1, 0, 3, 64, 64), (5, 3, 0, 64, 64), (11, 4, 2, 8, 8)]


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,Hq,Hkv,d,rot", SHAPES)
def test_norm_and_rotation(N, Hq, Hkv, d, rot, dtype, pairs):
    for norm in (True, False):
        q, k, _, w, cos, sin, pos = _case(N, Hq, Hkv, d, rot, dtype, norm, seed=N + d)
        qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, w[0], w[1], 1e-5, interleaved=pairs)
        assert qo.dtype == dtype and qo.is_contiguous() and ko.is_contiguous()
        _near(qo, q, w[0], cos, sin, pos, pairs, 1e-5)
        _near(ko, k, w[1], cos, sin, pos, pairs, 1e-5)


@pytest.mark.parametrize("which", [0, 1])
def test_one_weight_alone(which):
    q, k, _, w, cos, sin, pos = _case(20, 4, 2, 128, 128, BF16, True)
    w[which] = None
    qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, *w)
    _near(qo, q, w[0], cos, sin, pos, False)
    _near(ko, k, w[1], cos, sin, pos, False)


@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("dtype,page", [(BF16, 16), (F32, 16), (BF16, 5)])
@pytest.mark.parametrize("N,Hq,Hkv,d,rot", [(1, 4, 1, 128, 128), (40, 8, 2, 64, 64), (300, 6, 6, 96, 32), (8, 32, 8, 128, 128)])
def test_append(N, Hq, Hkv, d, rot, dtype, page, slot_major):
    q, k, v, w, cos, sin, pos = _case(N, Hq, Hkv, d, rot, dtype, True, seed=N)
    n_pages = -(-N // page) + 4
    shape = (n_pages, page, Hkv, d) if slot_major else (n_pages, Hkv, page, d)
    kp, vp = (torch.full(shape, 9.0, dtype=dtype, device=DEV) for _ in range(2))
    if slot_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    slots = torch.randperm(n_pages * page, generator=gen(N), device=DEV)[:N]
    written = torch.ones(N, dtype=torch.bool, device=DEV)
    if N > 5:  # padded tokens, and slots that no page has
        for i, s in ((1, -1), (3, n_pages * page), (4, 2 ** 62), (5, -2 ** 62)):
            slots[i], written[i] = s, False
    qo = P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)
    _near(qo, q, w[0], cos, sin, pos, False)
    at = slots[written]
    _near(kp[at // page, :, at % page], k[written], w[1], cos, sin, pos[written], False)
    assert torch.equal(vp[at // page, :, at % page], v[written])
    rest = torch.ones(n_pages * page, dtype=torch.bool, device=DEV)
    rest[at] = False
    for t in (kp, vp):
        assert (t.transpose(1, 2).reshape(n_pages * page, -1)[rest] == 9).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_head_major_operands_and_far_rows(dtype):
    q, k, _, w, cos, sin, pos = _case(70, 4, 2, 128, 128, dtype, True, packed=False)
    qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, *w)
    _near(qo, q, w[0], cos, sin, pos, False)
    _near(ko, k, w[1], cos, sin, pos, False)


def test_positions_outside_the_tables():
    q, k, v, w, cos, sin, pos = _case(8, 4, 2, 64, 32, BF16, True)
    pos[2], pos[5], pos[7] = -1, cos.shape[0], 2 ** 62
    qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, *w)
    _near(qo, q, w[0], cos, sin, pos, False)
    _near(ko, k, w[1], cos, sin, pos, False)
    assert torch.isnan(qo[2, :, :32]).all() and not torch.isnan(qo[2, :, 32:]).any() and not torch.isnan(qo[3]).any()


def test_values_that_are_not_finite_stay_in_their_rows():
    q, k, v, w, cos, sin, pos = _case(6, 2, 2, 128, 128, BF16, True)
    q[2, 1, 5], k[3, 0, 7] = float("nan"), float("inf")
    qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, *w)
    assert torch.isnan(qo[2, 1]).all() and torch.isnan(ko[3, 0, 7])
    bad = torch.zeros((6, 2), dtype=torch.bool, device=DEV)
    bad[2, 1] = True
    assert not torch.isnan(qo[~bad]).any()
    z = torch.zeros((3, 2, 128), dtype=BF16, device=DEV)
    zo, _ = P.qk_norm_rope(z, z, cos, sin, pos[:3], *w)
    assert (zo == 0).all()


def test_pages_past_32_bit_offsets():
    page, Hkv, d = 64, 8, 128
    n_pages = (1 << 31) // (page * Hkv * d) + 9
    kp, vp = (torch.empty((n_pages, Hkv, page, d), dtype=BF16, device=DEV) for _ in range(2))
    kp[-1], vp[-1] = 0, 0
    q, k, v, w, cos, sin, pos = _case(5, 16, Hkv, d, d, BF16, True)
    slots = n_pages * page - 1 - 7 * torch.arange(5, device=DEV)
    P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)
    at = slots % page
    _near(kp[-1][:, at].transpose(0, 1), k, w[1], cos, sin, pos, False)
    assert torch.equal(vp[-1][:, at].transpose(0, 1), v)


def test_captured_and_on_a_side_stream():
    q, k, v, w, cos, sin, pos = _case(9, 8, 2, 128, 128, BF16, True)
    kp, vp = (torch.zeros((4, 2, 16, 128), dtype=BF16, device=DEV) for _ in range(2))
    slots = torch.arange(9, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)
    for step in range(4):
        pos.copy_(torch.randint(0, cos.shape[0], (9,), generator=gen(step), device=DEV))
        slots.copy_(torch.randperm(64, generator=gen(step), device=DEV)[:9])
        kp.zero_()
        g.replay()
        torch.cuda.synchronize()
        k2, v2 = torch.zeros_like(kp), vp.clone()
        want = P.qk_norm_rope_append(q, k, v, cos, sin, pos, k2, v2, slots, *w)
        assert torch.equal(out, want) and torch.equal(kp, k2) and torch.equal(vp, v2)


@pytest.mark.parametrize("dtype,N", [(BF16, 7000), (F32, 3500)])
def test_rows_past_the_caches(dtype, N):
    """More than 256 MB of rows: the same bits as in parts."""
    q, k, v, w, cos, sin, pos = _case(N, 64, 8, 128, 128, dtype, True)
    kp, vp = (torch.zeros((N // 16 + 1, 8, 16, 128), dtype=dtype, device=DEV) for _ in range(2))
    slots = torch.randperm(N, generator=gen(1), device=DEV)
    qo = P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)
    for a in range(0, N, 1000):
        r = slice(a, min(a + 1000, N))
        qe, ke = P.qk_norm_rope(q[r], k[r], cos, sin, pos[r], *w)
        assert torch.equal(qo[r], qe) and torch.equal(kp[slots[r] // 16, :, slots[r] % 16], ke)
        assert torch.equal(vp[slots[r] // 16, :, slots[r] % 16], v[r])
    _near(qo[-50:], q[-50:], w[0], cos, sin, pos[-50:], False)


def test_one_row_of_the_tables_for_every_position_and_axes_of_one_entry():
    q, k, v, w, cos, sin, _ = _case(6, 4, 1, 64, 64, BF16, True)
    pos = torch.arange(6, device=DEV)
    c, s = (t[5:6].expand(6, -1) for t in (cos, sin))
    qo, ko = P.qk_norm_rope(q, k, c, s, pos, *w)
    wq, wk = P.qk_norm_rope(q, k, cos, sin, torch.full_like(pos, 5), *w)
    assert torch.equal(qo, wq) and torch.equal(ko, wk)
    one = (t[5:6].as_strided((1, 32), (3, 1)) for t in (cos, sin))
    k1 = k.as_strided(k.shape, (k.stride(0), 19, 1))  # one key head
    qo, ko = P.qk_norm_rope(q, k1, *one, torch.zeros_like(pos), *w)
    assert torch.equal(qo, wq) and torch.equal(ko, wk)


def test_no_pages():
    q, k, v, w, cos, sin, pos = _case(6, 4, 2, 64, 64, BF16, True)
    none = torch.empty((0, 2, 16, 64), dtype=BF16, device=DEV)
    qo = P.qk_norm_rope_append(q, k, v, cos, sin, pos, none, none.clone(), torch.full_like(pos, -1), *w)
    _near(qo, q, w[0], cos, sin, pos, False)


def test_no_tokens():
    q, k, v, w, cos, sin, pos = _case(0, 4, 2, 64, 64, BF16, True)
    qo, ko = P.qk_norm_rope(q, k, cos, sin, pos, *w)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)


def test_refusals():
    q, k, v, w, cos, sin, pos = _case(4, 4, 2, 64, 64, BF16, True)
    kp, vp = (torch.zeros((4, 2, 16, 64), dtype=BF16, device=DEV) for _ in range(2))
    slots = torch.arange(4, device=DEV)

    def bad(exc, q=q, k=k, cos=cos, sin=sin, pos=pos, qw=w[0], kw=w[1]):
        with pytest.raises(exc):
            P.qk_norm_rope(q, k, cos, sin, pos, qw, kw)

    bad(ValueError, q=q.cpu())
    bad(NotImplementedError, q=q.half(), k=k.half(), qw=None, kw=None)
    bad(ValueError, k=k.float())
    bad(ValueError, k=k[:3])
    bad(ValueError, q=q[0])
    bad(ValueError, pos=pos[:3])
    bad(ValueError, pos=pos.int())
    bad(ValueError, cos=cos.double())
    bad(ValueError, sin=sin[:, :4])
    bad(ValueError, qw=w[0][:32])
    bad(ValueError, kw=w[1].float())
    wide = _tables(128)
    bad(ValueError, cos=wide[0], sin=wide[1])
    x = randn(gen(0), 4, 2, 264)
    bad(NotImplementedError, q=x, k=x, qw=None, kw=None)

    def bad_append(exc, v=v, kp=kp, vp=vp, slots=slots):
        with pytest.raises(exc):
            P.qk_norm_rope_append(q, k, v, cos, sin, pos, kp, vp, slots, *w)

    bad_append(TypeError, slots=None)
    bad_append(ValueError, slots=ints([0, 1, 2, 3]))
    bad_append(ValueError, v=v[:, :1])
    bad_append(ValueError, kp=kp.float(), vp=vp.float())
    bad_append(ValueError, kp=kp[:, :1], vp=vp[:, :1])
    bad_append(ValueError, vp=kp)
    bad_append(ValueError, kp=kp[:1].expand(4, -1, -1, -1))
    bad_append(ValueError, kp=kp[..., :32])
    assert math.isfinite(float(kp.float().sum()))
