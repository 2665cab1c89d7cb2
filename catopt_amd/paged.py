"""Operators of a key/value cache kept in pages, for serving.

The cache of one layer is two tensors of pages ``k_pages`` and ``v_pages``,
each ``(n_pages, Hkv, page_size, d)`` with a contiguous last axis (other
strides as they are, for attention and eviction multiples of 16 bytes: pass a
``(n_pages, page_size, Hkv, d)`` storage transposed).  Key
``j`` of sequence ``b`` lies in slot ``j % page_size`` of page
``block_table[b, j // page_size]``; one table serves every layer.  Lengths,
tables, positions and slots are device tensors that no call reads back, so a
step recorded into a hipGraph replays with new ones.

A layer's step over new tokens:

* :func:`qk_norm_rope_append` norms and rotates their queries and keys and
  writes keys and values into the cache (:func:`qk_norm_rope` returns them
  instead);
* :func:`paged_attention` attends from each sequence's new tokens to its
  cached keys, a prompt, a chunk of one or a single token alike, and can add
  up every key's attention weight;
* :func:`paged_evict` moves each head's most attended and most recent keys
  into a smaller cache.

As in :mod:`catopt_amd.kernels`, operands are device tensors checked on the
host before any launch, outputs and workspace come from torch's caching
allocator, and work is enqueued on torch's current stream of the operands'
device.  What only the device knows (a length past the table, a page index
outside the pages) never leads out of bounds: lengths are cut to the table's
reach, keys of an invalid page count as masked, and a write to one is dropped.

What the host knows chooses the kernels: tokens, sequences and the table's width.
So a call is fastest with tables about as wide as its longest sequence and
without idle sequences beside a long chunk.
"""

from __future__ import annotations

import functools
import struct

import torch

from . import _lib as L
from .kernels import _DT, _need_device, _stream_of

__all__ = ["qk_norm_rope", "qk_norm_rope_append", "paged_attention", "paged_evict", "PAGED_ATTENTION_MAX_HEAD_DIM",
           "QK_NORM_ROPE_MAX_HEAD_DIM"]

PAGED_ATTENTION_MAX_HEAD_DIM = 128
QK_NORM_ROPE_MAX_HEAD_DIM = 256

# host arrays of strides, as the C entries take them
_S12, _S14, _S16 = (struct.Struct(f"{n}q").pack for n in (12, 14, 16))


_get_device = torch.Tensor.get_device


def _device(ts: tuple) -> int:
    """The device index that all operands share; raises as ``kernels`` does where they do not."""
    try:
        devs = {*map(_get_device, ts)}
        if len(devs) == 1:
            dev = devs.pop()
            if dev >= 0:
                return dev
    except TypeError:  # not a tensor
        pass
    return _need_device(*ts)


def _launch(dev: int, fn, *args) -> int:
    """``fn(*args, stream)`` with the operands' device as the current one."""
    if torch._C._cuda_getDevice() == dev:
        return fn(*args, _stream_of(dev))
    with torch.cuda.device(dev):
        return fn(*args, _stream_of(dev))


def _heads(name: str, t: torch.Tensor, step: int) -> tuple[torch.Tensor, torch.Size, tuple, int]:
    """``(N, H, d)`` with a contiguous last axis, rows readable in 16-byte pieces (``step`` elements) where a copy makes
    them so; its shape, strides and address."""
    s, at = t.stride(), t.data_ptr()
    if len(s) != 3:
        raise ValueError(f"{name} is (tokens, heads, head dim), got {tuple(t.shape)}")
    if s[2] != 1 or s[0] % step or s[1] % step or at % 16:
        t = t.contiguous()
        s, at = t.stride(), t.data_ptr()
    return t, t.shape, s, at


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, what: str = "") -> tuple[torch.Size, tuple, tuple]:
    """The shape and strides of a cache's two page tensors, which are used in place: nothing is copied to fit."""
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"the {what}pages are two tensors (n_pages, heads, page size, head dim) of one type, got "
                         f"{tuple(shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"the {what}pages need a contiguous head dim, got strides {ks} and {vs}")
    return shape, ks, vs


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, n: int) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != (n,):
        raise ValueError(f"{name} is an {dtype} vector of {n}, got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _table(name: str, t: torch.Tensor, B: int) -> tuple[torch.Tensor, int, int]:
    """An int32 table of B rows, its entries a row and the rows' distance."""
    shape, s = t.shape, t.stride()
    if t.dtype is not torch.int32 or len(shape) != 2 or shape[0] != B:
        raise ValueError(f"{name} is an int32 ({B}, pages of a sequence) tensor, got {t.dtype} {tuple(shape)}")
    if s[1] != 1 and shape[1] > 1:
        t = t.contiguous()
        s = t.stride()
    return t, shape[1], s[0]


def _check(fn: str, status: int) -> None:
    """A refusal of the library's own checks (what overlaps what) as the argument error that it is."""
    if status == L.E_INVAL:
        raise ValueError(f"{fn}: an output overlaps another operand or itself, or rows are not 16-byte aligned")
    if status == L.E_UNSUPPORTED:
        raise NotImplementedError(f"{fn}: the call is beyond what one launch takes")
    L.check(fn, status)


def _norm_rope(q, k, v, cos, sin, positions, q_weight, k_weight, eps, interleaved, k_pages, v_pages, slots):
    ts = (q, k, cos, sin, positions) if slots is None else (q, k, cos, sin, positions, v, k_pages, v_pages, slots)
    if q_weight is not None:
        ts += (q_weight,)
    if k_weight is not None:
        ts += (k_weight,)
    dev = _device(ts)
    dtype = q.dtype
    dt = _DT.get(dtype)
    if dt is None:
        raise NotImplementedError(f"qk_norm_rope runs on fp32 and bf16 operands, got {dtype}")
    step = 8 if dt == L.BF16 else 4
    q, qshape, (q0, q1, _), q_at = _heads("q", q, step)
    k, kshape, (k0, k1, _), k_at = _heads("k", k, step)
    N, Hq, d = qshape
    kn, Hkv, kd = kshape
    if k.dtype is not dtype or kn != N or kd != d:
        raise ValueError(f"q and k share tokens, head dim and type: {tuple(qshape)} {dtype}, {tuple(kshape)} {k.dtype}")
    if not 1 <= d <= QK_NORM_ROPE_MAX_HEAD_DIM:
        raise NotImplementedError(f"qk_norm_rope takes head dims up to {QK_NORM_ROPE_MAX_HEAD_DIM}, got {d}")
    table, cs = cos.shape, cos.stride()
    if len(table) != 2 or sin.shape != table or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError("cos and sin are fp32 tables (positions, rotated dims / 2) of one shape")
    n_pos, half = table
    rot, ld = 2 * half, cs[0]
    if rot > d:
        raise ValueError(f"the tables rotate {rot} dims of a head of {d}")
    if rot and (cs[1] != 1 or ld < half or sin.stride() != cs):
        cos, sin, ld = cos.contiguous(), sin.contiguous(), half
    qw = kw = None
    if q_weight is not None:
        q_weight = _norm_weight(q_weight, dtype, d)
        qw = q_weight.data_ptr()
    if k_weight is not None:
        k_weight = _norm_weight(k_weight, dtype, d)
        kw = k_weight.data_ptr()
    positions = _vector("positions", positions, torch.int64, N)
    q_out = q.new_empty(qshape)
    if slots is None:
        k_out = q.new_empty(kshape)
        v_at = slots_at = v_out = None
        k_to, n_pages, page = k_out.data_ptr(), 0, 0
        strides = _S12(q0, q1, k0, k1, 0, 0, 0, 0, 0, 0, 0, 0)
    else:
        v, vshape, (v0, v1, _), v_at = _heads("v", v, step)
        if vshape != kshape or v.dtype is not dtype:
            raise ValueError(f"v has k's shape and type: {tuple(vshape)} {v.dtype}, {tuple(kshape)} {dtype}")
        (n_pages, ph, page, pd), (ko0, ko1, ko2, _), (vo0, vo1, vo2, _) = _pages(k_pages, v_pages)
        if ph != Hkv or pd != d or k_pages.dtype is not dtype:
            raise ValueError(f"the pages hold {ph} heads of {pd} {k_pages.dtype}, k has {Hkv} of {d} {dtype}")
        slots = _vector("slots", slots, torch.int64, N)
        k_out, slots_at, k_to, v_out = None, slots.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
        strides = _S12(q0, q1, k0, k1, v0, v1, ko0, ko1, ko2, vo0, vo1, vo2)
    st = _launch(dev, L.load().catopt_hip_qk_norm_rope, dt, N, Hq, Hkv, d, rot, 1 if interleaved else 0, q_at, k_at,
                 v_at, qw, kw, eps, cos.data_ptr(), sin.data_ptr(), n_pos, ld, positions.data_ptr(), q_out.data_ptr(),
                 k_to, v_out, strides, slots_at, n_pages, page)
    if st:
        _check("qk_norm_rope", st)
    return q_out, k_out


def _norm_weight(w: torch.Tensor, dtype: torch.dtype, d: int) -> torch.Tensor:
    if w.dtype is not dtype or w.numel() != d:
        raise ValueError(f"a norm weight holds one value of q's type for each head dim, got {tuple(w.shape)} {w.dtype}")
    return w.contiguous()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6, *,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The RMS norm of every head of ``q (N, Hq, d)`` and ``k (N, Hkv, d)``
    and their position rotation, in one pass (fp32 or bf16; computed in fp32,
    rounded once).

    ``x * rsqrt(mean(x²) + eps) * weight`` over the head dim (a weight of
    ``None``: no norm), then each pair ``(a, b)`` of the first ``rot`` dims
    becomes ``(a c - b s, b c + a s)``: pairs ``(i, i + rot/2)``, or ``(2i,
    2i+1)`` when ``interleaved``, with ``c, s`` of row ``positions[n]`` of the
    fp32 tables ``cos, sin (positions, rot/2)``.  ``q`` and ``k`` may be views
    of one projection's rows.  ``positions`` is int64; one outside the tables
    gives NaN in the rotated dims.  Returns new ``(q, k)``."""
    return _norm_rope(q, k, None, cos, sin, positions, q_weight, k_weight, eps, interleaved, None, None, None)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                        positions: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        *, interleaved: bool = False) -> torch.Tensor:
    """:func:`qk_norm_rope` whose keys go into the cache, with ``v (N, Hkv,
    d)`` as it is: token ``n`` to slot ``slots[n] % page_size`` of page
    ``slots[n] // page_size`` of ``k_pages`` and ``v_pages``.  ``slots`` is
    int64 and names no slot twice; a token whose slot lies outside the pages
    (-1 for padding) is not written.  Returns the new ``q``."""
    if slots is None or k_pages is None or v_pages is None or v is None:
        raise TypeError("qk_norm_rope_append needs v, k_pages, v_pages and slots")
    return _norm_rope(q, k, v, cos, sin, positions, q_weight, k_weight, eps, interleaved, k_pages, v_pages, slots)[0]


@functools.lru_cache(maxsize=4096)
def _attn_workspace(B: int, N: int, Hq: int, Hkv: int, d: int, n_table: int, page: int, weights: int) -> int:
    n = L.load().catopt_hip_paged_attn_workspace_bytes(B, N, Hq, Hkv, d, n_table, page, weights)
    if n < 0:
        raise NotImplementedError("paged attention: the call is beyond what one launch takes")
    return n


def _weight_rows(name: str, w: torch.Tensor, B: int, H: int, width: int) -> tuple[int, int]:
    shape, s = w.shape, w.stride()
    if w.dtype is not torch.float32 or len(shape) != 3 or shape[0] != B or shape[1] != H or shape[2] < width:
        raise ValueError(f"{name} is an fp32 ({B}, {H}, at least {width}) tensor, got {w.dtype} {tuple(shape)}")
    if s[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name} needs a contiguous last axis, got strides {s}")
    return s[0], s[1]


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, q_starts: torch.Tensor, scale: float, *, causal: bool = True,
                    weights: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
                    return_ml: bool = False, empty_rows: str = "nan", out: torch.Tensor | None = None):
    """Attention of each sequence's new tokens over its cached keys (bf16).

    ``q (N, Hq, d)`` holds the tokens of all sequences, sequence ``b``'s in
    rows ``q_starts[b]`` to ``q_starts[b + 1]`` (int32, ``B + 1`` ascending
    values); ``kv_lens (B,)`` int32 counts its cached keys, the new tokens'
    own the last of them (write them first, :func:`qk_norm_rope_append`); more
    than the table reaches are cut to its reach.
    ``block_table (B, n)`` is int32.  With ``causal`` token ``i`` of ``n``
    sees keys ``j <= kv_len - n + i``, else every key.  Query head ``h`` reads
    key head ``h // (Hq // Hkv)``.  ``d`` is a multiple of 8 up to 128, the
    page size a multiple of 8.

    Returns ``o (N, Hq, d)``, written to ``out`` when given (memory of its
    own: not between the operands' first and last rows); rows behind the
    last sequence are neither read nor written.  ``return_ml`` adds the fp32
    ``(m, l)`` om carriers of the sequences' rows, ``(N, Hq)``, so that a part
    of the keys kept elsewhere can be combined: ``(m, l, o.float() * l[...,
    None])`` is what :func:`catopt_amd.kernels.om_compose` takes.  A row that
    sees no key is NaN (``empty_rows="nan"``) or 0 (``"zero"``), as in
    :func:`catopt_amd.kernels.attention`; its carrier is ``(-inf, 0)``, that of
    a row with a NaN score NaN.  Scores, statistics and sums are fp32; the
    softmax terms are rounded to bf16 for the product with the values, and the
    result once more.

    ``weights_out (B, Hkv, L)`` fp32, ``L`` at least the table's reach,
    receives the sum over the new tokens and the key head's query heads of
    each key's softmax weight, on top of ``weights`` (the sums so far; none:
    zeros), which is not read for the new tokens' own keys.  Entries from
    ``kv_lens[b]`` on are left as they were.  ``weights_out`` may be
    ``weights``.  With few new tokens the products are kept in between, 4 bytes
    for each token, query head and key of the table's reach, up to 1 GiB."""
    if empty_rows not in ("nan", "zero"):
        raise ValueError(f"empty_rows is 'nan' or 'zero', got {empty_rows!r}")
    ts = (q, k_pages, v_pages, block_table, kv_lens, q_starts)
    if out is not None:
        ts += (out,)
    if weights_out is not None:
        ts += (weights_out,) if weights is None else (weights_out, weights)
    elif weights is not None:
        raise ValueError("weights need a weights_out to go to")
    dev = _device(ts)
    if q.dtype is not torch.bfloat16 or k_pages.dtype is not torch.bfloat16:
        raise NotImplementedError(f"paged attention runs on bf16 operands, got {q.dtype} and {k_pages.dtype} pages")
    q, qshape, (q0, q1, _), q_at = _heads("q", q, 8)
    if q_at % 16:
        q = q.clone()
        q_at = q.data_ptr()
    N, Hq, d = qshape
    (n_pages, Hkv, page, pd), (k0, k1, k2, _), (v0, v1, v2, _) = _pages(k_pages, v_pages)
    if pd != d or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"q has {Hq} heads of {d}, the pages {Hkv} heads of {pd}: the head dims agree and the query "
                         "heads are a multiple of the key heads")
    if d % 8 or not 8 <= d <= PAGED_ATTENTION_MAX_HEAD_DIM:
        raise NotImplementedError(f"paged attention takes head dims that are multiples of 8 up to "
                                  f"{PAGED_ATTENTION_MAX_HEAD_DIM}, got {d}")
    if page < 1 or page % 8:
        raise NotImplementedError(f"paged attention takes page sizes that are multiples of 8, got {page}")
    scale = float(scale)
    if not 0 < scale < 1e38:
        raise ValueError(f"the scale is a positive number below 1e38, got {scale}")
    B = q_starts.numel() - 1
    kv_lens = _vector("kv_lens", kv_lens, torch.int32, B)
    q_starts = _vector("q_starts", q_starts, torch.int32, B + 1)
    table, n_table, table_ld = _table("block_table", block_table, B)
    if out is None:
        out = q.new_empty(qshape)
    elif out.shape != qshape or out.dtype is not torch.bfloat16:
        raise ValueError(f"out has q's shape and type, got {tuple(out.shape)} {out.dtype}")
    o0, o1, o2 = out.stride()
    if o2 != 1:
        raise ValueError(f"out needs a contiguous head dim, got strides {out.stride()}")
    wi0 = wi1 = wo0 = wo1 = 0
    wi = wo = m = l = mp = lp = ws_at = None
    if weights_out is not None:
        wo0, wo1 = _weight_rows("weights_out", weights_out, B, Hkv, n_table * page)
        wo = weights_out.data_ptr()
        if weights is not None:
            wi0, wi1 = _weight_rows("weights", weights, B, Hkv, n_table * page)
            wi = weights.data_ptr()
    if return_ml:
        m, l = q.new_empty((N, Hq), dtype=torch.float32), q.new_empty((N, Hq), dtype=torch.float32)
        mp, lp = m.data_ptr(), l.data_ptr()
    if B and (N or wo is not None):
        wsb = _attn_workspace(B, N, Hq, Hkv, d, n_table, page, wo is not None)
        if wsb:
            ws = q.new_empty(wsb // 2)
            ws_at = ws.data_ptr()
        st = _launch(dev, L.load().catopt_hip_paged_attn_fwd, L.BF16, B, N, Hq, Hkv, d, q_at, k_pages.data_ptr(),
                     v_pages.data_ptr(), n_pages, page, table.data_ptr(), table_ld, n_table, kv_lens.data_ptr(),
                     q_starts.data_ptr(), scale, 1 if causal else 0, 2 if empty_rows == "zero" else 1, out.data_ptr(),
                     mp, lp, wi, wo, _S14(q0, q1, k0, k1, k2, v0, v1, v2, o0, o1, wi0, wi1, wo0, wo1), ws_at, wsb)
        if st:
            _check("paged_attention", st)
    return (out, m, l) if return_ml else out


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                weights: torch.Tensor, out_table: torch.Tensor, budget: int, recent: int = 0, *,
                k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None,
                weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut each sequence's cache to ``budget`` keys a head, by accumulated
    attention weight (fp32 or bf16 pages).

    Of the ``n = kv_lens[b]`` keys of head ``h``, ``min(n, budget)`` stay: the
    last ``recent`` ones and, of the others, those of the largest ``weights[b,
    h, :]`` (:func:`paged_attention`'s sums; the lowest index first among
    equals, a NaN above every number).  Each head keeps its own, in their
    order: they move to slots 0, 1, … of the pages ``out_table (B, n')`` names
    in ``k_out, v_out (n_out_pages, Hkv, out_page_size, d)``, a cache of its
    own (say of a fixed size for generation) or, by default, ``k_pages,
    v_pages``.  In that case the pages of ``out_table`` are free ones: none
    may be in ``block_table``, whose pages can be given back afterwards.  No
    page is in ``out_table`` twice.
    Rows behind the last kept key are left as they were.

    Returns ``kept (B, Hkv, budget)`` int32 (the keys' indices, -1 behind the
    last), ``new_lens (B,)`` int32 and their weights, in ``weights_out (B,
    Hkv, at least budget)`` when given (it may be ``weights``), else in a new
    tensor whose entries behind the last kept key are 0."""
    if (k_out is None) != (v_out is None):
        raise ValueError("give both k_out and v_out, or neither")
    ts = (k_pages, v_pages, block_table, kv_lens, weights, out_table)
    if k_out is not None:
        ts += (k_out, v_out)
    if weights_out is not None:
        ts += (weights_out,)
    dev = _device(ts)
    dtype = k_pages.dtype
    dt = _DT.get(dtype)
    if dt is None:
        raise NotImplementedError(f"eviction runs on fp32 and bf16 pages, got {dtype}")
    (n_pages, Hkv, page, d), (k0, k1, k2, _), (v0, v1, v2, _) = _pages(k_pages, v_pages)
    if k_out is None:
        k_out, v_out = k_pages, v_pages
    (n_out, ho, page_out, do), (ko0, ko1, ko2, _), (vo0, vo1, vo2, _) = _pages(k_out, v_out, "output ")
    if ho != Hkv or do != d or k_out.dtype is not dtype:
        raise ValueError(f"the output pages hold {ho} heads of {do} {k_out.dtype}, the cache {Hkv} of {d} {dtype}")
    if d < 1 or Hkv < 1 or page < 1 or page_out < 1 or d % (8 if dt == L.BF16 else 4):
        raise NotImplementedError(f"eviction takes rows of a multiple of 16 bytes, got {d} of {dtype}")
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"a budget of at least 1 with 0 <= recent <= budget, got {budget} and {recent}")
    B = kv_lens.numel()
    kv_lens = _vector("kv_lens", kv_lens, torch.int32, B)
    table, n_table, table_ld = _table("block_table", block_table, B)
    to, n_to, to_ld = _table("out_table", out_table, B)
    if n_to * page_out < budget:
        raise ValueError(f"out_table reaches {n_to * page_out} keys, the budget is {budget}")
    wi0, wi1 = _weight_rows("weights", weights, B, Hkv, n_table * page)
    fresh = weights_out is None
    if fresh:
        weights_out = weights.new_empty((B, Hkv, budget))
    wo0, wo1 = _weight_rows("weights_out", weights_out, B, Hkv, budget)
    kept = kv_lens.new_empty((B, Hkv, budget))
    new_lens = kv_lens.new_empty((B,))
    if B:
        st = _launch(dev, L.load().catopt_hip_paged_evict, dt, B, Hkv, d, k_pages.data_ptr(), v_pages.data_ptr(), n_pages,
                     page, table.data_ptr(), table_ld, n_table, kv_lens.data_ptr(), weights.data_ptr(), budget, recent,
                     k_out.data_ptr(), v_out.data_ptr(), n_out, page_out, to.data_ptr(), to_ld, n_to, kept.data_ptr(),
                     new_lens.data_ptr(), weights_out.data_ptr(), 1 if fresh else 0,
                     _S16(k0, k1, k2, v0, v1, v2, ko0, ko1, ko2, vo0, vo1, vo2, wi0, wi1, wo0, wo1))
        if st:
            _check("paged_evict", st)
    return kept, new_lens, weights_out
