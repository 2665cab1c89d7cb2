"""float64 references of the paged cache's operators, and caches to run them on."""

from __future__ import annotations

import math

import torch

DEV = "cuda:0"
BF16 = torch.bfloat16
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # of a rounding, relative to the value


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


class Cache:
    """Pages dealt in no order; slots outside the sequences hold NaN, so that a read of one shows."""

    def __init__(self, lens, Hkv, d, page, seed=0, dtype=BF16, slot_major=False, table_extra=1):
        g = gen(seed + 1000)
        need = [-(-n // page) for n in lens]
        self.n_pages, self.page, self.Hkv, self.d, self.lens = sum(need) + 3, page, Hkv, d, list(lens)
        shape = (self.n_pages, page, Hkv, d) if slot_major else (self.n_pages, Hkv, page, d)
        self.k, self.v = (torch.full(shape, float("nan"), device=DEV, dtype=dtype) for _ in range(2))
        if slot_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(self.n_pages, generator=g, device=DEV).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need, default=0), 1) + table_extra), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        for b, n in enumerate(lens):
            for t in (self.k, self.v):
                self.put(t, b, randn(g, Hkv, n, d, dtype=dtype))

    def where(self, b, n):
        j = torch.arange(n, device=DEV)
        return self.table[b].long()[j // self.page], j % self.page

    def put(self, pages, b, rows):
        p, s = self.where(b, rows.shape[1])
        pages[p, :, s] = rows.transpose(0, 1)

    def rows(self, pages, b, n=None):
        """(Hkv, n, d) of a sequence, in float64."""
        p, s = self.where(b, self.lens[b] if n is None else n)
        return pages[p, :, s].transpose(0, 1).double()


def starts_of(nq):
    out = [0]
    for n in nq:
        out.append(out[-1] + n)
    return ints(out)


def attention(q, k, v, scale, causal=True, keep=None):
    """One sequence: q (n, Hq, d), k and v (Hkv, len, d) -> o, m, l, p (Hq, n, len) and the error bounds that the
    operands' magnitudes give.  Sums run over seen keys only, so what lies in the others cannot matter."""
    n, Hq, d = q.shape
    Hkv, length = k.shape[:2]
    g = Hq // Hkv
    qd = q.double().transpose(0, 1)
    seen = torch.ones((n, length), dtype=torch.bool, device=DEV)
    if causal:
        seen = torch.arange(length, device=DEV)[None] <= length - n + torch.arange(n, device=DEV)[:, None]
    if keep is not None:
        seen = seen & keep[None]
    res = {x: [] for x in ("o", "m", "l", "p", "mag", "es")}
    for h in range(Hq):
        kh = torch.where(seen.any(0)[:, None], k[h // g], 0.0)
        s = torch.where(seen, scale * (qd[h] @ kh.T), -math.inf)
        m = s.amax(-1) if length else torch.full((n,), -math.inf, dtype=torch.float64, device=DEV)
        some = torch.isfinite(m)
        e = torch.where(some[:, None], torch.exp(s - torch.where(some, m, 0.0)[:, None]), 0.0)
        l = e.sum(-1)
        # sum over seen keys alone: 0 * NaN of a key that the row does not see never enters
        vh = v[h // g]
        clean = torch.nan_to_num(vh, nan=0.0, posinf=0.0, neginf=0.0)
        a, mag = e @ clean, e @ clean.abs()
        odd = ~torch.isfinite(vh)
        if bool((odd.any(-1)[None] & seen).any()):
            for i in range(n):
                a[i] += torch.where(odd & seen[i][:, None], vh, 0.0).sum(0)
        # a score is a sum of d products in fp32, then scaled and offset in fp32
        es = (d + 8) * 2.0 ** -24 * scale * (qd[h].abs() @ kh.abs().T)
        es = torch.where(seen, es, 0.0).amax(-1) if length else torch.zeros_like(l)
        es = es + 2.0 ** -22 * torch.where(some, m, 0.0).abs()
        res["o"].append(a / l[:, None])
        for name, t in (("m", m), ("l", l), ("p", e / torch.where(some, l, 1.0)[:, None]), ("mag", mag / l[:, None]), ("es", es)):
            res[name].append(t)
    return {x: torch.stack(t) for x, t in res.items()}


def check_attention(cache, q, nq, lens, got, *, scale, causal=True, m=None, l=None, weights=None, before=None, keep=None,
                    empty="nan"):
    """``got`` (and ``m``, ``l``, ``weights``) against float64, each within the bound that its arithmetic gives: the
    score's error es shifts a softmax term by a factor exp(es); the term is rounded to bf16 for the value product and
    the result once more; sums of n terms in fp32 lose at most n steps."""
    at = 0
    for b, (n, length) in enumerate(zip(nq, lens)):
        rows = slice(at, at + n)
        at += n
        if n == 0:
            if weights is not None and length:
                want = before[b, :, :length].double() if before is not None else torch.zeros_like(weights[b, :, :length]).double()
                assert torch.equal(weights[b, :, :length].double(), want), b
            continue
        r = attention(q[rows], cache.rows(cache.k, b, length), cache.rows(cache.v, b, length), scale, causal,
                      None if keep is None else keep[b])
        o = got[rows].double().transpose(0, 1)
        some = torch.isfinite(r["m"])
        es = torch.expm1(2 * r["es"]) + (length + 64) * 2.0 ** -24
        fin = torch.isfinite(r["o"]) & some[..., None]
        tol = (HALF_STEP[BF16] + es)[..., None] * r["mag"] * 1.01 + HALF_STEP[BF16] * r["o"].abs() + 1e-37
        err = (o - r["o"]).abs()
        assert (err <= tol)[fin].all(), (b, float((err / tol)[fin].max()))
        odd = some[..., None] & ~torch.isfinite(r["o"])
        assert torch.equal(torch.nan_to_num(o[odd], 5.0), torch.nan_to_num(r["o"][odd], 5.0)), b
        none = o[~some]
        assert (torch.isnan(none) if empty == "nan" else none == 0).all(), b
        if m is not None:
            gm, gl = m[rows].double().t(), l[rows].double().t()
            assert torch.equal(torch.isneginf(gm), ~some) and (gl[~some] == 0).all()
            assert ((gm - r["m"]).abs() <= r["es"] + 1e-37)[some].all()
            assert ((gl - r["l"]).abs() <= es * r["l"] * 1.01)[some].all()
        if weights is not None:
            g = r["p"].shape[0] // cache.Hkv
            terms = r["p"].unflatten(0, (cache.Hkv, g))
            want = terms.sum((1, 2))
            tol = ((2 * es + (n * g + 64) * 2.0 ** -24).unflatten(0, (cache.Hkv, g))[..., None] * terms).sum((1, 2)) * 1.01
            if before is not None:
                old = before[b, :, :length].double().clone()
                old[:, max(length - n, 0):] = 0
                want = want + old
            tol = tol + HALF_STEP[torch.float32] * want.abs() + 1e-37
            err = (weights[b, :, :length].double() - want).abs()
            assert (err <= tol).all(), (b, float((err / tol).max()))


def rope(x, w, cos, sin, positions, pairs, eps=1e-6):
    """float64 norm and rotation of x (N, H, d), and the bound of the fp32 arithmetic: a sum of d squares, a reciprocal
    root, three products and a sum."""
    d, half = x.shape[-1], cos.shape[1]
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    z, mag = y.clone(), y.abs()
    i = torch.arange(half, device=DEV)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    known = (positions >= 0) & (positions < cos.shape[0])
    p = torch.where(known, positions, 0)
    c, s = (torch.where(known[:, None], t[p].double(), math.nan)[:, None] for t in (cos, sin))
    z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    both = y[..., a].abs() + y[..., b].abs()
    mag[..., a], mag[..., b] = both, both
    return z, (d / 2 + 16) * 2.0 ** -24 * mag + HALF_STEP[x.dtype] * z.abs() * 1.01 + 1e-37


def evict(weights, length, budget, recent):
    """The kept indices of one head, by the definition."""
    m = min(length, budget)
    old = length - min(recent, m)
    w = weights[:old].double().cpu()
    order = sorted(range(old), key=lambda j: (0 if math.isnan(w[j]) else 1, -float(w[j]) if not math.isnan(w[j]) else 0.0, j))
    return sorted(order[:m - (length - old)] + list(range(old, length)))
