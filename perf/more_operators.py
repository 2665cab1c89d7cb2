"""The operators around a paged cache's attention in a serving step, as measurable cases.

A case is a plain dict; ``kind`` names the operator it calls:

* ``extend``  -- block tables, slots and positions of a step's new tokens from the requests' lengths
                 (``paged.paged_extend``);
* ``release`` -- the pages of finished requests back to the free ones (``paged.paged_release``);
* ``prefix``  -- attention of each sequence's new tokens over a prefix that it shares with others and its own keys
                 (``paged.paged_prefix_attention``);
* ``sample``  -- the next tokens from logits by temperature, top-k, top-p and min-p and given random numbers
                 (``sampling.sample``), with ``probs`` also the distribution that is left.

``run`` computes the plain form in elementary torch operations; with ``own`` set it calls the kernels.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16


def listed() -> list[dict]:
    return [
        # one generation step of 8 requests: the smallest call, nothing but latency
        {"name": "extend_step_b8", "kind": "extend", "B": 8, "q_lo": 1, "q_hi": 1, "ctx_lo": 300, "ctx_hi": 3000,
         "page": 16, "pad": 0, "offsets": False, "spare": 64},
        # a mixed step of a busy server: single tokens, chunks and prompts behind shared prefixes, in a padded batch
        {"name": "extend_mixed_b500", "kind": "extend", "B": 500, "q_lo": 1, "q_hi": 900, "ctx_lo": 0, "ctx_hi": 16000,
         "page": 16, "pad": 117, "offsets": True, "spare": 1000},
        # a few of 16 requests have ended
        {"name": "release_b16", "kind": "release", "B": 16, "ctx_lo": 100, "ctx_hi": 2000, "page": 16, "ended": 0.25,
         "spare": 40},
        # half of 512 requests of up to 16000 keys end at once
        {"name": "release_b512", "kind": "release", "B": 512, "ctx_lo": 50, "ctx_hi": 16000, "page": 16, "ended": 0.5,
         "spare": 500},
        # a step of 4 requests with a short instruction before them
        {"name": "prefix_step_b4", "kind": "prefix", "P": 1, "B": 4, "q_lo": 1, "q_hi": 1, "pre_lo": 500, "pre_hi": 500,
         "ctx_lo": 10, "ctx_hi": 200, "hq": 32, "hkv": 8, "d": 128, "page": 16, "ml": False, "pad": 0},
        # a step of 64 requests behind one long instruction
        {"name": "prefix_step_b64", "kind": "prefix", "P": 1, "B": 64, "q_lo": 1, "q_hi": 1, "pre_lo": 8192,
         "pre_hi": 8192, "ctx_lo": 100, "ctx_hi": 1500, "hq": 32, "hkv": 8, "d": 128, "page": 64, "ml": False, "pad": 2},
        # three documents of odd lengths with questions of a few tokens each, head dim 64, with the rows' statistics
        {"name": "prefix_groups_d64", "kind": "prefix", "P": 3, "B": 22, "q_lo": 1, "q_hi": 43, "pre_lo": 333,
         "pre_hi": 2999, "ctx_lo": 0, "ctx_hi": 150, "hq": 12, "hkv": 4, "d": 64, "page": 16, "ml": True, "pad": 3},
        # 32 first questions enter behind one instruction at once
        {"name": "prefix_chunks_b32", "kind": "prefix", "P": 1, "B": 32, "q_lo": 20, "q_hi": 200, "pre_lo": 8000,
         "pre_hi": 8000, "ctx_lo": 0, "ctx_hi": 0, "hq": 32, "hkv": 8, "d": 128, "page": 16, "ml": False, "pad": 0},
        # one request's next token
        {"name": "sample_b1", "kind": "sample", "B": 1, "V": 32000, "dtype": "bf16", "temperature": 0.7, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "rows": False, "masked": 0.0, "probs": False},
        # a batch whose requests each have their own settings, an odd vocabulary, half of it forbidden by a grammar
        {"name": "sample_rows_b64", "kind": "sample", "B": 64, "V": 50021, "dtype": "f32", "temperature": 0.9,
         "top_k": 50, "top_p": 0.95, "min_p": 0.02, "rows": True, "masked": 0.5, "probs": False},
        # a large batch over a large vocabulary, nucleus sampling alone
        {"name": "sample_b256", "kind": "sample", "B": 256, "V": 131072, "dtype": "f32", "temperature": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0, "rows": False, "masked": 0.0, "probs": False},
        # the distributions that a check of guessed tokens needs
        {"name": "sample_probs_b48", "kind": "sample", "B": 48, "V": 65536, "dtype": "bf16", "temperature": 0.8,
         "top_k": 200, "top_p": 0.98, "min_p": 0.0, "rows": False, "masked": 0.0, "probs": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["extend", "extend", "release", "prefix", "prefix", "prefix", "sample", "sample", "sample"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "extend":
        B = _log(rng, 1, 500)
        q = rng.choice([1, 1, _log(rng, 2, 5), _log(rng, 8, max(9, min(4096, 60000 // B)))])
        ctx = rng.choice([0, _log(rng, 10, 16000)])
        return {"kind": kind, "B": B, "q_lo": rng.choice([0, 1, q]), "q_hi": q, "ctx_lo": ctx // rng.choice([1, 2, 16]),
                "ctx_hi": ctx, "page": page, "pad": rng.choice([0, 0, _log(rng, 1, 300)]), "offsets": rng.random() < 0.4,
                # now and then the pool runs out
                "spare": rng.choice([1000, 200, 200, -3])}
    if kind == "release":
        hi = _log(rng, 16, 16000)
        return {"kind": kind, "B": _log(rng, 1, 512), "ctx_lo": hi // rng.choice([1, 3, 16]), "ctx_hi": hi, "page": page,
                "ended": rng.choice([0.05, 0.25, 0.5, 1.0]), "spare": rng.choice([0, 100, 1000])}
    if kind == "prefix":
        hkv = rng.choice([1, 2, 4, 8, 8, 12])
        hq = hkv * rng.choice([1, 2, 3, 4, 4, 7, 8])
        d = rng.choice([64, 128, 128, 128, 96])
        P = rng.choice([1, 1, 1, 2, 5])
        pre = _log(rng, 64, 16384)
        if rng.random() < 0.6:  # a generation step, now and then with a few guessed tokens
            B, q = max(P, _log(rng, 2, 128)), rng.choice([1, 1, 1, 2, 4])
            lo, ctx = q, rng.choice([0, _log(rng, 1, 2000)])
        else:
            B, q = max(P, _log(rng, 2, 32)), _log(rng, 8, 400)
            lo, ctx = max(1, q // 10), rng.choice([0, 0, _log(rng, 1, 1000)])
        while hq * B * q * (pre + ctx + q) > 5 << 27:  # no more pairs than the largest listed case
            pre, ctx, q = max(64, pre * 3 // 4), ctx * 3 // 4, max(lo, q * 3 // 4)
        return {"kind": kind, "P": P, "B": B, "q_lo": lo, "q_hi": q, "pre_lo": pre // rng.choice([1, 4]), "pre_hi": pre,
                "ctx_lo": ctx // 8, "ctx_hi": ctx, "hq": hq, "hkv": hkv, "d": d, "page": page,
                "ml": rng.random() < 0.3, "pad": rng.choice([0, 0, 3])}
    B = _log(rng, 1, 256)
    V = _log(rng, 1000, min(160000, (1 << 25) // B))
    return {"kind": kind, "B": B, "V": V, "dtype": rng.choice(["bf16", "f32"]),
            "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.3]), "top_k": rng.choice([0, 0, 1, 20, 50, 400]),
            "top_p": rng.choice([1.0, 0.99, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.01, 0.1]),
            "rows": rng.random() < 0.4, "masked": rng.choice([0.0, 0.0, 0.7]), "probs": rng.random() < 0.25}


# ------------------------------------------------------------------ inputs


def _spread(lo: int, hi: int, n: int) -> list[int]:
    """``n`` lengths between ``lo`` and ``hi``, even in their logarithm, short and long ones mixed."""
    if n == 1:
        return [hi]
    v = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]
    return v[::2] + v[1::2][::-1]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 31))


def _ints(v, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(v, dtype=dtype, device=DEV)


def _starts(n: list[int]) -> list[int]:
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _shuffled(g, v: list[int]) -> list[int]:
    """The same lengths dealt to the sequences in an order of the seed's."""
    return [v[i] for i in torch.randperm(len(v), device=DEV, generator=g).tolist()]


def _deal(order: torch.Tensor, need: list[int], width: int) -> torch.Tensor:
    """A table of rows of ``need`` pages each, in the order given, -1 behind the last."""
    want = _ints(need, torch.int64)
    at = torch.arange(width, device=DEV)[None, :]
    first = (torch.cumsum(want, 0) - want)[:, None]
    i = torch.clamp(first + at, max=max(order.numel() - 1, 0))
    return torch.where(at < want[:, None], order[i] if order.numel() else -1, -1).to(torch.int32)


def _pages_of(n: int, page: int) -> int:
    return -(-n // page)


def prepare(case: dict, seed: int) -> dict:
    g, kind = _gen(seed), case["kind"]
    st: dict = {"case": case}
    if kind in ("extend", "release"):
        B, page = case["B"], case["page"]
        ctx = _shuffled(g, _spread(case["ctx_lo"], case["ctx_hi"], B))
        held = [_pages_of(n, page) for n in ctx]
        new = _shuffled(g, _spread(case["q_lo"], case["q_hi"], B)) if kind == "extend" else [0] * B
        after = [_pages_of(n + x, page) for n, x in zip(ctx, new)]
        # the free pages that the step wants, and a few more or fewer of them
        free = max(sum(after) - sum(held) + case["spare"], 0)
        total = sum(held) + free
        order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
        st["table"] = _deal(order[:sum(held)], held, _pages_of(case["ctx_hi"] + case.get("q_hi", 0), page) + 2)
        st["lens"] = _ints(ctx)
        st["free"] = torch.full((max(total, 1),), -1, dtype=torch.int32, device=DEV)
        st["free"][:free] = order[sum(held):]
        st["count"] = _ints([free])
        if kind == "extend":
            st["n"], st["new"], st["ctx_host"], st["new_host"] = sum(new) + case["pad"], _ints(new), ctx, new
            st["offsets"] = None
            if case["offsets"]:
                st["offsets"] = torch.randint(0, 8192, (B,), device=DEV, generator=g, dtype=torch.int32)
        else:
            st["ended"] = torch.rand((B,), device=DEV, generator=g) < case["ended"]
        return st
    if kind == "prefix":
        P, B, hq, hkv, d, page = (case[x] for x in ("P", "B", "hq", "hkv", "d", "page"))
        nq, ctx = _prefix_lens(case)
        nq, ctx = _shuffled(g, nq), _shuffled(g, ctx)
        pre = _spread(case["pre_lo"], case["pre_hi"], P)
        lens = [a + b for a, b in zip(nq, ctx)]
        st["nq"], st["pre_host"], st["lens_host"] = nq, pre, lens
        st["groups"] = [B * p // P for p in range(P + 1)]
        need, pre_need = [_pages_of(n, page) for n in lens], [_pages_of(n, page) for n in pre]
        total = sum(need) + sum(pre_need)
        n_pages = total + max(1, total // 8)
        order = torch.randperm(n_pages, device=DEV, generator=g)[:total].to(torch.int32)
        rows = B + case["pad"]  # idle entries keep their rows of a padded batch
        st["table"] = _deal(order[sum(pre_need):], need + [0] * case["pad"], max(max(need), 1))
        st["pre_table"] = _deal(order, pre_need, max(max(pre_need), 1))
        st["lens"], st["pre_lens"] = _ints(lens + [0] * case["pad"]), _ints(pre)
        st["starts"] = _ints(_starts(nq + [0] * case["pad"]))
        st["pre_starts"] = _ints(st["groups"])
        n = sum(nq) + case["pad"]
        qkv = torch.randn((n, (hq + 2 * hkv) * d), device=DEV, generator=g).to(BF16)  # one projection's rows
        st["q"] = qkv[:, :hq * d].unflatten(1, (-1, d))
        st["kp"], st["vp"] = (torch.randn((n_pages, hkv, page, d), device=DEV, generator=g).to(BF16) for _ in range(2))
        st["out"] = torch.zeros((n, hq, d), dtype=BF16, device=DEV)
        assert rows == st["table"].shape[0]
        return st
    B, V = case["B"], case["V"]
    # sharp and flat distributions, a few words far above the others
    x = torch.randn((B, V), device=DEV, generator=g)
    x *= 1 + 2 * torch.rand((B, 1), device=DEV, generator=g)
    top = torch.randint(0, V, (B, 24), device=DEV, generator=g)
    x.scatter_add_(1, top, 4 + 8 * torch.rand((B, 24), device=DEV, generator=g))
    if case["masked"]:
        off = torch.rand((B, V), device=DEV, generator=g) < case["masked"]
        off[:, :7] = False
        x = torch.where(off, -math.inf, x)
    st["logits"] = x.to(BF16 if case["dtype"] == "bf16" else torch.float32)
    st["u"] = torch.rand((B,), device=DEV, generator=g)
    for name, dt in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
        st[name] = case[name]
        if case["rows"]:  # some requests leave a setting off, some are greedy
            v = torch.full((B,), case[name], dtype=torch.float32, device=DEV)
            v *= 0.6 + 0.4 * torch.rand((B,), device=DEV, generator=g)
            neutral = {"temperature": 0.0, "top_k": 0.0, "top_p": 1.0, "min_p": 0.0}[name]
            v = torch.where(torch.rand((B,), device=DEV, generator=g) < 0.2, neutral, v)
            st[name] = v.to(dt)
    return st


def _prefix_lens(case: dict) -> tuple[list[int], list[int]]:
    """The sequences' new tokens and the own keys cached before them, before they are dealt out."""
    return _spread(case["q_lo"], case["q_hi"], case["B"]), _spread(case["ctx_lo"], case["ctx_hi"], case["B"])


# --------------------------------------------------------------- plain forms


def _plain_extend(st: dict) -> dict:
    case, table = st["case"], st["table"]
    page, n, reach = case["page"], st["n"], st["table"].shape[1] * case["page"]
    kv = st["lens"].long()
    starts = torch.zeros((kv.numel() + 1,), dtype=torch.int64, device=DEV)
    starts[1:] = torch.clamp(torch.cumsum(torch.clamp(st["new"], min=0), 0), max=n)
    after = torch.clamp(kv + starts[1:] - starts[:-1], max=reach)
    held = (kv + page - 1) // page
    need = (after + page - 1) // page - held
    first = torch.cumsum(need, 0) - need
    # a new page takes the last free one that is left
    i = torch.arange(table.shape[1], device=DEV)[None, :] - held[:, None]
    left = st["count"].long() - 1 - (first[:, None] + i)
    page_id = torch.where(left >= 0, st["free"][torch.clamp(left, min=0)], -1)
    table.copy_(torch.where((i >= 0) & (i < need[:, None]), page_id, table))
    t = torch.arange(n, device=DEV)
    b = torch.searchsorted(starts[1:], t, right=True)
    real = b < kv.numel()
    b = torch.clamp(b, max=kv.numel() - 1)
    key = kv[b] + t - starts[b]
    at = table[b, torch.clamp(key // page, max=table.shape[1] - 1)].long()
    slots = torch.where(real & (at >= 0) & (key < reach), at * page + key % page, -1)
    if st["offsets"] is not None:
        key = key + st["offsets"].long()[b]
    return {"starts": starts.int(), "positions": torch.where(real, key, 0), "slots": slots, "lens": after.int(),
            "count": torch.clamp(st["count"] - need.sum(), min=0).int(), "table": table}


def _plain_release(st: dict) -> dict:
    case, table, free = st["case"], st["table"], st["free"]
    held = (st["lens"] + case["page"] - 1) // case["page"]
    i = torch.arange(table.shape[1], device=DEV)[None, :]
    gone = (st["ended"][:, None] & (i < held[:, None]) & (table >= 0)).flatten()
    to = st["count"] - 1 + torch.cumsum(gone, 0)
    # what is not given back lands behind the pool's end
    grown = torch.cat([free, free[:1]])
    grown[torch.where(gone, to, free.numel())] = table.flatten()
    free.copy_(grown[:-1])
    return {"free": free, "lens": torch.where(st["ended"], 0, st["lens"]), "count": st["count"] + gone.sum().int()}


def _part(q, k, v, seen, scale):
    """Scores of padded rows q (R, Q, hq, d) with k and v (R, hkv, L, d): m, l (R, Q, hq) and the numerators."""
    R, Q, hq, d = q.shape
    hkv = k.shape[1]
    rows = q.transpose(1, 2).reshape(R, hkv, hq // hkv * Q, d)
    s = (torch.matmul(rows, k.transpose(-1, -2)) * scale).unflatten(2, (hq // hkv, Q))
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.amax(-1)
    e = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0)[..., None])
    acc = torch.matmul(e.flatten(2, 3), v).unflatten(2, (hq // hkv, Q))
    return tuple(t.flatten(1, 2).transpose(1, 2) for t in (m, e.sum(-1), acc))


def _keys(pages: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    rows = pages[torch.clamp(table, min=0).long()]
    return rows.transpose(1, 2).flatten(2, 3)[:, :, :n].float()


def _plain_prefix(st: dict) -> dict:
    case, q, out = st["case"], st["q"], st["out"]
    B, P, n, scale = case["B"], case["P"], sum(st["nq"]), case["d"] ** -0.5
    starts, firsts = st["starts"].long(), st["pre_starts"].long()
    t = torch.arange(n, device=DEV)
    b = torch.searchsorted(starts[1:B + 1], t, right=True)
    p = torch.searchsorted(firsts[1:], b, right=True)
    i, r = t - starts[b], t - starts[firsts[p]]
    Q, L = max(st["nq"]), max(st["lens_host"])
    qs = torch.zeros((B, Q, *q.shape[1:]), device=DEV)
    qs[b, i] = q[:n].float()
    lens, nq = st["lens"][:B].long(), starts[1:B + 1] - starts[:B]
    last = (lens - nq)[:, None] + torch.arange(Q, device=DEV)
    seen = torch.arange(L, device=DEV) <= torch.minimum(last, lens[:, None] - 1)[..., None]
    mo, lo, ao = (x[b, i] for x in _part(qs, _keys(st["kp"], st["table"][:B], L), _keys(st["vp"], st["table"][:B], L), seen, scale))
    # the prefix: all rows of a group against the same keys
    R, L = max(sum(st["nq"][x:y]) for x, y in zip(st["groups"], st["groups"][1:])), max(st["pre_host"])
    qs = torch.zeros((P, R, *q.shape[1:]), device=DEV)
    qs[p, r] = q[:n].float()
    seen = (torch.arange(L, device=DEV) < st["pre_lens"][:, None])[:, None].expand(P, R, L)
    mp, lp, ap = (x[p, r] for x in _part(qs, _keys(st["kp"], st["pre_table"], L), _keys(st["vp"], st["pre_table"], L), seen, scale))
    m = torch.maximum(mo, mp)
    fo, fp = torch.exp(mo - m), torch.exp(mp - m)
    l = lo * fo + lp * fp
    out[:n] = ((ao * fo[..., None] + ap * fp[..., None]) / l[..., None]).to(BF16)
    return {"o": out, "m": m, "l": l} if case["ml"] else {"o": out}


def _rows_of(st: dict, name: str, dtype=torch.float64) -> torch.Tensor:
    v = st[name]
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((st["case"]["B"], 1), v, dtype=dtype, device=DEV)


def _plain_sample(st: dict) -> dict:
    # in 64 bits: a token is the first whose sum of weights passes a border
    x = st["logits"]
    V = x.shape[1]
    T, k, p, low = (_rows_of(st, n) for n in ("temperature", "top_k", "top_p", "min_p"))
    top, order = torch.sort(x.float(), dim=-1, descending=True, stable=True)
    z = top.double() - top[:, :1].double()
    w = torch.exp(torch.where(z == 0, 0.0, z / T))  # temperature 0: nothing below the largest
    rank = torch.arange(V, device=DEV)
    k = torch.where(T == 0, 1.0, torch.where(k > 0, k, float(V)))
    w = torch.where(rank < k, w, 0.0)
    cum = torch.cumsum(w, -1)
    kept = (w > 0) & (w >= low) & ((cum - w < p * cum[:, -1:]) | (p >= 1))
    kept[:, 0] = True
    w = torch.where(kept, w, 0.0)
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    at = torch.clamp((cum <= st["u"].double()[:, None] * total).sum(-1, keepdim=True), max=V - 1)
    at = torch.minimum(at, kept.sum(-1, keepdim=True) - 1)
    res = {"tokens": torch.gather(order, 1, at)[:, 0],
           "logprobs": torch.log(torch.gather(w, 1, at) / total)[:, 0].float()}
    if st["case"]["probs"]:
        res["probs"] = torch.zeros_like(w).scatter_(1, order, w / total).float()
    return res


# -------------------------------------------------------------------- calls


def run(state: dict):
    st, case = state, state["case"]
    kind = case["kind"]
    if not own:
        return {"extend": _plain_extend, "release": _plain_release, "prefix": _plain_prefix, "sample": _plain_sample}[kind](st)
    from catopt_amd import paged, sampling

    if kind == "extend":
        r = paged.paged_extend(st["table"], st["lens"], st["new"], st["free"], st["count"], st["n"], case["page"],
                               offsets=st["offsets"])
        return {"starts": r.q_starts, "positions": r.positions, "slots": r.slots, "lens": r.kv_lens,
                "count": r.free_count, "table": st["table"]}
    if kind == "release":
        lens, count = paged.paged_release(st["table"], st["lens"], st["ended"], st["free"], st["count"], case["page"])
        return {"free": st["free"], "lens": lens, "count": count}
    if kind == "prefix":
        r = paged.paged_prefix_attention(st["q"], st["kp"], st["vp"], st["pre_table"], st["pre_lens"], st["pre_starts"],
                                         st["table"], st["lens"], st["starts"], case["d"] ** -0.5, out=st["out"],
                                         return_ml=case["ml"])
        if not case["ml"]:
            return {"o": r}
        return {"o": r[0], "m": r[1][:sum(st["nq"])], "l": r[2][:sum(st["nq"])]}
    r = sampling.sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
                        return_probs=case["probs"])
    return dict(zip(("tokens", "logprobs", "probs"), r))


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind in ("extend", "release"):
        ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["B"])
        held = sum(_pages_of(n, case["page"]) for n in ctx)
        if kind == "release":  # every ended sequence's pages read and written once
            return {"bytes": 9 * case["B"] + 8 * held * case["ended"], "flops": held * case["ended"]}
        n = sum(_spread(case["q_lo"], case["q_hi"], case["B"]))
        # lengths in and out, a slot and a position per token, the new pages out of the pool and into the table
        return {"bytes": case["B"] * (16 + 4 * case["offsets"]) + 16 * (n + case["pad"]) + 8 * (n // case["page"] + 1),
                "flops": 4 * n}
    if kind == "prefix":
        (nq, ctx), hq, hkv, d = _prefix_lens(case), case["hq"], case["hkv"], case["d"]
        pre = _spread(case["pre_lo"], case["pre_hi"], case["P"])
        pairs = sum(q * (q + 1) // 2 for q in nq) + sum(nq) * (sum(pre) / len(pre) + sum(ctx) / len(ctx))
        keys = sum(nq) + sum(ctx) + sum(pre)
        return {"bytes": 4 * sum(nq) * hq * d + 4 * keys * hkv * d + 4 * keys // case["page"] + 8 * sum(nq) * hq * case["ml"],
                "flops": 4 * pairs * hq * d}
    n = case["B"] * case["V"]
    return {"bytes": n * ((2 if case["dtype"] == "bf16" else 4) + 4 * case["probs"]) + 16 * case["B"], "flops": 8 * n}


# ---------------------------------------------------------- 64-bit references


def _exact_extend(st: dict) -> dict:
    page, n = st["case"]["page"], st["n"]
    table, free, left = st["table"].cpu().numpy().copy(), st["free"].cpu().numpy(), int(st["count"])
    slots, positions = np.full((n,), -1, dtype=np.int64), np.zeros((n,), dtype=np.int64)
    offsets = np.zeros(len(st["new_host"]), dtype=np.int64) if st["offsets"] is None else st["offsets"].cpu().numpy()
    at, starts, lens = 0, [0], []
    for b, (have, new) in enumerate(zip(st["ctx_host"], st["new_host"])):
        for i in range(_pages_of(have, page), _pages_of(have + new, page)):
            left -= 1
            table[b, i] = free[left] if left >= 0 else -1
        keys = np.arange(have, have + new)
        ids = table[b, keys // page].astype(np.int64)
        slots[at:at + new] = np.where(ids >= 0, ids * page + keys % page, -1)
        positions[at:at + new] = keys + offsets[b]
        at += new
        starts.append(at)
        lens.append(have + new)
    return {"starts": _ints(starts), "positions": torch.from_numpy(positions).to(DEV), "slots": torch.from_numpy(slots).to(DEV),
            "lens": _ints(lens), "count": _ints([max(left, 0)]), "table": torch.from_numpy(table).to(DEV)}


def _exact_release(st: dict) -> dict:
    page, table, free = st["case"]["page"], st["table"].tolist(), st["free"].tolist()
    ended, lens, count = st["ended"].tolist(), st["lens"].tolist(), int(st["count"])
    for b, gone in enumerate(ended):
        if gone:
            for x in table[b][:_pages_of(lens[b], page)]:
                free[count] = x
                count += 1
            lens[b] = 0
    return {"free": _ints(free), "lens": _ints(lens), "count": _ints([count])}


def _exact_prefix(st: dict) -> dict:
    case = st["case"]
    hq, hkv, d, page = (case[x] for x in ("hq", "hkv", "d", "page"))
    n = sum(st["nq"])
    o = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV)
    m, l = (torch.zeros((n, hq), dtype=torch.float64, device=DEV) for _ in range(2))
    row0 = 0
    for p, pre in enumerate(st["pre_host"]):
        for b in range(st["groups"][p], st["groups"][p + 1]):
            nq, mine = st["nq"][b], st["lens_host"][b]
            jp, jo = torch.arange(pre, device=DEV), torch.arange(mine, device=DEV)
            slot = torch.cat([st["pre_table"][p].long()[jp // page] * page + jp % page,
                              st["table"][b].long()[jo // page] * page + jo % page])
            late = torch.arange(pre + mine, device=DEV)[None] > (pre + mine - nq + torch.arange(nq, device=DEV))[:, None]
            rows = slice(row0, row0 + nq)
            for kv in range(hkv):
                keys = st["kp"][:, kv].reshape(-1, d)[slot].double()
                vals = st["vp"][:, kv].reshape(-1, d)[slot].double()
                h = slice(kv * (hq // hkv), (kv + 1) * (hq // hkv))
                s = torch.tensordot(st["q"][rows, h].double(), keys, dims=([2], [1])) / math.sqrt(d)  # (nq, heads, keys)
                s.masked_fill_(late[:, None], -math.inf)
                o[rows, h] = torch.softmax(s, -1) @ vals
                m[rows, h] = s.max(-1).values
                l[rows, h] = torch.exp(torch.logsumexp(s, -1) - m[rows, h])
            row0 += nq
    return {"o": o, "m": m, "l": l} if case["ml"] else {"o": o}


def _exact_sample(st: dict) -> dict:
    case = st["case"]
    x = st["logits"].double().cpu().numpy()
    B, V = x.shape
    T, k, p, low = ((st[n].double().cpu().numpy() if isinstance(st[n], torch.Tensor) else np.full(B, float(st[n])))
                    for n in ("temperature", "top_k", "top_p", "min_p"))
    u = st["u"].double().cpu().numpy()
    tokens, logs = np.zeros(B, dtype=np.int64), np.zeros(B)
    probs = np.zeros((B, V)) if case["probs"] else None
    for b in range(B):
        order = np.argsort(-x[b], kind="stable")
        if T[b] == 0:
            order = order[:1]
        if k[b] > 0:
            order = order[:int(k[b])]
        z = x[b, order] - x[b, order[0]]
        w = np.exp(z / T[b]) if T[b] else np.ones(1)
        if p[b] < 1:  # up to the first rank whose sum reaches the share
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p[b] * w.sum(), side="left"))]
        order = order[w[:len(order)] >= max(low[b], 1e-300)]
        w = w[:len(order)]
        total = w.sum()
        i = min(int(np.searchsorted(np.cumsum(w), u[b] * total, side="right")), len(w) - 1)
        tokens[b], logs[b] = order[i], np.log(w[i] / total)
        if probs is not None:
            probs[b, order] = w / total
    res = {"tokens": torch.from_numpy(tokens).to(DEV), "logprobs": torch.from_numpy(logs).to(DEV)}
    if probs is not None:
        res["probs"] = torch.from_numpy(probs).to(DEV)
    return res


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"extend": _exact_extend, "release": _exact_release, "prefix": _exact_prefix, "sample": _exact_sample}[case["kind"]](st)
