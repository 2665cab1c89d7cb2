"""The operators of a paged key/value cache as measurable cases.

A case is a plain dict; ``kind`` names the operator it calls:

* ``rope``  -- the per-head RMS norm of queries and keys and their position rotation in one pass, returned
               (``paged.qk_norm_rope``) or, with ``append``, with keys and values written into the cache's pages
               (``paged.qk_norm_rope_append``);
* ``attn``  -- attention of each sequence's chunk of new tokens over its paged cache
               (``paged.paged_attention``), with ``weights`` also adding every key's attention weight to a running sum;
* ``evict`` -- the move of each head's most attended and most recent keys into a cache of fixed size
               (``paged.paged_evict``).

``run`` computes the plain form in elementary torch operations; with ``own`` set it calls the kernels.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
POSITIONS = 32768  # rows of the cos / sin tables


def listed() -> list[dict]:
    return [
        # one generation step of 8 sequences: the smallest call, a few microseconds of work
        {"name": "rope_step_n8", "kind": "rope", "n": 8, "B": 8, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "pairs": False, "norm": True, "append": True, "page": 16, "dtype": "bf16"},
        # chunks of an odd length, a partial rotation of adjacent pairs, kept out of the cache
        {"name": "rope_n1237_d64", "kind": "rope", "n": 1237, "B": 3, "hq": 12, "hkv": 12, "d": 64, "rot": 32,
         "pairs": True, "norm": True, "append": False, "page": 16, "dtype": "f32"},
        # the prompts of the attention configuration (4 x 4096 tokens, 32 heads of 128) entering the cache
        {"name": "rope_n16384", "kind": "rope", "n": 16384, "B": 4, "hq": 32, "hkv": 32, "d": 128, "rot": 128,
         "pairs": False, "norm": True, "append": True, "page": 64, "dtype": "bf16"},
        # one token of one sequence against a cache of 8192 keys, eight key heads
        {"name": "attn_step_b1_k8192", "kind": "attn", "B": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 8191, "ctx_hi": 8191,
         "hq": 32, "hkv": 8, "d": 128, "page": 16, "weights": False, "ml": False, "pad": 0},
        # a generation step of 32 sequences of very different lengths, two idle entries behind them
        {"name": "attn_step_b32", "kind": "attn", "B": 32, "q_lo": 1, "q_hi": 1, "ctx_lo": 300, "ctx_hi": 16000,
         "hq": 32, "hkv": 8, "d": 128, "page": 64, "weights": False, "ml": False, "pad": 2},
        # short chunks of odd lengths over odd contexts, head dim 64, with the rows' statistics
        {"name": "attn_chunk_q77_d64", "kind": "attn", "B": 5, "q_lo": 33, "q_hi": 171, "ctx_lo": 517,
         "ctx_hi": 1999, "hq": 12, "hkv": 4, "d": 64, "page": 16, "weights": False, "ml": True, "pad": 0},
        # one long chunk of a prompt behind an already cached part
        {"name": "attn_chunk_q2048", "kind": "attn", "B": 1, "q_lo": 2048, "q_hi": 2048, "ctx_lo": 6144,
         "ctx_hi": 6144, "hq": 32, "hkv": 8, "d": 128, "page": 16, "weights": False, "ml": False, "pad": 0},
        # whole prompts at the attention configuration's shape
        {"name": "attn_prompt_b4_q4096", "kind": "attn", "B": 4, "q_lo": 4096, "q_hi": 4096, "ctx_lo": 0,
         "ctx_hi": 0, "hq": 32, "hkv": 32, "d": 128, "page": 64, "weights": False, "ml": False, "pad": 0},
        # a generation step that also adds up the keys' weights for a later eviction
        {"name": "attn_step_weights", "kind": "attn", "B": 8, "q_lo": 1, "q_hi": 1, "ctx_lo": 2000, "ctx_hi": 12000,
         "hq": 32, "hkv": 8, "d": 128, "page": 16, "weights": True, "ml": False, "pad": 0},
        # a chunk of a prompt whose keys' weights are added up
        {"name": "attn_chunk_weights", "kind": "attn", "B": 2, "q_lo": 700, "q_hi": 1100, "ctx_lo": 1500,
         "ctx_hi": 3500, "hq": 32, "hkv": 8, "d": 128, "page": 16, "weights": True, "ml": False, "pad": 0},
        # one sequence leaves three quarters of 2048 keys behind
        {"name": "evict_b1_k2048", "kind": "evict", "B": 1, "len_lo": 2048, "len_hi": 2048, "budget": 512, "recent": 64,
         "hkv": 8, "d": 128, "page": 16},
        # long prompts cut to 2048 keys a head before generation, one shorter than that
        {"name": "evict_b8_k16000", "kind": "evict", "B": 8, "len_lo": 1500, "len_hi": 16000, "budget": 2048,
         "recent": 256, "hkv": 8, "d": 128, "page": 64},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "rope", "attn", "attn", "attn", "attn", "evict"])
    d = rng.choice([64, 128, 128, 128, 96])
    hkv = rng.choice([1, 2, 4, 8, 8, 12])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "rope":
        n = _log(rng, 1, 8192)
        pairs = rng.random() < 0.4
        return {"kind": kind, "n": n, "B": min(n, _log(rng, 1, 32)), "hq": hkv * rng.choice([1, 2, 3, 4, 8]),
                "hkv": hkv, "d": d, "rot": rng.choice([d, d, 32]), "pairs": pairs, "norm": rng.random() < 0.8,
                "append": rng.random() < 0.6, "page": page, "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    if kind == "attn":
        g = rng.choice([1, 2, 3, 4, 4, 7, 8])
        hq = hkv * g
        weights = rng.random() < 0.4
        if rng.random() < 0.5:  # a generation step, now and then with a few guessed tokens
            B, q = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
            hi = _log(rng, 16, max(17, min(16384, (1 << 22) // (B * hkv))))
            return {"kind": kind, "B": B, "q_lo": q, "q_hi": q, "ctx_lo": _log(rng, 8, hi), "ctx_hi": hi, "hq": hq,
                    "hkv": hkv, "d": d, "page": page, "weights": weights, "ml": rng.random() < 0.3,
                    "pad": rng.choice([0, 0, 3])}
        B = rng.randint(1, 5)
        q = _log(rng, 8, 2048)
        ctx = rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 8192)])
        while hq * B * q * (ctx + q) > 1 << 30:  # no more pairs than the largest listed case
            B, q = max(1, B // 2), q - q // 4
        return {"kind": kind, "B": B, "q_lo": max(1, q // 3), "q_hi": q, "ctx_lo": ctx // 2, "ctx_hi": ctx,
                "hq": hq, "hkv": hkv, "d": d, "page": page, "weights": weights, "ml": rng.random() < 0.3, "pad": 0}
    B = _log(rng, 1, 16)
    hi = _log(rng, 64, 16384)
    budget = _log(rng, 16, min(hi, 4096))
    return {"kind": kind, "B": B, "len_lo": max(1, hi // rng.choice([1, 2, 8])), "len_hi": hi, "budget": budget,
            "recent": rng.choice([0, budget // 8, budget // 2, budget]), "hkv": hkv, "d": d, "page": page}


# ------------------------------------------------------------------ inputs


def _spread(lo: int, hi: int, n: int) -> list[int]:
    """``n`` lengths between ``lo`` and ``hi``, even in their logarithm, short and long ones mixed."""
    v = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / max(n - 1, 1)))) - 1 for i in range(n)]
    if n == 1:
        v = [hi]
    return v[::2] + v[1::2][::-1]


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's new tokens and the keys cached before them."""
    return _spread(case["q_lo"], case["q_hi"], case["B"]), _spread(case["ctx_lo"], case["ctx_hi"], case["B"])


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 31))


def _randn(g, *shape, dtype=BF16, scale: float = 1.0) -> torch.Tensor:
    t = torch.randn(shape, device=DEV, generator=g)
    return (t.mul_(scale) if scale != 1.0 else t).to(dtype)


def _tables(g, lens: list[int], page: int, rows: int) -> tuple[torch.Tensor, int]:
    """A block table for sequences of these lengths (pages dealt in no order, -1 behind the last), and the pages."""
    need = [-(-n // page) for n in lens]
    total = sum(need)
    n_pages = total + max(1, total // 8)
    order = torch.randperm(n_pages, device=DEV, generator=g)[:total].to(torch.int32)
    table = torch.full((rows, max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, n_pages


def _ints(v, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(v, dtype=dtype, device=DEV)


def _starts(n: list[int]) -> list[int]:
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _rope_tables(rot: int) -> tuple[torch.Tensor, torch.Tensor]:
    # angles of far positions lose their fraction in 32 bits
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    ang = torch.arange(POSITIONS, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cos(ang).float(), torch.sin(ang).float()


def prepare(case: dict, seed: int) -> dict:
    g, kind = _gen(seed), case["kind"]
    st: dict = {"case": case}
    if kind == "rope":
        n, B, hq, hkv, d, page = (case[x] for x in ("n", "B", "hq", "hkv", "d", "page"))
        dt = BF16 if case["dtype"] == "bf16" else torch.float32
        qkv = _randn(g, n, (hq + 2 * hkv) * d, dtype=dt)  # one projection's rows, as a model has them
        st["q"], st["k"], st["v"] = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
        st["qw"] = st["kw"] = None
        if case["norm"]:
            st["qw"], st["kw"] = (1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(dt), \
                (1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(dt)
        st["cos"], st["sin"] = _rope_tables(case["rot"])
        lens = [n // B + (b < n % B) for b in range(B)]
        ctx = torch.randint(0, POSITIONS - max(lens), (B,), device=DEV, generator=g).tolist()
        st["pos"] = torch.cat([torch.arange(c, c + x, device=DEV) for c, x in zip(ctx, lens)])
        if case["append"]:
            table, n_pages = _tables(g, [page - 1 + x for x in lens], page, B)  # wherever in a page they begin
            at = [torch.arange(c % page, c % page + x, device=DEV) for c, x in zip(ctx, lens)]
            st["slots"] = torch.cat([table[b].long()[a // page] * page + a % page for b, a in enumerate(at)])
            st["kp"], st["vp"] = _randn(g, n_pages, hkv, page, d, dtype=dt), _randn(g, n_pages, hkv, page, d, dtype=dt)
        return st
    hkv, d, page = (case[x] for x in ("hkv", "d", "page"))
    if kind == "attn":
        nq, ctx = _lens(case)
        lens = [a + b for a, b in zip(nq, ctx)]
        rows = case["B"] + case["pad"]
        st["nq"], st["lens_host"] = nq, lens
        st["table"], n_pages = _tables(g, lens, page, rows)
        starts = _starts(nq + [0] * case["pad"])
        st["starts"], st["lens"] = _ints(starts), _ints(lens + [0] * case["pad"])
        n = starts[-1]
        qkv = _randn(g, n + case["pad"], (case["hq"] + 2 * hkv) * d)  # idle entries keep their rows of a padded batch
        st["q"] = qkv[:, :case["hq"] * d].unflatten(1, (-1, d))
        st["kp"], st["vp"] = _randn(g, n_pages, hkv, page, d), _randn(g, n_pages, hkv, page, d)
        st["out"] = torch.zeros((n + case["pad"], case["hq"], d), dtype=BF16, device=DEV)
        if case["weights"]:
            cap = st["table"].shape[1] * page
            st["w"] = torch.rand((rows, hkv, cap), device=DEV, generator=g).pow_(3).mul_(4)
            st["w_out"] = torch.zeros_like(st["w"])
        return st
    lens = _spread(case["len_lo"], case["len_hi"], case["B"])
    st["lens_host"], st["lens"] = lens, _ints(lens)
    st["table"], n_pages = _tables(g, lens, page, case["B"])
    st["kp"], st["vp"] = _randn(g, n_pages, hkv, page, d), _randn(g, n_pages, hkv, page, d)
    w = torch.rand((case["B"], hkv, st["table"].shape[1] * page), device=DEV, generator=g).pow_(3).mul_(8)
    st["w"] = torch.where(w < 1e-3, torch.zeros_like(w), w)  # keys that no query looked at tie at zero
    st["out_table"], out_pages = _tables(g, [min(n, case["budget"]) for n in lens], page, case["B"])
    st["ko"], st["vo"] = (torch.zeros((out_pages, hkv, page, d), dtype=BF16, device=DEV) for _ in range(2))
    st["w_out"] = torch.zeros((case["B"], hkv, case["budget"]), device=DEV)
    return st


# --------------------------------------------------------------- plain forms


def _rotate(x: torch.Tensor, w, cos: torch.Tensor, sin: torch.Tensor, rot: int, pairs: bool) -> torch.Tensor:
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if pairs else (y[..., :rot // 2], y[..., rot // 2:rot])
    c, s = cos[:, None, :], sin[:, None, :]
    ra, rb = a * c - b * s, b * c + a * s
    head = torch.stack([ra, rb], -1).flatten(-2) if pairs else torch.cat([ra, rb], -1)
    return torch.cat([head, y[..., rot:]], -1).to(x.dtype)


def _plain_rope(st: dict):
    case = st["case"]
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    q = _rotate(st["q"], st["qw"], cos, sin, case["rot"], case["pairs"])
    k = _rotate(st["k"], st["kw"], cos, sin, case["rot"], case["pairs"])
    if not case["append"]:
        return {"q": q, "k": k}
    page, off = st["slots"] // case["page"], st["slots"] % case["page"]
    st["kp"][page, :, off] = k
    st["vp"][page, :, off] = st["v"]
    return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"]}


def _cached(pages: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """The first ``n`` cached rows of one sequence, ``(heads, n, d)``."""
    page = pages.shape[2]
    rows = pages[table[:-(-n // page)].long()]
    return rows.transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_attn(st: dict):
    case, out = st["case"], st["out"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, at = hq // hkv, 0
    ms, ls = [], []
    for b, (nq, n) in enumerate(zip(st["nq"], st["lens_host"])):
        k, v = (_cached(st[p], st["table"][b], n).float() for p in ("kp", "vp"))
        seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(n - nq, n, device=DEV)[:, None]
        q = st["q"][at:at + nq].float().transpose(0, 1).unflatten(0, (hkv, g))
        heads = max(1, min(hkv, (1 << 27) // (g * nq * n)))  # as many at once as fit beside their scores
        for h in range(0, hkv, heads):
            kh, vh = k[h:h + heads, None], v[h:h + heads, None]
            s = torch.matmul(q[h:h + heads], kh.transpose(-1, -2)) * d ** -0.5
            s = torch.where(seen, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - m)
            l = e.sum(-1, keepdim=True)
            out[at:at + nq, h * g:(h + heads) * g] = (torch.matmul(e, vh) / l).flatten(0, 1).transpose(0, 1).to(BF16)
            if case["weights"]:
                w = (e / l).sum((1, 2))
                w[:, :n - nq] += st["w"][b, h:h + heads, :n - nq]  # the new keys start from nothing
                st["w_out"][b, h:h + heads, :n] = w
            if case["ml"]:
                ms.append(m.flatten(0, 1)[..., 0])
                ls.append(l.flatten(0, 1)[..., 0])
        if case["ml"]:  # this sequence's head groups side by side, (tokens, heads)
            for t in (ms, ls):
                groups = -(-hkv // heads)
                t[-groups:] = [torch.cat(t[-groups:]).t()]
        at += nq
    res = {"o": out}
    if case["weights"]:
        res["weights"] = st["w_out"]
    if case["ml"]:
        res["m"], res["l"] = torch.cat(ms), torch.cat(ls)
    return res


def _plain_evict(st: dict):
    case = st["case"]
    budget, recent, page = case["budget"], case["recent"], case["page"]
    kept = torch.full((case["B"], case["hkv"], budget), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(st["lens_host"]):
        m = min(n, budget)
        # the last `recent` keys, and the most attended of the others, the first of equals
        old = max(n - min(recent, m), 0)
        best = torch.sort(st["w"][b, :, :old], dim=-1, descending=True, stable=True).indices[:, :m - (n - old)]
        last = torch.arange(old, n, device=DEV).expand(case["hkv"], -1)
        idx = torch.sort(torch.cat([best, last], -1), dim=-1).values
        kept[b, :, :m] = idx.to(torch.int32)
        st["w_out"][b, :, :m] = torch.gather(st["w"][b], 1, idx)
        to = torch.arange(m, device=DEV)
        dst, off = st["out_table"][b].long()[to // page], to % page
        for src, out in ((st["kp"], st["ko"]), (st["vp"], st["vo"])):
            rows = torch.gather(_cached(src, st["table"][b], n), 1, idx[..., None].expand(-1, -1, case["d"]))
            out[dst, :, off] = rows.transpose(0, 1)
    return {"kept": kept, "lens": torch.clamp(st["lens"], max=budget), "weights": st["w_out"], "k_pages": st["ko"],
            "v_pages": st["vo"]}


# -------------------------------------------------------------------- calls


def run(state: dict):
    st, case = state, state["case"]
    kind = case["kind"]
    if not own:
        return {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict}[kind](st)
    from catopt_amd import paged

    if kind == "rope":
        norm = {"q_weight": st["qw"], "k_weight": st["kw"], "eps": 1e-6, "interleaved": case["pairs"]}
        if not case["append"]:
            q, k = paged.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], st["pos"], **norm)
            return {"q": q, "k": k}
        q = paged.qk_norm_rope_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["kp"], st["vp"],
                                      st["slots"], **norm)
        return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"]}
    if kind == "attn":
        kw = {"weights": st["w"], "weights_out": st["w_out"]} if case["weights"] else {}
        r = paged.paged_attention(st["q"], st["kp"], st["vp"], st["table"], st["lens"], st["starts"], case["d"] ** -0.5,
                                  out=st["out"], return_ml=case["ml"], **kw)
        res = {"o": r[0] if case["ml"] else r}
        if case["weights"]:
            res["weights"] = st["w_out"]
        if case["ml"]:
            n = st["nq"]
            res["m"], res["l"] = (t[:sum(n)] for t in r[1:])
        return res
    kept, lens, w = paged.paged_evict(st["kp"], st["vp"], st["table"], st["lens"], st["w"], st["out_table"],
                                      case["budget"], case["recent"], k_out=st["ko"], v_out=st["vo"],
                                      weights_out=st["w_out"])
    return {"kept": kept, "lens": lens, "weights": w, "k_pages": st["ko"], "v_pages": st["vo"]}


def work(case: dict) -> dict:
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind == "rope":
        n, hq, size = case["n"], case["hq"], 2 if case["dtype"] == "bf16" else 4
        heads = hq + (2 if case["append"] else 1) * hkv
        # the rows in and out, one row of each table per token, positions and slots
        return {"bytes": n * (2 * heads * d * size + 4 * case["rot"] + 8 * (1 + case["append"])),
                "flops": n * (hq + hkv) * (4 * d * case["norm"] + 3 * case["rot"])}
    if kind == "attn":
        nq, ctx = _lens(case)
        pairs = sum(q * c + q * (q + 1) // 2 for q, c in zip(nq, ctx))
        keys = sum(nq) + sum(ctx)
        nbytes = 4 * sum(nq) * case["hq"] * d + 4 * keys * hkv * d + 4 * keys // case["page"]
        if case["weights"]:
            nbytes += 4 * hkv * (sum(ctx) + keys)
        if case["ml"]:
            nbytes += 8 * sum(nq) * case["hq"]
        return {"bytes": nbytes, "flops": 4 * pairs * case["hq"] * d}
    lens = _spread(case["len_lo"], case["len_hi"], case["B"])
    left = sum(min(n, case["budget"]) for n in lens)
    # every weight read; the kept keys' rows moved, their indices and weights written
    return {"bytes": hkv * (4 * sum(lens) + left * (8 * d + 8)), "flops": hkv * sum(lens)}


# ---------------------------------------------------------- 64-bit references


def _exact_rope(st: dict) -> dict:
    case = st["case"]
    d, rot = case["d"], case["rot"]
    half = rot // 2
    first = np.arange(half) * 2 if case["pairs"] else np.arange(half)
    first = torch.from_numpy(first).to(DEV)
    second = first + (1 if case["pairs"] else half)
    # a rotation by the position's angles in the planes (first, second), as one complex product
    turn = torch.complex(st["cos"].double()[st["pos"]], st["sin"].double()[st["pos"]])[:, None]

    def one(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = one(st["q"], st["qw"]), one(st["k"], st["kw"])
    if not case["append"]:
        return {"q": q, "k": k}
    kp, vp = st["kp"].double(), st["vp"].double()
    for pages, rows in ((kp, k), (vp, st["v"].double())):
        flat = pages.transpose(1, 2).reshape(-1, case["hkv"], d).clone()  # (slot, head, d)
        flat[st["slots"]] = rows
        pages.copy_(flat.view(-1, case["page"], case["hkv"], d).transpose(1, 2))
    return {"q": q, "k_pages": kp, "v_pages": vp}


def _exact_attn(st: dict) -> dict:
    case = st["case"]
    hq, hkv, d, page = (case[x] for x in ("hq", "hkv", "d", "page"))
    n_rows = st["q"].shape[0]
    o = torch.zeros((n_rows, hq, d), dtype=torch.float64, device=DEV)
    m = torch.zeros((sum(st["nq"]), hq), dtype=torch.float64, device=DEV)
    l = torch.zeros_like(m)
    w = st["w_out"].double() if case["weights"] else None
    row0 = 0
    for b in range(case["B"]):
        nq, n = st["nq"][b], st["lens_host"][b]
        j = torch.arange(n, device=DEV)
        slot = st["table"][b].long()[j // page] * page + j % page
        late = j[None, :] > (n - nq + torch.arange(nq, device=DEV))[:, None]
        for h in range(hq):
            kv = h // (hq // hkv)
            keys = st["kp"][:, kv].reshape(-1, d)[slot].double()
            vals = st["vp"][:, kv].reshape(-1, d)[slot].double()
            s = (st["q"][row0:row0 + nq, h].double() @ keys.T) / math.sqrt(d)
            s.masked_fill_(late, -math.inf)
            p = torch.softmax(s, -1)
            o[row0:row0 + nq, h] = p @ vals
            top = s.max(-1).values
            m[row0:row0 + nq, h] = top
            l[row0:row0 + nq, h] = torch.exp(torch.logsumexp(s, -1) - top)
            if w is not None:
                if h % (hq // hkv) == 0:
                    w[b, kv, :n] = torch.where(j < n - nq, st["w"][b, kv, :n].double(), 0.0)
                w[b, kv, :n] += p.sum(0)
        row0 += nq
    res = {"o": o}
    if w is not None:
        res["weights"] = w
    if case["ml"]:
        res["m"], res["l"] = m, l
    return res


def _exact_evict(st: dict) -> dict:
    case = st["case"]
    B, hkv, budget, page, d = (case[x] for x in ("B", "hkv", "budget", "page", "d"))
    kept = torch.full((B, hkv, budget), -1, dtype=torch.int32)
    w_in, w_out = st["w"].double().cpu().numpy(), st["w_out"].double()
    ko, vo = st["ko"].double(), st["vo"].double()
    for b, n in enumerate(st["lens_host"]):
        m = min(n, budget)
        for h in range(hkv):
            rank = w_in[b, h, :n].copy()
            rank[n - min(case["recent"], n):] = np.inf
            # numpy's lexsort: the last key first; the highest rank, then the lowest index
            idx = np.sort(np.lexsort((np.arange(n), -rank))[:m])
            kept[b, h, :m] = torch.from_numpy(idx.astype(np.int32))
            i = torch.from_numpy(idx).to(DEV)
            src = st["table"][b].long()[i // page] * page + i % page
            to = torch.arange(m, device=DEV)
            pg, off = st["out_table"][b].long()[to // page], to % page
            ko[pg, h, off] = st["kp"][:, h].reshape(-1, d)[src].double()
            vo[pg, h, off] = st["vp"][:, h].reshape(-1, d)[src].double()
            w_out[b, h, :m] = st["w"][b, h].double()[i]
    return {"kept": kept.to(DEV), "lens": _ints([min(n, budget) for n in st["lens_host"]]), "weights": w_out,
            "k_pages": ko, "v_pages": vo}


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "evict": _exact_evict}[case["kind"]](st)
