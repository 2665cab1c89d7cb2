"""A server's step through its operators together: tables and slots from the requests' lengths, norm and rotation into the
cache, attention over a shared prefix and the requests' own keys, the next tokens, finished requests' pages given back."""

from __future__ import annotations

import pytest
import torch

from catopt_amd import paged as P
from catopt_amd import sampling as S
from paged_ref import BF16, DEV, attention, gen, ints, randn, rope
from test_sampling_gpu import row_ref

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE, VOCAB, HIDDEN, MAX_POS = 8, 2, 64, 16, 500, 96, 512
SCALE = D ** -0.5


class Server:
    """One layer between an embedding and the logits, a pool of pages, a prefix in the cache that every request shares."""

    def __init__(self, B, prefix, n_pages, width, seed):
        g = gen(seed)
        self.B, self.prefix = B, prefix
        self.embed, self.w_qkv = randn(g, VOCAB, HIDDEN), randn(g, HIDDEN, (HQ + 2 * HKV) * D, scale=HIDDEN ** -0.5)
        self.w_out = randn(g, HQ * D, VOCAB, scale=0.2)
        self.q_norm, self.k_norm = randn(g, D) * 0.1 + 1, randn(g, D) * 0.1 + 1
        ang = torch.arange(MAX_POS, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.k, self.v = (torch.full((n_pages, HKV, PAGE, D), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
        self.lens, self.pre_lens, self.pre_starts = ints([0] * B), ints([prefix]), ints([0, B])
        order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        self.free, self.count = order.contiguous(), ints([n_pages])
        self.offsets = ints([prefix] * B)
        # the prefix enters the cache as a request of its own
        self.pre_table = torch.full((1, -(-prefix // PAGE)), -1, dtype=torch.int32, device=DEV)
        step = P.paged_extend(self.pre_table, ints([0]), ints([prefix]), self.free, self.count, prefix, PAGE)
        self.count.copy_(step.free_count)
        tokens = torch.randint(0, VOCAB, (prefix,), generator=g, device=DEV)
        self.append(tokens, step)

    def append(self, tokens, step):
        qkv = (self.embed[tokens] @ self.w_qkv)
        self.last = tuple(t.unflatten(1, (-1, D)) for t in qkv.split([HQ * D, HKV * D, HKV * D], 1))
        q, k, v = self.last
        return P.qk_norm_rope_append(q, k, v, self.cos, self.sin, step.positions, self.k, self.v, step.slots, self.q_norm,
                                     self.k_norm)

    def step(self, tokens, new, u, settings):
        """tokens: the step's rows, padded; the logits of each request's last row and the tokens drawn from them."""
        step = P.paged_extend(self.table, self.lens, new, self.free, self.count, tokens.shape[0], PAGE, offsets=self.offsets,
                              kv_lens_out=self.lens, free_count_out=self.count)
        q = self.append(tokens, step)
        o = P.paged_prefix_attention(q, self.k, self.v, self.pre_table, self.pre_lens, self.pre_starts, self.table, self.lens,
                                     step.q_starts, SCALE, empty_rows="zero", out=torch.zeros_like(q))
        last = o[(step.q_starts[1:].long() - 1).clamp(min=0)]
        logits = last.flatten(1) @ self.w_out
        return step, q, o, logits, S.sample(logits, u, *settings)

    def release(self, done):
        P.paged_release(self.table, self.lens, done, self.free, self.count, PAGE, kv_lens_out=self.lens,
                        free_count_out=self.count)


def test_requests_come_and_go():
    """Eager steps, each operator's outcome against its definition on that step's inputs; pages are never in use twice."""
    B, prefix = 6, 45
    s = Server(B, prefix, n_pages=40, width=8, seed=1)
    g = gen(2)
    settings = (0.8, 40, 0.95, 0.01)
    keys = [[] for _ in range(B)]  # the dense caches
    pre_q, pre_k, pre_v = s.last
    pre_pos = torch.arange(prefix, device=DEV)
    k_pre = rope(pre_k, s.k_norm, s.cos, s.sin, pre_pos, False)
    new = [7, 1, 30, 2, 16, 17]
    tokens = [torch.randint(0, VOCAB, (n,), generator=g, device=DEV) for n in new]
    for step_no in range(14):
        pad = step_no % 3
        rows = torch.cat(tokens + [torch.zeros((pad,), dtype=torch.int64, device=DEV)])
        u = torch.rand((B,), generator=g, device=DEV)
        lens_before = s.lens.tolist()
        step, q, o, logits, (drawn, logp) = s.step(rows, ints([len(t) for t in tokens]), u, settings)
        q_in, k_in, v_in = s.last
        assert s.lens.tolist() == [a + len(t) for a, t in zip(lens_before, tokens)]
        starts = step.q_starts.tolist()
        used = [x for b in range(B) for x in s.table[b, :-(-s.lens[b].item() // PAGE)].tolist()] + s.pre_table[0].tolist()
        left = s.free[:s.count.item()].tolist()
        assert sorted(used + left) == list(range(40))
        zq, eq = rope(q_in, s.q_norm, s.cos, s.sin, step.positions, False)
        zk, ek = rope(k_in, s.k_norm, s.cos, s.sin, step.positions, False)
        assert ((q.double() - zq).abs() <= eq).all()
        for b in range(B):
            r = slice(starts[b], starts[b + 1])
            n, length = starts[b + 1] - starts[b], s.lens[b].item()
            if n == 0:
                continue
            assert step.positions[r].tolist() == list(range(prefix + lens_before[b], prefix + lens_before[b] + n))
            # the cache's rows are the rotated keys (one rounding) and the values as they are
            j = torch.arange(length, device=DEV)
            kc, vc = (t[s.table[b].long()[j // PAGE], :, j % PAGE].transpose(0, 1) for t in (s.k, s.v))
            assert ((kc[:, -n:].double().transpose(0, 1) - zk[r]).abs() <= ek[r]).all() and torch.equal(vc[:, -n:], v_in[r].transpose(0, 1))
            if keys[b]:
                assert torch.equal(kc[:, :-n], keys[b][0]) and torch.equal(vc[:, :-n], keys[b][1])
            keys[b] = [kc.clone(), vc.clone()]
            i = torch.arange(prefix, device=DEV)
            kp, vp = (t[s.pre_table[0].long()[i // PAGE], :, i % PAGE].transpose(0, 1) for t in (s.k, s.v))
            assert ((kp.double().transpose(0, 1) - k_pre[0]).abs() <= k_pre[1]).all() and torch.equal(vp, pre_v.transpose(0, 1))
            ref = attention(q[r], torch.cat([kp, kc], 1).double(), torch.cat([vp, vc], 1).double(), SCALE)
            es = torch.expm1(2 * ref["es"]) + (prefix + length + 64) * 2.0 ** -24
            tol = (2.0 ** -8 + es)[..., None] * ref["mag"] * 1.01 + 2.0 ** -8 * ref["o"].abs() + 1e-37
            assert ((o[r].double().transpose(0, 1) - ref["o"]).abs() <= tol).all()
            token, log, _, near, off = row_ref(logits[b].double().cpu().numpy(), u[b].double().item(), *settings)
            assert near > off and drawn[b].item() == token and abs(logp[b].item() - log) <= 2.0 ** -24 * abs(log) + off
        assert (o[starts[-1]:] == 0).all()
        # some end and give their pages back, others begin in their place
        done = torch.rand((B,), generator=g, device=DEV) < 0.25
        s.release(done)
        tokens = []
        for b, out in enumerate(done.tolist()):
            if out:
                keys[b] = []
                tokens.append(torch.randint(0, VOCAB, (int(torch.randint(0, 20, (1,), generator=g, device=DEV)),), generator=g, device=DEV))
            else:
                tokens.append(drawn[b:b + 1] if starts[b + 1] > starts[b] else drawn[:0])


def test_a_captured_generation_step_is_the_eager_one():
    """One graph replayed for every token of a generation: lengths, pages and tokens are its own state."""
    B, prefix, n = 5, 70, 40
    servers = [Server(B, prefix, n_pages=60, width=8, seed=3) for _ in range(2)]
    settings = (1.0, 0, 0.9, 0.0)
    u = torch.rand((n, B), generator=gen(4), device=DEV)
    first = torch.randint(0, VOCAB, (B,), generator=gen(5), device=DEV)
    ones = torch.ones((B,), dtype=torch.int32, device=DEV)
    history = []
    tokens = first
    for i in range(n):
        out = servers[0].step(tokens, ones, u[i], settings)
        tokens = out[4][0]
        history.append((tokens, out[3], out[4][1]))
    s = servers[1]
    tokens, numbers, new = first.clone(), u[0].clone(), torch.zeros_like(ones)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step(tokens, new, numbers, settings)  # no new tokens: nothing changes
    torch.cuda.current_stream().wait_stream(side)
    new.copy_(ones)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, _, _, logits, (drawn, logp) = s.step(tokens, new, numbers, settings)
        tokens.copy_(drawn)
    for i in range(n):
        numbers.copy_(u[i])
        graph.replay()
        assert torch.equal(tokens, history[i][0]) and torch.equal(logits, history[i][1]) and torch.equal(logp, history[i][2]), i
    assert s.lens.tolist() == [n] * B and torch.equal(s.table, servers[0].table) and s.count.item() == servers[0].count.item()
