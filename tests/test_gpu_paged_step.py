"""Steps of a batch as a server runs them -- plan, rotary write, attention, rules on
the logits, pages given back -- against float64 on each request by itself, eager and
from a captured graph."""
import math

import pytest
import torch

from rocmforge_amd import paged

from . import paged_util as P

pytestmark = pytest.mark.gpu
NH, NKV, D, PAGE, ROT, BASE = 8, 2, 128, 16, 64, 1e6


class Server:
    """Up to `slots` requests in a pool of pages, steps of up to `rows` token rows."""

    def __init__(self, slots, pages, rows, width):
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=P.DEV)
        self.slots, self.rows, self.width, self.pages = slots, rows, width, pages
        self.kc, self.vc = P.cache_tensors(pages, PAGE, NKV, D)
        self.cache = P.cache_block(self.kc, self.vc)
        self.new, self.ctx, self.kv, self.q_start = z(slots), z(slots), z(slots), z(slots + 1)
        self.tab, self.pos, self.slot = z(slots, width), z(rows), z(rows)
        self.free = torch.randperm(pages, generator=P.gen(1), device=P.DEV).int()
        self.n_free = P.ints([pages])
        self.ended = z(slots)
        f = lambda n: torch.zeros(rows, n * D, device=P.DEV)
        self.q, self.k, self.v = f(NH), f(NKV), f(NKV)
        g = P.gen(2)
        self.qn, self.kn = [1 + 0.1 * torch.randn(D, generator=g, device=P.DEV) for _ in range(2)]
        self.q16 = torch.zeros(rows, NH * D, dtype=torch.float16, device=P.DEV)
        self.out = torch.zeros_like(self.q16)
        self.turns = torch.zeros(ROT // 2, dtype=torch.float64, device=P.DEV)
        paged.rope_turns_table(self.turns, ROT, BASE, paged.ROPE_YARN, 4.0, 4096.0)
        self.factor = 0.1 * math.log(4.0) + 1
        self.ws = torch.zeros((paged.attention_workspace_bytes(NH, NKV, D) + 3) // 4, device=P.DEV)
        self.p = paged.PagedPlan(new_lens=self.new, ctx_in=self.ctx, ctx_out=self.ctx, free_pages=self.free,
                                 free_in=self.n_free, free_out=self.n_free, block_tables=self.tab,
                                 q_start=self.q_start, kv_lens=self.kv, positions=self.pos, slots=self.slot,
                                 num_seqs=slots, max_blocks=width, page_size=PAGE, max_rows=rows, num_pages=pages)
        self.r = paged.PagedRope(q=self.q, k=self.k, v=self.v, q_norm=self.qn, k_norm=self.kn, q16=self.q16,
                                 positions=self.pos, slots=self.slot, turns=self.turns, ld_q=NH * D, ld_k=NKV * D,
                                 ld_v=NKV * D, ld_q16=NH * D, rows=rows, num_heads=NH, rot_dim=ROT, neox=1, eps=1e-6,
                                 attn_factor=self.factor)
        self.a = paged.PagedAttention(q=self.q16, out=self.out, block_tables=self.tab, q_start=self.q_start,
                                      kv_lens=self.kv, workspace=self.ws, workspace_bytes=4 * self.ws.numel(),
                                      ld_q=NH * D, ld_out=NH * D, num_seqs=slots, max_blocks=width, rows=rows,
                                      num_heads=NH, max_new=rows, window=0, out_f32=0, scale=1 / math.sqrt(D))
        self.seen = [[] for _ in range(slots)]          # (k, v) rows of every token a request was granted

    def step(self, stream=None):
        paged.plan(self.p, stream)
        paged.rope_write(self.r, self.cache, stream)
        paged.attention(self.a, self.cache, stream)

    def release(self, which):
        self.ended.zero_()
        self.ended[which] = 1
        paged.release(self.ended, self.ctx, self.tab, self.free, self.n_free, self.slots, self.width, PAGE, self.pages)
        for b in which:
            self.seen[b] = []

    def fill(self, new, seed):
        g = P.gen(seed)
        for t in (self.q, self.k, self.v):
            t.normal_(generator=g)
        self.new.copy_(P.ints(new))

    def rotated(self, x, norm, pos):
        """float64, one row a position"""
        x = x.double().reshape(len(pos), -1, D)
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.double()
        ang = 2 * math.pi * pos.double()[:, None] * self.turns
        c, s = [(f * self.factor)[:, None] for f in (ang.cos(), ang.sin())]
        h = ROT // 2
        a, b = x[..., :h], x[..., h:ROT]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., ROT:]], -1)

    def check(self, new, granted):
        torch.cuda.synchronize()
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            got = self.out[at:at + n].double().reshape(n, NH, D)
            if not granted[b]:
                assert bool((got == 0).all())
                at += n
                continue
            first = len(self.seen[b])
            pos = torch.arange(first, first + n, device=P.DEV)
            q = self.rotated(self.q[at:at + n], self.qn, pos).half().double()
            k = self.rotated(self.k[at:at + n], self.kn, pos).half().double()
            v = self.v[at:at + n].half().double().reshape(n, NKV, D)
            self.seen[b] += list(zip(k, v))
            ks, vs = [torch.stack(t) for t in zip(*self.seen[b])]
            hidden = torch.arange(first + n, device=P.DEV) > pos[:, None]
            for h in range(NH):
                s = (q[:, h] @ ks[:, h // 4].t().contiguous()) / math.sqrt(D)
                w = s.masked_fill(hidden, -math.inf).softmax(-1)
                want, mag = w @ vs[:, h // 4], w @ vs[:, h // 4].abs()
                # q and k are off by a rounding to fp16 here or there, so scores of |q||k| / sqrt(D) ~ 13
                # by 2^-10 of that at most (both, aligned) and weights by 2^-6; weights and output by 2^-11
                assert bool(((got[:, h] - want).abs() <= (2.0 ** -6 + 2 * P.U16) * mag + P.U16 * want.abs()).all())
            at += n
        assert self.ctx.tolist() == [len(s) for s in self.seen]


SCRIPT = [            # new tokens of each request, and who ends after the step
    ([37, 1, 0, 120, 5], []),
    ([1, 1, 64, 1, 1], [1]),
    ([1, 200, 1, 1, 16], []),
    ([1, 1, 1, 1, 1], [0, 3]),
    ([90, 0, 1, 33, 1], []),
    ([1, 1, 1, 1, 1], []),
]


def test_steps_of_a_batch(rf, dev):
    s = Server(5, 64, 264, 20)
    for i, (new, ended) in enumerate(SCRIPT):
        print(f"[gpu] step {i}: {new}", flush=True)
        s.fill(new, 10 + i)
        s.step()
        s.check(new, [True] * 5)
        if ended:
            s.release(ended)
    # everyone out: every page is back, once
    s.release(range(5))
    torch.cuda.synchronize()
    assert s.n_free.tolist() == [64] and sorted(s.free.tolist()) == list(range(64))


def test_a_step_without_enough_pages(rf, dev):
    s = Server(4, 8, 128, 8)
    s.fill([40, 50, 20, 0], 3)                   # 3 + 4 pages, then 2 of the 1 left
    s.step()
    s.check([40, 50, 20, 0], [True, True, False, False])
    assert s.n_free.tolist() == [1]
    s.release([0])
    s.fill([0, 1, 20, 3], 4)
    s.step()
    s.check([0, 1, 20, 3], [True, True, True, True])


def test_captured_steps(rf, dev):
    s = Server(5, 64, 264, 20)
    side = torch.cuda.Stream()
    s.fill([0] * 5, 1)
    s.step()                                     # (warm: kernels loaded before the capture)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        s.step()
    for i, (new, ended) in enumerate(SCRIPT):
        s.fill(new, 30 + i)
        torch.cuda.synchronize()
        g.replay()
        s.check(new, [True] * 5)
        if ended:
            s.release(ended)                     # eager work between the replays


def test_picking_tokens_of_a_batch(rf, dev):
    """Rules on the logits, then the framework's argmax a row."""
    from . import gpu_util as G
    rows, vocab = 3, 5000
    x = torch.randn(rows, vocab, generator=P.gen(5), device=P.DEV)
    x[:, 77] = 50.0                              # everyone's favourite, already said twice ...
    x[:, 99] = 49.5
    hist = P.ints([[77, 77, 5], [77, 6, 7], [1, 2, 3]])
    out = torch.empty_like(x)
    f = lambda v: torch.full((rows,), v, device=P.DEV)
    allowed = torch.full((rows, 157), -1, dtype=torch.int32, device=P.DEV)
    allowed[2, 77 // 32] &= ~(1 << (77 % 32))    # ... or against the third one's grammar
    paged.logits_rules(paged.LogitsRules(
        logits=x, out=out, ld_logits=vocab, ld_out=vocab, history=hist, ld_history=3, prompt_lens=P.ints([0, 1, 0]),
        total_lens=P.ints([3, 3, 3]), repetition=f(1.0), frequency=f(0.4), presence=f(0.0), allowed=allowed,
        ld_allowed=157, rows=rows, vocab=vocab))
    pv, pi, best = torch.empty(8, device=P.DEV), G.empty(8, torch.int32), G.empty(1, torch.int32)
    got = []
    for r in range(rows):
        G.call(rf.gpu_argmax_f32_on_stream, G.ptr(out[r]), G.ptr(pv), G.ptr(pi), G.ptr(best), vocab)
        got.append(best.item())
    assert got == [99, 77, 99]
