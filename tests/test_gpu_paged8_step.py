"""Steps of a batch on 8-bit pages as a server runs them -- plan, rotary write, attention,
the requests' adapters beside the output projection, requests taken out and pages given
back -- each against float64 on what the one before left, eager and captured."""
import math

import pytest
import torch

from rocmforge_amd import lora, paged

from . import paged8_util as E
from . import paged_util as P
from .test_gpu_paged_step import D, NH, NKV, PAGE, ROT, SCRIPT, Server

pytestmark = pytest.mark.gpu
RANK, OUT = 16, 256
OF, RANKS, SCALES = [0, -1, 2, 1, 2], [16, 4, 9], [0.5, 2.0, 1.0]


class Server8(Server):
    def __init__(self, slots, pages, rows, width):
        super().__init__(slots, pages, rows, width)
        self.p8 = E.Pages(pages, PAGE, NKV, D)
        self.cache = self.p8.cache()
        g = P.gen(9)
        r = lambda *s: torch.randn(*s, generator=g, device=P.DEV)
        self.la = (r(3, RANK, NH * D) / math.sqrt(NH * D)).half()
        self.lb, self.base = r(3, OUT, RANK).half(), r(rows, OUT)
        self.y = torch.zeros(rows, OUT, device=P.DEV)
        self.target = lora.LoraTarget(a=self.la, b=self.lb, base=self.base, y=self.y, a_stride=RANK * NH * D,
                                      b_stride=OUT * RANK, ld_base=OUT, ld_y=OUT, out_dim=OUT)
        self.adapters = lora.LoraStep(x=self.out, adapters=P.ints(OF), q_start=self.q_start, ranks=P.ints(RANKS),
                                      scales=torch.tensor(SCALES, device=P.DEV), ld_x=NH * D, rows=rows, num_seqs=slots,
                                      num_adapters=3, max_rank=RANK, in_dim=NH * D, x_f16=1)
        self.count = [0] * slots

    def step(self, stream=None):
        paged.plan(self.p, stream)
        paged.rope_write8(self.r, self.cache, stream)
        paged.attention8(self.a, self.cache, stream)
        lora.add(self.adapters, self.target, stream)

    def release(self, which):
        super().release(which)
        for b in which:
            self.count[b] = 0

    def check(self, new):
        torch.cuda.synchronize()
        k8, v8 = self.p8.values()
        kv = [c + n for c, n in zip(self.count, new)]
        assert self.kv.tolist() == kv and self.ctx.tolist() == kv
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            rows = slice(at, at + n)
            t = torch.arange(self.count[b], kv[b], device=P.DEV)
            pg, row = self.tab[b].long()[t // PAGE], t % PAGE
            want = (self.rotated(self.k[rows], self.kn, t), self.v[rows].double().reshape(n, NKV, D))
            for x, s, w in ((k8, self.p8.ks, want[0]), (v8, self.p8.vs, want[1])):
                # half a step of e4m3: 2^-4, or 2^-10 2^e where it is subnormal; and once more the latter where
                # a block's exponent grew after the row was written (rows of one step: it did not); fp32 before
                by = torch.exp2(s[pg, row // 16].double() - 127)[..., None]
                assert bool(((x[pg, row] - w).abs() <= torch.maximum(2.0 ** -4 * w.abs(), 2.0 ** -10 * by) + 2.0 ** -18).all())
            at += n
        q = self.q16[:at].reshape(at, NH, D)
        out, bound = P.attention64(q, k8, v8, self.tab, new, kv, 0, 1 / math.sqrt(D))
        got = self.out[:at].reshape(at, NH, D).double()
        assert bool(((got - out).abs() <= bound).all())
        at = 0
        for b, n in enumerate(new):
            x, y = self.out[at:at + n].double(), self.base[at:at + n].double()
            if OF[b] >= 0:
                i, r = OF[b], RANKS[OF[b]]
                y = y + SCALES[i] * ((x @ self.la[i, :r].double().t().contiguous()) @ self.lb[i, :, :r].double().t().contiguous())
            # sums of 1024 and 16 products in fp32
            assert bool(((self.y[at:at + n].double() - y).abs() <= 2.0 ** -17 * (1 + y.abs())).all())
            at += n
        self.count = kv

    def taken_out(self, which):
        """Requests' K and V, as a server sets them aside."""
        lens = [self.count[b] for b in which]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        k, v = [torch.zeros(starts[-1], NKV * D, dtype=torch.float16, device=P.DEV) for _ in range(2)]
        tab = self.tab[which].contiguous()
        paged.read8(paged.PagedRead(k=k, v=v, block_tables=tab, row_start=P.ints(starts), ld_out=NKV * D,
                                    num_seqs=len(which), max_blocks=self.width, rows=starts[-1]), self.cache)
        torch.cuda.synchronize()
        for got, x in ((k, self.p8.values()[0]), (v, self.p8.values()[1])):
            for i, b in enumerate(which):
                t = torch.arange(lens[i], device=P.DEV)
                want = x[tab[i].long()[t // PAGE], t % PAGE].flatten(1)
                assert torch.equal(got[starts[i]:starts[i + 1]].double(), want)


def test_steps_of_a_batch(rf, dev):
    s = Server8(5, 64, 264, 20)
    for i, (new, ended) in enumerate(SCRIPT):
        print(f"[gpu] step {i}: {new}", flush=True)
        s.fill(new, 10 + i)
        s.step()
        s.check(new)
        s.taken_out([0, 2, 4])
        if ended:
            s.release(ended)
    s.release(range(5))
    torch.cuda.synchronize()
    assert s.n_free.tolist() == [64] and sorted(s.free.tolist()) == list(range(64))


def test_captured_steps(rf, dev):
    s = Server8(5, 64, 264, 20)
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
        s.check(new)
        s.taken_out([1, 3])                      # eager work between the replays
        if ended:
            s.release(ended)


def test_a_refused_request(rf, dev):
    # rows of a refused request are not written, and its attention is zero
    s = Server8(5, 8, 264, 8)
    s.fill([40, 50, 20, 0, 0], 3)                # 3 + 4 pages, then 2 of the 1 left
    before = s.p8.k.clone()
    s.step()
    torch.cuda.synchronize()
    assert s.kv.tolist()[:3] == [40, 50, 0]
    assert bool((s.out[90:110] == 0).all()) and bool((s.out[:90] != 0).any(1).all())
    left = [p for p in range(8) if p not in set(s.tab[0, :3].tolist() + s.tab[1, :4].tolist())]
    assert torch.equal(s.p8.k[left], before[left])
    assert torch.equal(s.y[90:110], s.base[90:110])      # (an adapter of zeros adds nothing)
