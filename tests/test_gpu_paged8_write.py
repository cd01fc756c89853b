"""The rotary step into 8-bit pages (rf_paged_rope_write8_launch) against float64:
codes and exponents where values are as given, bounds where they are turned, old rows of
a block under a grown exponent, and what has to stay as it was."""
import math

import pytest
import torch

from rocmforge_amd import paged

from . import paged8_util as E
from . import paged_util as P
from .test_gpu_paged_rope import turns64

pytestmark = pytest.mark.gpu


class Step:
    """Rows at slots; positions in front of them hold codes under exponents of their own."""

    def __init__(self, slots, nh=4, nkv=2, d=128, rot=0, neox=1, norm=False, page=16, pages=8, by_head=False, extra=0,
                 wide=0, seed=0, size=1.0, old=1.0):
        g = P.gen(seed + 31 * len(slots) + d)
        rows = len(slots)
        mk = lambda n, by: by * torch.randn(rows, n * d + wide, generator=g, device=P.DEV)[:, :n * d]
        self.q, self.k, self.v = mk(nh, 1.0), mk(nkv, size), mk(nkv, size)
        w = lambda: 1 + 0.2 * torch.randn(d, generator=g, device=P.DEV) if norm else None
        self.qn, self.kn = w(), w()
        self.p = E.Pages(pages, page, nkv, d, by_head, extra)
        self.p.hold(*[old * torch.randn(pages, page, nkv, d, generator=g, device=P.DEV) for _ in range(2)])
        self.q16 = torch.full((rows, nh * d + 8), 9.0, dtype=torch.float16, device=P.DEV)
        self.turns = turns64(rot, 1e6) if rot else torch.zeros(1, dtype=torch.float64, device=P.DEV)
        self.slots = list(slots)
        self.pos, self.slot = P.ints([(17 * i) % 5000 for i in range(rows)]), P.ints(slots)
        self.dims = (rows, nh, nkv, d, rot, neox, page)
        self.args = paged.PagedRope(q=self.q, k=self.k, v=self.v, q_norm=self.qn, k_norm=self.kn, q16=self.q16,
                                    positions=self.pos, slots=self.slot, turns=self.turns, ld_q=self.q.stride(0),
                                    ld_k=self.k.stride(0), ld_v=self.v.stride(0), ld_q16=self.q16.stride(0), rows=rows,
                                    num_heads=nh, rot_dim=rot, neox=neox, eps=1e-6, attn_factor=1.0)

    def run(self):
        print(f"[gpu] rope write8 {self.dims}", flush=True)
        paged.rope_write8(self.args, self.p.cache())
        torch.cuda.synchronize()

    def turned(self, x, w):
        rows, nh, nkv, d, rot, neox, page = self.dims
        x = x.double().reshape(rows, -1, d)
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        y, size = x.clone(), x.abs()
        if rot:
            ang = 2 * math.pi * (self.pos.double()[:, None] * self.turns)[:, None, :]
            i = torch.arange(rot // 2, device=P.DEV)
            i0, i1 = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
            y[..., i0], y[..., i1] = (x[..., i0] * ang.cos() - x[..., i1] * ang.sin(),
                                      x[..., i0] * ang.sin() + x[..., i1] * ang.cos())
            size[..., i0] = size[..., i1] = x[..., i0].abs() + x[..., i1].abs()
        return y, size

    def check(self):
        rows, nh, nkv, d, rot, neox, page = self.dims
        p = self.p
        total, blk = p.k.shape[0] * page, p.block
        exact = rot == 0 and self.kn is None
        before = [(c.clone(), s.clone()) for c, s in ((p.k, p.ks), (p.v, p.vs))]
        self.run()
        live = [i for i, s in enumerate(self.slots) if 0 <= s < total]
        # q: as the step into fp16 pages has it (a few fp32 roundings of the pair, one to fp16)
        want, size = self.turned(self.q, self.qn)
        got = self.q16[live][:, :nh * d].reshape(-1, nh, d).double()
        assert bool(((got - want[live]).abs() <= P.U16 * want[live].abs() + 2.0 ** -25 + 11 * 2.0 ** -23 * size[live]).all())
        dead = [i for i in range(rows) if i not in set(live)]
        assert bool((self.q16[dead] == 9.0).all()) and bool((self.q16[:, nh * d:] == 9.0).all())
        for name, x, w, (codes0, scale0) in (("k", self.k, self.kn, before[0]), ("v", self.v, None, before[1])):
            codes, scale = (p.k, p.ks) if name == "k" else (p.v, p.vs)
            y, size = self.turned(x, w) if name == "k" else (x.double().reshape(rows, nkv, d), x.abs().double().reshape(rows, nkv, d))
            off = torch.zeros_like(size) if exact or name == "v" else 11 * 2.0 ** -23 * size
            flat, flat0 = scale.view(-1, nkv), scale0.view(-1, nkv)
            touched = {}
            for i in live:
                touched.setdefault(self.slots[i] // blk, []).append(i)
            stay = torch.ones(codes.shape[:2], dtype=torch.bool, device=P.DEV)
            for b, rs in touched.items():
                fine = torch.where(y[rs].isfinite(), y[rs].abs(), 0.0)
                low = E.exponent((fine - off[rs]).clamp(min=0).amax((0, 2)))
                high = E.exponent((fine + off[rs]).amax((0, 2)))
                old = flat0[b].long().clamp(112, 134) - 127
                first = min(self.slots[i] % blk for i in rs)
                if first > 0:
                    low, high = torch.maximum(low, old), torch.maximum(high, old)
                e = flat[b].long() - 127
                assert bool(((low <= e) & (e <= high)).all()), (name, b, low, e, high)
                by = torch.exp2(e.double())[:, None]
                for i in rs:
                    at = self.slots[i] // page, self.slots[i] % page
                    stay[at] = False
                    got = codes[at]
                    if exact or name == "v":
                        assert torch.equal(got & 127, E.nearest(y[i] / by) & 127), (name, i)
                        keep = (got & 127 != 0) & (got & 127 != E.NAN)
                        assert torch.equal(got[keep] >= 128, y[i][keep] < 0)
                    else:
                        # half a step of e4m3 (2^-4, or 2^-10 in its subnormal range), and what the value is off
                        v = E.values(got[None, None], torch.zeros(1, 1, nkv, device=P.DEV) + e + 127, 1)[0, 0]
                        bound = torch.maximum(2.0 ** -4 * y[i].abs(), 2.0 ** -10 * by) + 1.125 * off[i]
                        assert bool(((v - y[i]).abs() <= bound).all()), (name, i)
                for r in range(first):
                    at = (b * blk + r) // page, (b * blk + r) % page
                    stay[at] = False
                    was = E.values(codes0[at][None, None], torch.zeros(1, 1, nkv, device=P.DEV) + old + 127, 1)[0, 0]
                    grown = torch.where((e > old)[:, None], E.nearest(was / by), codes0[at])
                    assert torch.equal(codes[at] & 127, grown & 127), (name, b, r)
            assert torch.equal(codes[stay], codes0[stay])
            rest = [b for b in range(flat.shape[0]) if b not in touched]
            assert torch.equal(flat[rest], flat0[rest])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("slots", [[0], [5], [15], list(range(16)), list(range(3, 40)), [17, 18, 64, 65, 66, 33],
                                   list(range(48, 64)) + [1, 20, 100], [-1, 7, 8, 9, -1, 1 << 30, 40]])
def test_values_as_given(rf, dev, slots, page, d):
    Step(slots, d=d, page=page, pages=128 // page).check()


@pytest.mark.parametrize("size,old", [(100.0, 0.01), (0.01, 100.0), (1e-6, 1e-6), (30000.0, 1.0), (3e5, 1.0), (1e-30, 1.0)])
@pytest.mark.parametrize("slots", [[5], [3, 4, 5, 6], list(range(6, 30)), [2, 33, 77, 120]])
def test_exponents_that_grow_and_stay(rf, dev, slots, size, old):
    Step(slots, size=size, old=old).check()
    Step(slots, size=size, old=old, page=8, pages=16, d=64).check()


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (128, 128), (128, 96), (128, 8), (256, 256), (256, 64)])
@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("norm", [False, True])
def test_turned(rf, dev, d, rot, neox, norm):
    Step(list(range(2, 50)) + [70, 100], d=d, rot=rot, neox=neox, norm=norm, page=32, pages=4).check()


@pytest.mark.parametrize("nh,nkv", [(1, 1), (5, 1), (28, 4), (33, 3)])
@pytest.mark.parametrize("by_head", [False, True])
def test_heads_orders_and_strides(rf, dev, nh, nkv, by_head):
    Step(list(range(5, 45)), nh, nkv, rot=64, by_head=by_head, extra=16, wide=8).check()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 200])
@pytest.mark.parametrize("start", [0, 1, 9, 15])
@pytest.mark.parametrize("d", [64, 256])
def test_runs_over_the_workgroups(rf, dev, rows, start, d):
    # rows of one request: its blocks lie across the groups of 16 rows
    Step(list(range(start, start + rows)), d=d, pages=16).check()


@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_single_tokens(rf, dev, rows):
    # every row in a block of its own, at every place of one
    Step([16 * ((7 * i) % rows) + i % 16 for i in range(rows)], pages=rows, old=0.05).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("singles", [1, 14, 15, 16, 30, 31, 32])
def test_long_runs_behind_single_tokens(rf, dev, singles, d):
    # more rows start in a group than its threads take at once
    slots = [16 * (4 + i) + i % 16 for i in range(singles)] + list(range(32)) + [35, 37, 39]
    Step(slots, d=d, pages=40, old=0.05).check()
    Step(slots, d=d, pages=80, page=8, rot=d, norm=True).check()


def test_heads_of_all_kinds_in_a_workgroup(rf, dev):
    Step(list(range(7, 1507)), 33, 8, rot=128, norm=True, pages=100).check()


def test_many_rows(rf, dev):
    # heads shared among few workgroups a row
    s = Step(list(range(7, 3007)), 8, 2, 64, pages=200)
    s.check()


def test_ties_and_borders(rf, dev):
    """Every code's value, every middle of two and its neighbours, under every exponent."""
    t = torch.tensor(E.table(), dtype=torch.float64)
    mid = (t[1:] + t[:-1]) / 2
    near = [torch.nextafter(mid.float(), torch.tensor(v)).double() for v in (0.0, 1000.0)]
    x = torch.cat([t, mid, *near])
    x = torch.cat([x, -x])
    for e in range(E.E_LO, E.E_HI + 1):
        rows = -(-x.numel() // (2 * 127))
        s = Step([16 * i for i in range(rows)], d=128, nkv=2, pages=rows)
        val = torch.zeros(rows, 2, 128, dtype=torch.float64)
        flat = torch.zeros(rows * 2 * 127, dtype=torch.float64)
        flat[:x.numel()] = x
        val[..., 1:] = flat.view(rows, 2, 127)
        val[..., 0] = 448.0
        s.v.copy_((val * 2.0 ** e).float().view(rows, 256).to(P.DEV))
        s.check()
        assert bool((s.p.vs[:rows, 0] == e + 127).all())


@pytest.mark.parametrize("top,e", [(448.0, 0), (448.0 * (1 + 2.0 ** -23), 1), (447.9, 0), (224.0, -1), (224.1, 0), (0.0, -15),
                                   (1e-45, -15), (2.0 ** -15 * 448, -15), (2.0 ** -14 * 449, -13), (448.0 * 128, 7), (3e38, 7)])
def test_the_exponent_of_a_block(rf, dev, top, e):
    s = Step([0], size=0.0)
    s.v.zero_()
    s.v[0, 5] = -top
    s.v[0, 128 + 77] = top
    s.check()
    assert s.p.vs[0, 0].tolist() == [e + 127] * 2


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("slots", [[4], list(range(20))])
def test_what_is_not_finite(rf, dev, bad, slots):
    # it is stored as NaN, and does not enter the exponent
    s = Step(slots)
    s.v[0, 3] = bad
    s.v[0, 200] = bad
    s.k[0, 64] = bad
    s.check()
    assert s.p.v[slots[0] // 16, slots[0] % 16, 0, 3].item() & 127 == E.NAN


@pytest.mark.parametrize("byte", [0, 100, 111, 135, 255])
def test_exponents_outside_the_range(rf, dev, byte):
    s = Step([5, 30])
    s.p.ks.fill_(byte)
    s.p.vs.fill_(byte)
    s.check()


def test_nan_among_old_rows(rf, dev):
    s = Step([9], size=100.0)
    s.p.v[0, 4, 0, 7] = 0xff
    s.check()
    assert s.p.v[0, 4, 0, 7].item() & 127 == E.NAN


def test_a_second_run_changes_nothing(rf, dev):
    s = Step(list(range(5, 40)), rot=64, norm=True, old=0.1)
    s.run()
    kept = [t.clone() for t in (s.p.k, s.p.v, s.p.ks, s.p.vs, s.q16)]
    s.run()
    assert all(torch.equal(a, b) for a, b in zip(kept, (s.p.k, s.p.v, s.p.ks, s.p.vs, s.q16)))


def test_token_by_token_and_at_once(rf, dev):
    """A block written row by row stands for what it stands for when it is written at once, but for what a grown
    exponent rounded twice: codes that became subnormal."""
    one, all_ = Step(list(range(16)), seed=5), Step(list(range(16)), seed=5)
    all_.run()
    for i in range(16):
        one.slot.fill_(-1)
        one.slot[i] = i
        one.run()
    assert torch.equal(one.p.ks[0], all_.p.ks[0]) and torch.equal(one.p.vs[0], all_.p.vs[0])
    for a, b, s in ((one.p.k, all_.p.k, all_.p.ks), (one.p.v, all_.p.v, all_.p.vs)):
        normal = (b[0] & 127) >= 16
        assert torch.equal(a[0][normal], b[0][normal])
        x, y = [E.values(t[:1], s[:1], 16)[0] for t in (a, b)]
        step = 2.0 ** -9 * torch.exp2(s[0, 0].double() - 127)[:, None]
        assert bool(((x - y).abs() <= step).all())


def test_far_into_a_large_cache(rf, dev):
    # offsets beyond 32 bits
    page, nkv, d = 16, 2, 128
    pages = 5 * (1 << 30) // (page * nkv * d)
    k, v = [torch.empty(pages, page, nkv, d, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    ks, vs = [torch.empty(pages, 1, nkv, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    s = Step(list(range(3, 60)), rot=64, pages=4)
    far = pages - 4
    for a, b in ((k, s.p.k), (v, s.p.v), (ks, s.p.ks), (vs, s.p.vs)):
        a[far:] = b
    s.run()
    want = [t.clone() for t in (s.p.k, s.p.v, s.p.ks, s.p.vs)]
    s.slot += far * page
    s.p.k, s.p.v, s.p.ks, s.p.vs = k, v, ks, vs
    s.run()
    assert all(torch.equal(a[far:], b) for a, b in zip((k, v, ks, vs), want))


def test_replays(rf, dev):
    s = Step(list(range(5, 40)), rot=64, old=0.1)
    cache = s.p.cache()
    start = [t.clone() for t in (s.p.k, s.p.v, s.p.ks, s.p.vs)]
    paged.rope_write8(s.args, cache)
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        paged.rope_write8(s.args, cache)
    for step in range(3):
        for t in (s.q, s.k, s.v):
            t.normal_(generator=P.gen(step))
        s.slots = [40 + 3 * step + i for i in range(35)]
        s.slot.copy_(P.ints(s.slots))
        for t, w in zip((s.p.k, s.p.v, s.p.ks, s.p.vs), start):
            t.copy_(w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (s.p.k, s.p.v, s.p.ks, s.p.vs, s.q16)]
        for t, w in zip((s.p.k, s.p.v, s.p.ks, s.p.vs), start):
            t.copy_(w)
        s.check()
        assert all(torch.equal(a, b) for a, b in zip(got, (s.p.k, s.p.v, s.p.ks, s.p.vs, s.q16)))
