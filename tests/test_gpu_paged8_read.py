"""Requests out of 8-bit pages (rf_paged_read8_launch): exactly what the codes stand for."""
import pytest
import torch

from rocmforge_amd import paged

from . import paged8_util as E
from . import paged_util as P

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, lens, first=None, nkv=2, d=128, page=16, by_head=False, extra=0, wide=0, pad=0, seed=0):
        g = P.gen(seed + sum(lens) + d)
        first = [0] * len(lens) if first is None else first
        ends = [a + b for a, b in zip(first, lens)]
        pages = sum(-(-max(n, 0) // page) for n in ends) + 2
        self.p = E.Pages(pages, page, nkv, d, by_head, extra)
        for t in (self.p.k, self.p.v):
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device=P.DEV, dtype=torch.uint8))
        for t in (self.p.ks, self.p.vs):
            t.copy_(torch.randint(105, 140, t.shape, generator=g, device=P.DEV, dtype=torch.uint8))
        self.tab = P.tables([max(n, 0) for n in ends], page, pages, g)
        self.lens, self.firsts, self.width = lens, first, nkv * d
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        rows = starts[-1] + pad
        self.out = [torch.full((rows, nkv * d + wide), 7.0, dtype=torch.float16, device=P.DEV) for _ in range(2)]
        self.args = paged.PagedRead(k=self.out[0], v=self.out[1], block_tables=self.tab, row_start=P.ints(starts),
                                    first=P.ints(first), ld_out=nkv * d + wide, num_seqs=len(lens),
                                    max_blocks=self.tab.shape[1], rows=rows)

    def run(self):
        print(f"[gpu] read8 {self.lens[:6]} {tuple(self.p.k.shape)}", flush=True)
        paged.read8(self.args, self.p.cache())
        torch.cuda.synchronize()

    def want(self):
        """Skipped rows, and what lies behind a row, keep their 7."""
        page = self.p.page
        res = []
        for x, out in zip(self.p.values(), self.out):
            w = torch.full(out.shape, 7.0, dtype=torch.float64, device=P.DEV)
            at = 0
            for b, (n, f) in enumerate(zip(self.lens, self.firsts)):
                t = torch.arange(f, f + n, device=P.DEV)
                there = (t >= 0) & (t < self.tab.shape[1] * page)
                pg = self.tab[b].long()[t.clamp(0, self.tab.shape[1] * page - 1) // page]
                there &= (pg >= 0) & (pg < x.shape[0])
                rows = x[pg.clamp(0, x.shape[0] - 1), t % page].flatten(1)
                w[at:at + n, :self.width] = torch.where(there[:, None], rows, w[at:at + n, :self.width])
                at += n
            res.append(w)
        return res

    def check(self, which=(0, 1)):
        self.run()
        want = self.want()
        for i in which:
            got = self.out[i].double()
            assert bool(((got == want[i]) | (got.isnan() & want[i].isnan())).all()), i


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nkv", [1, 3, 8])
@pytest.mark.parametrize("lens", [[1], [640], [15, 16, 17], [0, 5, 0, 0, 33, 0], [1] * 70, [3 + i % 40 for i in range(200)],
                                  [0] * 100 + [1] + [0] * 150 + [2, 1, 0, 1] + [0] * 70 + [9], [40] * 120, [5000, 1, 1, 0, 1]])
def test_lengths_and_heads(rf, dev, lens, nkv, d):
    Case(lens, nkv=nkv, d=d).check()


@pytest.mark.parametrize("page", [8, 16, 32, 128, 1024])
@pytest.mark.parametrize("by_head", [False, True])
def test_pages_orders_and_strides(rf, dev, page, by_head):
    Case([100, 1, 0, 333], page=page, by_head=by_head, extra=32, wide=24, pad=9).check()


def test_positions_from_somewhere_on(rf, dev):
    c = Case([20, 5, 40, 7], first=[100, 0, 3, -4])
    c.check()
    c = Case([20, 100, 9], first=[0, 50, 0])                     # beyond the table, and past 32 bits
    c.firsts = [(1 << 31) - 100, 50, (1 << 31) - 3]
    c.args.first = P.ints(c.firsts)
    c.check()


def test_pages_outside_the_cache(rf, dev):
    c = Case([100, 100])
    c.tab[0, 2], c.tab[1, 0] = -1, 1 << 20
    c.check()


def test_row_ranges_are_clipped(rf, dev):
    c = Case([50, 60])
    c.args.rows = 80
    c.run()
    want = [w[:80] for w in c.want()]
    for i in range(2):
        got = c.out[i].double()
        assert bool(((got[:80] == want[i]) | (got[:80].isnan() & want[i].isnan())).all()) and bool((got[80:] == 7.0).all())


@pytest.mark.parametrize("one", [0, 1])
def test_keys_or_values_alone(rf, dev, one):
    c = Case([100, 20])
    setattr(c.args, "kv"[1 - one], None)
    c.check([one])
    assert bool((c.out[1 - one] == 7.0).all())


def test_no_first(rf, dev):
    c = Case([100, 20])
    c.args.first = None
    c.check()


def test_every_code_under_every_exponent(rf, dev):
    c = Case([23 * 16], nkv=2, d=128)
    c.p.k.copy_(torch.arange(256, device=P.DEV).to(torch.uint8).view(1, 1, 2, 128).expand_as(c.p.k))
    c.p.ks.copy_((112 + torch.arange(c.p.ks.shape[0], device=P.DEV) % 23).to(torch.uint8)[:, None, None].expand_as(c.p.ks))
    c.check()


def test_far_into_a_large_cache(rf, dev):
    page, nkv, d = 16, 2, 128
    pages = 5 * (1 << 30) // (page * nkv * d)
    k, v = [torch.empty(pages, page, nkv, d, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    ks, vs = [torch.empty(pages, 1, nkv, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    c = Case([100, 37])
    c.run()
    want = [t.clone() for t in c.out]
    n = c.p.k.shape[0]
    for a, b in ((k, c.p.k), (v, c.p.v), (ks, c.p.ks), (vs, c.p.vs)):
        a[pages - n:] = b
    c.p.k, c.p.v, c.p.ks, c.p.vs = k, v, ks, vs
    c.tab = torch.where(c.tab < n, c.tab + pages - n, c.tab)
    c.args.block_tables = c.tab
    for t in c.out:
        t.fill_(7.0)
    c.run()
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(c.out, want))


def test_replays(rf, dev):
    c = Case([100, 37, 5])
    cache = c.p.cache()
    paged.read8(c.args, cache)
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        paged.read8(c.args, cache)
    for lens in ([50, 60, 32], [0, 100, 7], [100, 37, 5]):
        c.lens = lens
        c.args._kept["row_start"].copy_(P.ints([0, lens[0], lens[0] + lens[1], sum(lens)]))
        for t in c.out:
            t.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(c.out, c.want()):
            got = got.double()
            # (entries of the tables behind a request's pages name none)
            assert bool(((got == want) | (got.isnan() & want.isnan())).all())


def test_more_rows_than_one_dimension_of_a_launch_has(rf, dev):
    # 2^26 rows and some, all of the same page
    rows, d = (1 << 26) + 5000, 64
    p = E.Pages(1, 1024, 1, d)
    g = P.gen(3)
    p.hold(*[torch.randn(1, 1024, 1, d, generator=g, device=P.DEV) for _ in range(2)])
    blocks = -(-rows // 1024)
    tab, starts = torch.zeros(1, blocks, dtype=torch.int32, device=P.DEV), P.ints([0, rows])
    out = torch.full((rows, d), 7.0, dtype=torch.float16, device=P.DEV)
    print(f"[gpu] read8 rows {rows}", flush=True)
    paged.read8(paged.PagedRead(k=out, block_tables=tab, row_start=starts, ld_out=d, num_seqs=1, max_blocks=blocks,
                                rows=rows), p.cache())
    torch.cuda.synchronize()
    page = p.values()[0].half().view(1024, d)
    for at in (0, (1 << 24) - 1024, (1 << 26) - 1024, (1 << 26) + 2048):
        assert torch.equal(out[at:at + 1024], page), at
    assert torch.equal(out[-(rows % 1024):], page[:rows % 1024])
