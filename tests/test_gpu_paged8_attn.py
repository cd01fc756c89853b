"""Attention of new rows over 8-bit pages (rf_paged_attention8_launch) against float64 on
what the codes stand for: batches, lengths around pages and tiles, head layouts, windows,
strides, empty rows, and what must not enter."""
import math

import pytest
import torch

from rocmforge_amd import paged

from . import paged8_util as E
from . import paged_util as P
from .test_gpu_paged_attn import Case as Case16

pytestmark = pytest.mark.gpu


class Case(Case16):
    """The fp16 case with its pages rounded to 8 bits; k and v: what they then hold, in fp16 (exact)."""

    def __init__(self, new, kv, nh=8, nkv=2, d=128, page=16, by_head=False, extra=0, sizes=1.0, **kw):
        super().__init__(new, kv, nh, nkv, d, page, **kw)
        self.p = E.Pages(self.k.shape[0], page, nkv, d, by_head, 2 * extra)
        if sizes != 1.0:                                     # blocks of different exponents
            for x in (self.k, self.v):
                x *= sizes ** torch.linspace(-1, 1, x.shape[0] * page, device=P.DEV).view(-1, page, 1, 1).half()
        self.p.hold(self.k, self.v)
        self.take()

    def take(self):
        self.k, self.v = [x.half() for x in self.p.values()]
        self.cache = self.p.cache()

    def run(self):
        print(f"[gpu] new {self.new[:6]} kv {self.kv[:6]} heads {self.nh} d {self.d} window {self.window}", flush=True)
        paged.attention8(self.args, self.cache)
        torch.cuda.synchronize()
        return self.live()

    def at(self, b, t):
        return self.tab[b, t // self.p.page].long(), t % self.p.page


@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 640, 1025, 5000])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_token(rf, dev, kv, d):
    Case([1], [kv], d=d).check()


@pytest.mark.parametrize("nh,nkv", [(1, 1), (4, 4), (5, 1), (7, 1), (8, 1), (16, 2), (28, 4), (17, 1), (64, 1), (33, 3)])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [40, 300, 77]), ([3, 70, 1], [3, 200, 1])])
def test_head_layouts(rf, dev, nh, nkv, new, kv):
    Case(new, kv, nh, nkv).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_and_orders(rf, dev, page, by_head, d):
    Case([1, 5, 100, 0, 1, 260], [700, 33, 100, 12, 1, 1300], page=page, by_head=by_head, d=d, extra=8).check()


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv", [([1, 1], [2000, 40]), ([150, 3], [2000, 60])])
def test_blocks_of_many_exponents(rf, dev, page, d, new, kv):
    Case(new, kv, page=page, d=d, sizes=8.0, dist=lambda *s, **k: torch.randn(*s, **k) * 0.5).check()


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 31, 32, 33, 63, 64, 65, 128, 200, 513])
@pytest.mark.parametrize("before", [0, 1, 63, 64, 500])
def test_pieces_of_prompt(rf, dev, n, before):
    Case([n], [n + before]).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 65, 200, 100000])
def test_windows(rf, dev, window, d):
    Case([1, 1, 130, 7, 300], [50, 1000, 130, 400, 1111], window=window, d=d).check()


@pytest.mark.parametrize("out_f32", [0, 1])
def test_padding_strides_and_types(rf, dev, out_f32):
    Case([1, 90, 2], [333, 120, 64], pad=13, wide=40, extra=16, out_f32=out_f32).check()


def test_empty_requests_and_rows(rf, dev):
    c = Case([0, 3, 0, 1, 40, 0, 1], [50, 0, 0, 0, 25, 7, 20])
    c.check()
    got = c.live()
    assert bool((got[:4] == 0).all()) and bool((got[4:19] == 0).all()) and bool((got[19] != 0).any())


def test_all_empty(rf, dev):
    assert bool((Case([2, 2], [0, 0]).run() == 0).all())


@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 700])
def test_many_requests(rf, dev, seqs):
    kv = [1 + (37 * i) % 211 for i in range(seqs)]
    new = [1 + (i % 7 == 0) * min(kv[i] - 1, i % 29) for i in range(seqs)]
    Case(new, kv, 4, 2, 64).check()
    Case([1] * seqs, kv, 4, 2, 64, seed=1).check()


@pytest.mark.parametrize("seqs", [16, 17, 64, 65])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_lengths_of_all_kinds(rf, dev, seqs, d):
    # parts of many lengths, in whichever order the kernels take them; empty requests among them
    kv = [(i % 5 > 0) * (1 + (1237 * i * i) % 6000) for i in range(seqs)]
    Case([min(1, n) for n in kv], kv, 8, 2, d, seed=2).check()


@pytest.mark.parametrize("seqs", [1, 5, 64, 65])
@pytest.mark.parametrize("window", [0, 100, 700])
def test_prompts_of_all_kinds(rf, dev, seqs, window):
    # tiles that grow and tiles that a window makes equal, with requests that begin somewhere and at 0
    new = [(i % 4 < 3) * (1 + (331 * i * i + 200) % 390) for i in range(seqs)]
    kv = [n + (i % 3) * (i * 97 % 900) for i, n in enumerate(new)]
    Case(new, kv, 4, 2, 256, window=window, seed=3).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_requests_beside_short_ones(rf, dev, d):
    Case([1, 1, 1, 1], [9000, 3, 20000, 250], nh=4, nkv=1, d=d).check()
    Case([40, 1, 300], [9000, 5000, 7000], nh=4, nkv=1, d=d, page=64).check()


@pytest.mark.parametrize("hint", [0, 1, 1 << 30])
def test_the_hint_changes_no_result(rf, dev, hint):
    c = Case([1, 6, 150], [400, 20, 900])
    c.args.max_new = hint
    c.check()


@pytest.mark.parametrize("new,kv", [([1], [900]), ([5], [800]), ([100], [700])])
@pytest.mark.parametrize("scale", [0.0, -0.11, 2.0])
def test_scales(rf, dev, new, kv, scale):
    # scores stay below 64: 128 dims of |q k| around 1 over 8, times the scale
    Case(new, kv, scale=scale, dist=lambda *s, **k: torch.randn(*s, **k) * 0.25).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new,kv", [([70], [70]), ([130, 1, 4], [300, 90, 77]), ([4], [64]), ([300], [2000])])
def test_what_a_row_does_not_see_stays_out(rf, dev, d, window, new, kv):
    """NaN in K and V at positions from a row on: the rows in front of it keep their bits."""
    c = Case(new, kv, window=window, d=d)
    want = c.run()
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        for i in (n - 1, n - n // 3, n // 2 + 1):
            if 0 < i < n:
                c.p.k[c.at(b, m - n + i)] = 0x7f
                c.p.v[c.at(b, m - n + i)] = 0xff
        if window:                                     # and behind every row's window
            for t in range(max(0, m - n + 1 - window)):
                c.p.k[c.at(b, t)] = 0xff
                c.p.v[c.at(b, t)] = 0x7f
        at += n
    got = c.run()
    at = 0
    for n in new:
        clean = min([i for i in (n - 1, n - n // 3, n // 2 + 1) if 0 < i < n] + [n])
        assert bool((got[at:at + clean] == want[at:at + clean]).all())
        if clean < n:                                  # who sees it has it
            assert bool((~got[at + n - 1].isfinite()).all())
        at += n


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv,window", [(4, 500, 0), (3, 130, 0), (100, 100, 0), (64, 700, 0), (300, 2000, 0), (130, 300, 60)])
def test_large_keys_behind_a_row(rf, dev, d, new, kv, window):
    """Codes and exponents that only the last rows see: the others keep their bits."""
    c = Case([new], [kv], window=window, d=d)
    block = 16 * ((kv - 1) // 16)                      # the last block starts here
    want = c.run().half().view(torch.int16).clone()
    seen = max(kv - block, 0)                          # by that many of the last rows
    if seen >= new:
        seen = new
    pg, row = c.at(0, block)
    for t in range(block, kv):
        c.p.k[c.at(0, t)] = 0x7e
        c.p.v[c.at(0, t)] = 0xfe
    c.p.ks[pg], c.p.vs[pg] = 127 + 3, 134
    got = c.run().half().view(torch.int16)
    assert torch.equal(got[:new - seen], want[:new - seen])
    assert not torch.equal(got[new - seen:], want[new - seen:])


def poison(c):
    """One request, NaN in its V at one position after the other, in dims of KV head 0."""
    n, kv, group = c.new[0], c.kv[0], c.nh // c.v.shape[2]
    dims = (0, c.d // 2, c.d - 1)
    want = c.run().clone()
    assert bool(want.isfinite().all())
    pos = torch.arange(kv - n, kv, device=P.DEV)
    first = kv - n
    near = {p for e in (0, first, first - c.window, kv - c.window, kv) for p in range(e - 67, e + 68, 3)}
    ok, at = [], sorted(p for p in (range(kv) if kv <= 200 else near) if 0 <= p < kv)
    for t in at:
        row = c.p.v[c.at(0, t)][0]
        kept = row.clone()
        for i, code in zip(dims, (0x7f, 0xff, 0x7f)):
            row[i] = code
        paged.attention8(c.args, c.cache)
        got = c.live()
        sees = (t <= pos) & ((t > pos - c.window) if c.window else torch.ones_like(pos, dtype=torch.bool))
        expect = want.clone()
        for i in dims:
            expect[:, :group, i] = torch.where(sees[:, None], math.nan, expect[:, :group, i])
        ok.append(((got == expect) | (got.isnan() & expect.isnan())).all())
        row.copy_(kept)
    torch.cuda.synchronize()
    wrong = [t for t, o in zip(at, torch.stack(ok).tolist()) if not o]
    assert not wrong, f"positions {wrong[:20]} of {len(wrong)}"


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40, 200])
@pytest.mark.parametrize("new,kv", [(1, 77), (4, 64), (3, 190), (4, 600), (40, 40), (100, 100), (33, 150), (70, 700)])
def test_nan_in_v(rf, dev, d, window, new, kv):
    poison(Case([new], [kv], window=window, d=d))


@pytest.mark.parametrize("new,kv", [(2, 3000), (90, 5000)])
def test_nan_in_v_of_requests_in_parts(rf, dev, new, kv):
    poison(Case([new], [kv], nh=4, nkv=1))


@pytest.mark.parametrize("new,kv", [([1], [500]), ([90], [500])])
def test_nan_in_k(rf, dev, new, kv):
    c = Case(new, kv)
    c.p.k[c.at(0, kv[0] - new[0] - 30)][0, 5] = 0x7f
    got = c.run()
    assert bool(got[:, :4].isnan().all()) and bool(got[:, 4:].isfinite().all())


@pytest.mark.parametrize("new,kv", [([1], [500]), ([2], [40]), ([90], [500])])
def test_infinite_scores(rf, dev, new, kv):
    # an infinity in q: products with keys of either sign, and of zero, are infinities and NaN as in the formula
    c = Case(new, kv)
    c.p.k[..., 7] = 0xb8                               # -1 2^e
    c.take()
    c.q[0, 7] = math.inf                               # head 0 of row 0: every score is -inf
    c.q[0, 128 + 7] = -math.inf                        # head 1: every score is +inf
    got = c.run()
    assert bool(got[0, :2].isnan().all()) and bool(got[0, 2:].isfinite().all()) and bool(got[1:].isfinite().all())


@pytest.mark.parametrize("new,kv", [([1, 1], [300, 300]), ([70, 80], [300, 300])])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_pages_outside_the_cache_are_not_read(rf, dev, new, kv, bad):
    c = Case(new, kv)
    want = c.run()
    c.tab[0, 3] = bad
    got = c.run()
    assert bool((got[new[0]:] == want[new[0]:]).all()) and bool(got[:new[0]].isnan().all())


@pytest.mark.parametrize("byte,e", [(0, -15), (111, -15), (112, -15), (134, 7), (135, 7), (255, 7)])
@pytest.mark.parametrize("new,kv", [([1], [100]), ([40], [100])])
def test_exponents_outside_the_range(rf, dev, new, kv, byte, e):
    c = Case(new, kv, scale=2.0 ** -20, dist=lambda *s, **k: torch.randn(*s, **k).clamp(-3, 3))
    c.p.ks.fill_(byte)
    c.p.vs.fill_(byte)
    c.take()
    assert c.v[c.at(0, 0)].abs().max() <= 448 * 2.0 ** e
    c.check()


@pytest.mark.parametrize("d,nh,nkv", [(64, 4, 1), (128, 8, 2), (128, 7, 1), (256, 6, 2)])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("new,kv", [([1], [500]), ([1, 1, 2], [130, 1000, 700]), ([100], [100]), ([3, 90, 1], [200, 2100, 900]),
                                    ([400], [3500]), ([9, 0, 140, 1], [160, 50, 1700, 3])])
def test_tables_wider_than_the_lengths(rf, dev, new, kv, window, d, nh, nkv):
    c = Case(new, kv, nh, nkv, d, window=window)
    c.tab = torch.nn.functional.pad(c.tab, (0, 6000 - c.tab.shape[1]), value=-3).contiguous()
    c.args.block_tables, c.args.max_blocks = c.tab, 6000
    c.check()


def test_lengths_beyond_the_table_are_clipped(rf, dev):
    c = Case([1, 60], [100, 100], page=32)
    c.args.max_blocks = 4
    tab = c.tab[:, :4].contiguous()
    c.args.block_tables = tab
    for b in range(2):
        t = torch.arange(100, 128, device=P.DEV)
        for x in (c.p.k, c.p.v):
            x[tab[b].long()[t // 32], t % 32] = 0x30
    c.take()
    c.kv_lens.copy_(P.ints([4000, 1 << 30]))
    c.kv = [128, 128]
    c.check()


def test_every_run_gives_the_same_bits(rf, dev):
    c = Case([1, 1, 200, 3], [9000, 700, 2000, 50])
    want = c.run()
    for _ in range(3):
        c.out.fill_(7.0)
        assert torch.equal(c.run(), want)


def test_far_into_a_large_cache(rf, dev):
    # offsets beyond 32 bits
    page, nkv, d = 16, 2, 128
    pages = 5 * (1 << 30) // (page * nkv * d)
    k, v = [torch.empty(pages, page, nkv, d, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    ks, vs = [torch.empty(pages, 1, nkv, dtype=torch.uint8, device=P.DEV) for _ in range(2)]
    c = Case([1, 90], [400, 500], nh=8, nkv=nkv, d=d, page=page)
    want = c.run()
    n = c.p.k.shape[0]
    for a, b in ((k, c.p.k), (v, c.p.v), (ks, c.p.ks), (vs, c.p.vs)):
        a[pages - n:] = b
    c.p.k, c.p.v, c.p.ks, c.p.vs = k, v, ks, vs
    c.tab = torch.where(c.tab < n, c.tab + pages - n, c.tab)
    c.args.block_tables, c.cache = c.tab, c.p.cache()
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("new,kv", [([1] * 5, [3000, 40, 900, 1, 257]), ([120, 1, 300], [700, 4000, 300])])
def test_replays(rf, dev, new, kv):
    """A captured launch reads lengths, rows and tables as they are at each replay."""
    c = Case(new, kv, pad=3)
    c.run()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        paged.attention8(c.args, c.cache)
    for step in range(4):
        c.kv = [max(m - 13 * step, 0) if i % 2 == 0 else m for i, m in enumerate(kv)]
        c.kv_lens.copy_(P.ints(c.kv))
        c.out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        replayed = c.live().clone()
        c.check(replayed)
        c.ws.fill_(math.nan)
        assert torch.equal(c.run(), replayed)


def test_two_streams_with_workspaces_of_their_own(rf, dev):
    cases = [Case([1, 1], [9000, 70], seed=1), Case([200, 1], [900, 8000], seed=2)]
    want = [c.run().clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            paged.attention8(c.args, c.cache, s)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.live(), w)


@pytest.mark.parametrize("lead", [8.0, 10.5, 12.0])
@pytest.mark.parametrize("new,kv", [([1], [16000]), ([40], [16000]), ([2], [3000])])
def test_many_small_weights_beside_a_large_one(rf, dev, lead, new, kv):
    # weights around and below fp16's smallest normal one, thousands of them: they count
    c = Case(new, kv, nh=2, nkv=1)
    c.p.k.fill_(0)
    c.p.ks.fill_(127)
    c.p.k[c.at(0, kv[0] // 3)][0, 0] = 0x38            # 1
    c.p.v &= 0x7f
    c.p.v.masked_fill_(c.p.v == 0x7f, 0)
    c.take()
    c.q.zero_()
    c.q.view(-1, 2, 128)[:, :, 0] = lead / c.scale
    c.check()
