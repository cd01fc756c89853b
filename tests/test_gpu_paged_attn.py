"""Attention of new rows over a paged cache (rf_paged_attention_launch) against
float64: batches from one token to pieces of prompt, lengths around pages and
tiles, head layouts, windows, strides, empty rows, and what must not enter."""
import math

import pytest
import torch

from rocmforge_amd import paged

from . import paged_util as P

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, new, kv, nh=8, nkv=2, d=128, page=16, window=0, by_head=False, extra=0, out_f32=0, pad=0,
                 wide=0, seed=0, scale=None, dist=torch.randn):
        g = P.gen(1000 * seed + 7 * sum(new) + sum(kv) + d)
        pages = sum(-(-n // page) for n in kv) + 3
        self.k, self.v = P.cache_tensors(pages, page, nkv, d, by_head, extra)
        self.tab = P.tables(kv, page, pages, g)
        P.fill(self.k, self.v, self.tab, kv, g, dist)
        self.new, self.kv, self.window = new, kv, window
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        rows = sum(new) + pad
        q = torch.randn(rows, nh * d + wide, generator=g, device=P.DEV).half()
        self.q = q[:, :nh * d]
        self.out = torch.full((rows, nh * d + wide), 7.0, device=P.DEV, dtype=torch.float32 if out_f32 else torch.float16)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.q_start, self.kv_lens = P.ints(starts), P.ints(kv)
        self.cache = P.cache_block(self.k, self.v)
        n = paged.attention_workspace_bytes(nh, nkv, d)
        self.ws = torch.full(((n + 3) // 4,), math.nan, device=P.DEV)
        self.nh, self.d, self.pad = nh, d, pad
        self.args = paged.PagedAttention(
            q=self.q, out=self.out, block_tables=self.tab, q_start=self.q_start, kv_lens=self.kv_lens,
            workspace=self.ws, workspace_bytes=n, ld_q=self.q.stride(0), ld_out=self.out.stride(0),
            num_seqs=len(new), max_blocks=self.tab.shape[1], rows=rows, num_heads=nh, max_new=max(new), window=window,
            out_f32=out_f32, scale=self.scale)

    def run(self):
        print(f"[gpu] new {self.new[:6]} kv {self.kv[:6]} heads {self.nh} d {self.d} window {self.window}", flush=True)
        paged.attention(self.args, self.cache)
        torch.cuda.synchronize()
        return self.live()

    def live(self):
        n = sum(self.new)
        return self.out[:n, :self.nh * self.d].reshape(n, self.nh, self.d).double()

    def check(self, got=None):
        got = self.run() if got is None else got
        n = sum(self.new)
        want, bound = P.attention64(self.q[:n].reshape(n, self.nh, self.d), self.k, self.v, self.tab, self.new, self.kv,
                                    self.window, self.scale)
        worst = ((got - want).abs() / bound).max().item() if n else 0.0
        print(f"largest error {worst:.2f} of the bound", flush=True)
        assert bool(((got - want).abs() <= bound).all()), worst
        assert bool((self.out[n:] == 7.0).all())                       # padding rows
        assert bool((self.out[:, self.nh * self.d:] == 7.0).all())     # between rows


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


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 31, 32, 33, 63, 64, 65, 128, 200, 513])
@pytest.mark.parametrize("before", [0, 1, 63, 64, 500])
def test_pieces_of_prompt(rf, dev, n, before):
    Case([n], [n + before], page=16).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 65, 200, 100000])
def test_windows(rf, dev, window, d):
    Case([1, 1, 130, 7, 300], [50, 1000, 130, 400, 1111], window=window, d=d).check()


@pytest.mark.parametrize("out_f32", [0, 1])
def test_padding_strides_and_types(rf, dev, out_f32):
    Case([1, 90, 2], [333, 120, 64], pad=13, wide=40, extra=16, out_f32=out_f32).check()


def test_empty_requests_and_rows(rf, dev):
    # requests without rows, refused ones (length 0), and more rows than positions
    c = Case([0, 3, 0, 1, 40, 0, 1], [50, 0, 0, 0, 25, 7, 20])
    c.check()
    got = c.live()
    assert bool((got[:4] == 0).all()) and bool((got[4:19] == 0).all()) and bool((got[19] != 0).any())


def test_all_empty(rf, dev):
    c = Case([2, 2], [0, 0])
    assert bool((c.run() == 0).all())


@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 700])
def test_many_requests(rf, dev, seqs):
    kv = [1 + (37 * i) % 211 for i in range(seqs)]
    new = [1 + (i % 7 == 0) * min(kv[i] - 1, i % 29) for i in range(seqs)]
    Case(new, kv, 4, 2, 64).check()
    Case([1] * seqs, kv, 4, 2, 64, seed=1).check()


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
    c = Case(new, kv, scale=scale, dist=lambda *s, **k: torch.randn(*s, **k) * 0.25)
    c.check()


@pytest.mark.parametrize("new,kv", [([1], [900]), ([1, 3, 200], [16000, 300, 500])])
def test_large_scores(rf, dev, new, kv):
    # one key leads by far: the row is its V with a weight of one
    c = Case(new, kv, nh=2, nkv=1)
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        first = m - n                                  # position 0 .. of the request's first row
        t = first // 2
        pg = c.tab[b, t // 16].long()
        c.q[at:at + n] = 200.0
        for j in range(m):
            c.k[c.tab[b, j // 16].long(), j % 16] = 200.0 * (0.5 if j != t else 1.0)
        at += n
    got = c.run()
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        t = (m - n) // 2
        v = c.v[c.tab[b, t // 16].long(), t % 16].double()
        assert bool((got[at:at + n] == v[0]).all())
        at += n


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new,kv", [([70], [70]), ([130, 1, 4], [300, 90, 77]), ([4], [64]), ([300], [2000])])
def test_what_a_row_does_not_see_stays_out(rf, dev, d, window, new, kv):
    """NaN and infinities in K and V at positions from a row on: the rows in front of
    it keep their bits."""
    c = Case(new, kv, window=window, d=d)
    want = c.run()
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        for i, bad in ((n - 1, math.nan), (n - n // 3, math.inf), (n // 2 + 1, -math.inf)):
            if 0 < i < n:
                t = m - n + i
                c.k[c.tab[b, t // 16].long(), t % 16] = bad
                c.v[c.tab[b, t // 16].long(), t % 16] = bad
        if window:                                     # and behind every row's window
            for t in range(max(0, m - n + 1 - window)):
                c.k[c.tab[b, t // 16].long(), t % 16] = math.nan
                c.v[c.tab[b, t // 16].long(), t % 16] = math.nan
        at += n
    got = c.run()
    at = 0
    for n in new:
        clean = min([i for i in (n - 1, n - n // 3, n // 2 + 1) if 0 < i < n] + [n])
        assert bool((got[at:at + clean] == want[at:at + clean]).all())
        if clean < n:                                  # who sees it has it
            assert bool((~got[at + n - 1].isfinite()).all())
        at += n


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("new,kv", [([1], [500]), ([90], [500])])
def test_what_a_row_sees_comes_through(rf, dev, where, new, kv):
    c = Case(new, kv)
    t = kv[0] - new[0] - 30
    getattr(c, where)[c.tab[0, t // 16].long(), t % 16, 0] = math.nan
    got = c.run()
    assert bool(got[:, :4].isnan().all()) and bool(got[:, 4:].isfinite().all())


@pytest.mark.parametrize("new,kv", [([1, 1], [300, 300]), ([70, 80], [300, 300])])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_pages_outside_the_cache_are_not_read(rf, dev, new, kv, bad):
    c = Case(new, kv)
    want = c.run()
    c.tab[0, 3] = bad
    got = c.run()
    assert bool((got[new[0]:] == want[new[0]:]).all()) and bool(got[:new[0]].isnan().all())


@pytest.mark.parametrize("d,nh,nkv", [(64, 4, 1), (128, 8, 2), (128, 7, 1), (256, 6, 2)])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("new,kv", [([1], [500]), ([1, 1, 2], [130, 1000, 700]), ([100], [100]), ([3, 90, 1], [200, 2100, 900]),
                                    ([400], [3500]), ([9, 0, 140, 1], [160, 50, 1700, 3])])
def test_tables_wider_than_the_lengths(rf, dev, new, kv, window, d, nh, nkv):
    # (the table's width bounds the parts that a request may be cut into)
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
        for x in (c.k, c.v):
            x[tab[b].long()[t // 32], t % 32] = 0.5
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
    # element offsets beyond 32 bits: pages at the end of 5 x 2^31 elements of K and V
    page, nkv, d = 16, 2, 128
    pages = 5 * (1 << 31) // (page * nkv * d)
    k, v = [torch.empty(pages, page, nkv, d, dtype=torch.float16, device=P.DEV) for _ in range(2)]
    g = P.gen(3)
    new, kv = [1, 90], [400, 500]
    c = Case(new, kv, nh=8, nkv=nkv, d=d, page=page)
    far = torch.randperm(1000, generator=g, device=P.DEV) + pages - 1000
    tab = c.tab.clone()
    at = 0
    for b, n in enumerate(kv):
        m = -(-n // page)
        own = far[at:at + m]
        k[own], v[own] = c.k[c.tab[b, :m].long()], c.v[c.tab[b, :m].long()]
        tab[b, :m] = own.int()
        at += m
    want = c.run()
    c.args.block_tables = tab
    c.cache = P.cache_block(k, v)
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("new,kv", [([1] * 5, [3000, 40, 900, 1, 257]), ([120, 1, 300], [700, 4000, 300])])
def test_replays(rf, dev, new, kv):
    """A captured launch reads lengths, rows and tables as they are at each replay."""
    c = Case(new, kv, pad=3)
    c.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        paged.attention(c.args, c.cache)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        paged.attention(c.args, c.cache)
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
            paged.attention(c.args, c.cache, s)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.live(), w)


@pytest.mark.parametrize("lead", [8.0, 10.0, 10.5, 11.0, 12.0])
@pytest.mark.parametrize("new,kv", [([1], [16000]), ([40], [16000]), ([2], [3000])])
def test_many_small_weights_beside_a_large_one(rf, dev, lead, new, kv):
    # weights around and below fp16's smallest normal one, thousands of them: they count
    c = Case(new, kv, nh=2, nkv=1)
    for j in range(-(-kv[0] // 16)):
        c.k[c.tab[0, j].long()] = 0.0
    t = kv[0] // 3
    c.k[c.tab[0, t // 16].long(), t % 16, 0, 0] = 1.0
    c.q.zero_()
    c.q.view(-1, 2, 128)[:, :, 0] = lead / c.scale
    c.v.copy_((c.v.float().abs() + 1).half())
    c.check()
