"""The plan of a batch's step (rf_paged_plan_launch) and the return of pages
(rf_paged_release_launch) against a host that serves one request after the other."""
import random

import pytest
import torch

from rocmforge_amd import paged

from . import paged_util as P

pytestmark = pytest.mark.gpu
INT_MAX = 2 ** 31 - 1


def host_plan(new, ctx, tab, free, n_free, page, max_rows, num_pages):
    tab = [list(r) for r in tab]
    left = min(max(n_free, 0), num_pages)
    asked = taken = start = 0
    pos, slot = [0] * max_rows, [-1] * max_rows
    q_start, kv, out = [0], [], []
    for b, (n, c) in enumerate(zip(new, ctx)):
        end = start + max(n, 0)
        have, want = -(-c // page), -(-(c + n) // page)
        ok = n >= 0 and c >= 0 and end <= max_rows and want <= len(tab[b]) and c + n <= INT_MAX
        if ok and want > have:
            asked += want - have
            ok = asked <= left
        if ok:
            for col in range(have, want):
                taken += 1
                tab[b][col] = free[left - taken]
            for i in range(n):
                pos[start + i] = c + i
                slot[start + i] = tab[b][(c + i) // page] * page + (c + i) % page
        start = end
        q_start.append(min(start, max_rows))
        kv.append(c + n if ok else 0)
        out.append(c + n if ok else c)
    return dict(tab=tab, q_start=q_start, kv=kv, ctx=out, pos=pos, slot=slot, n_free=left - taken)


class Step:
    def __init__(self, new, ctx, page=16, free=1000, max_rows=None, width=None, n_free=None, in_place=False, seed=0):
        rng = random.Random(seed)
        self.page = page
        width = max([-(-max(c + n, c, 0) // page) for n, c in zip(new, ctx)] + [1]) if width is None else width
        self.max_rows = sum(max(n, 0) for n in new) if max_rows is None else max_rows
        own = sum(min(-(-max(c, 0) // page), width) for c in ctx)
        self.num_pages = own + free
        ids = list(range(self.num_pages))
        rng.shuffle(ids)
        tab, at = [], 0
        for c in ctx:
            k = min(-(-max(c, 0) // page), width)
            tab.append(ids[at:at + k] + [-5] * (width - k))
            at += k
        self.free = ids[at:] + [-6] * own
        self.host = host_plan(new, ctx, tab, self.free, free if n_free is None else n_free, page, self.max_rows,
                              self.num_pages)
        B = len(new)
        z = lambda n: torch.full((max(n, 1),), -7, dtype=torch.int32, device=P.DEV)
        self.t = dict(new=P.ints(new), ctx_in=P.ints(ctx), free=P.ints(self.free + [0]),
                      n_in=P.ints([free if n_free is None else n_free]), tab=P.ints(tab).reshape(-1), q_start=z(B + 1),
                      kv=z(B), pos=z(self.max_rows), slot=z(self.max_rows))
        self.t["ctx"] = self.t["ctx_in"] if in_place else z(B)
        self.t["n_free"] = self.t["n_in"] if in_place else z(1)
        t = self.t
        self.args = paged.PagedPlan(new_lens=t["new"], ctx_in=t["ctx_in"], ctx_out=t["ctx"], free_pages=t["free"],
                                    free_in=t["n_in"], free_out=t["n_free"], block_tables=t["tab"],
                                    q_start=t["q_start"], kv_lens=t["kv"], positions=t["pos"], slots=t["slot"],
                                    num_seqs=B, max_blocks=width, page_size=page, max_rows=self.max_rows,
                                    num_pages=self.num_pages)

    def check(self):
        print(f"[gpu] plan of {self.args.num_seqs} requests, {self.max_rows} rows, page {self.page}", flush=True)
        paged.plan(self.args)
        torch.cuda.synchronize()
        self.same()

    def same(self):
        for name, want in self.host.items():
            got = self.t[name].tolist()
            want = [x for r in want for x in r] if name == "tab" else want if isinstance(want, list) else [want]
            n = self.max_rows if name in ("pos", "slot") else len(want)
            assert got[:n] == want[:n], name


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [8, 16, 64, 1024])
def test_few_requests(rf, dev, page, in_place):
    Step([1], [0], page, in_place=in_place).check()
    Step([1, 1, 1], [15, 16, 17], page, in_place=in_place).check()
    Step([5, 0, 100, 1, 64], [3, 0, 0, 63, 64], page, in_place=in_place).check()
    Step([0, 0], [0, 7], page, max_rows=5, in_place=in_place).check()


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 1023, 1024, 1025, 3100])
def test_many_requests(rf, dev, seqs):
    rng = random.Random(seqs)
    new = [rng.choice([0, 1, 1, 1, rng.randint(0, 40)]) for _ in range(seqs)]
    ctx = [rng.randint(0, 90) for _ in range(seqs)]
    Step(new, ctx, free=8000, max_rows=sum(new) + 9).check()


def test_many_rows(rf, dev):
    # more rows than one workgroup writes, one request with most of them
    Step([1, 20000, 3, 700], [5, 31, 0, 1000], 16, free=3000).check()
    Step([8192], [0], 16).check()
    Step([8193], [0], 16).check()


@pytest.mark.parametrize("free", [0, 1, 2, 3, 5, 8, 40])
@pytest.mark.parametrize("in_place", [False, True])
def test_pages_run_out(rf, dev, free, in_place):
    # the request that asks for too much, and those behind it that need pages, are refused
    Step([20, 1, 90, 1, 1, 17], [0, 16, 5, 3, 32, 0], 16, free=free, in_place=in_place).check()
    seqs = 2500
    Step([1] * seqs, [16 * (i % 3) + (i % 5 == 0) for i in range(seqs)], 16, free=40 * free, in_place=in_place).check()


def test_rows_and_tables_run_out(rf, dev):
    Step([10, 30, 5, 1], [0, 0, 0, 0], max_rows=20).check()
    Step([10, 30, 0, 1], [0, 0, 9, 0], max_rows=10).check()
    Step([10, 300, 5, 1], [0, 0, 40, 47], width=3).check()
    Step([1, 1], [2000, 3], max_rows=0).check()


@pytest.mark.parametrize("seqs", [1024, 1025])
def test_many_requests_and_no_rows(rf, dev, seqs):
    Step([0] * seqs, list(range(seqs)), free=0, max_rows=0).check()
    Step([1] * seqs, [16] * seqs, free=9, max_rows=0).check()


def test_bad_lengths_are_refused(rf, dev):
    Step([3, -4, 2, 1], [10, 5, -3, 1], width=4).check()
    Step([1, INT_MAX, 1], [0, 5, 0], width=4, max_rows=9).check()
    Step([INT_MAX, INT_MAX, INT_MAX, 1], [0] * 4, width=4, max_rows=9).check()
    Step([1, 1], [INT_MAX, 3], width=4).check()


@pytest.mark.parametrize("n_free", [-3, 5000])
def test_counts_outside_the_stack(rf, dev, n_free):
    Step([40, 1], [0, 3], free=10, n_free=n_free).check()


def test_a_step_without_requests_is_all_padding(rf, dev):
    s = Step([], [], max_rows=70, width=1)
    s.check()
    assert s.t["slot"].tolist() == [-1] * 70 and s.t["pos"].tolist() == [0] * 70


def host_release(ended, ctx, tab, free, n, page, num_pages):
    ctx, free = list(ctx), list(free)
    at = n
    for b, e in enumerate(ended):
        k = -(-max(ctx[b], 0) // page)
        if e and 0 < k <= len(tab[b]):
            at += k
            if at <= num_pages:
                free[at - k:at] = tab[b][:k]
                n = at
                ctx[b] = 0
    return ctx, free, n


@pytest.mark.parametrize("seqs", [1, 5, 64, 1300])
@pytest.mark.parametrize("short", [0, 3])
def test_release(rf, dev, seqs, short):
    """short: the stack has room for that many pages less than come back (a second
    return of the same pages): the last requests keep theirs."""
    rng = random.Random(seqs + short)
    page, width = 16, 20
    ctx = [rng.randint(0, 16 * width) for _ in range(seqs)]
    ctx[0] = 200
    ended = [rng.randint(-1, 1) for _ in range(seqs)]
    ended[0] = 1
    tab = [[rng.randint(0, 10 ** 6) for _ in range(width)] for _ in range(seqs)]
    back = sum(-(-c // page) for c, e in zip(ctx, ended) if e)
    n = 11
    num_pages = n + back - short
    free = list(range(num_pages))
    want = host_release(ended, ctx, tab, free, n, page, num_pages)
    d = [P.ints(x) for x in (ended, ctx, tab, free + [-9] * 5, [n])]
    print(f"[gpu] release of {sum(map(bool, ended))} of {seqs} requests", flush=True)
    paged.release(*d, seqs, width, page, num_pages)
    torch.cuda.synchronize()
    assert d[1].tolist() == want[0] and d[4].tolist() == [want[2]]
    assert d[3].tolist() == want[1] + [-9] * 5


def test_release_leaves_bad_lengths_alone(rf, dev):
    d = [P.ints(x) for x in ([1, 1, 1], [-4, 1000, 20], [[1, 2, 3]] * 3, [0] * 9, [2])]
    paged.release(*d, 3, 3, 16, 9)
    torch.cuda.synchronize()
    assert d[1].tolist() == [-4, 1000, 0] and d[4].tolist() == [4] and d[3].tolist()[:5] == [0, 0, 1, 2, 0]
