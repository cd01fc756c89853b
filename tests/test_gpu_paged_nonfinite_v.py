"""Infinities and NaN in V (rf_paged_attention_launch): every row that sees one has
it, every other row keeps its bits, wherever the position lies in a tile."""
import math

import pytest
import torch

from . import paged_util as P
from .test_gpu_paged_attn import Case

pytestmark = pytest.mark.gpu
BAD = (math.nan, math.inf, -math.inf)


def positions(kv, window, n):
    """All of a short request; of a long one those around its rows, their windows' edges and its start."""
    if kv <= 200:
        return range(kv)
    first = kv - n
    near = {p for e in (0, first, first - window, kv - window, kv) for p in range(e - 67, e + 68, 3)}
    near |= {p for e in (0, first, first - window, kv - window, kv) for b in (-64, -32, 0, 32, 64)
             for p in ((e + b) // 32 * 32 - 1, (e + b) // 32 * 32)}
    return sorted(p for p in near if 0 <= p < kv)


def check(c):
    """One request, its V poisoned at one position after the other, in KV head 0: NaN in
    dim 0, +inf in the middle, -inf in the last."""
    n, kv, d, group = c.new[0], c.kv[0], c.d, c.nh // c.v.shape[2]
    dims = (0, d // 2, d - 1)
    want = c.run().clone()
    assert bool(want.isfinite().all())
    pos = torch.arange(kv - n, kv, device=P.DEV)
    import rocmforge_amd.paged as paged
    ok, at = [], list(positions(kv, c.window, n))
    for t in at:
        row = c.v[c.tab[0, t // 16].long(), t % 16, 0]
        kept = row.clone()
        for i, bad in zip(dims, BAD):
            row[i] = bad
        paged.attention(c.args, c.cache)
        got = c.live()
        sees = (t <= pos) & ((t > pos - c.window) if c.window else torch.ones_like(pos, dtype=torch.bool))
        expect = want.clone()
        for i, bad in zip(dims, BAD):
            expect[:, :group, i] = torch.where(sees[:, None], bad, expect[:, :group, i])
        ok.append(((got == expect) | (got.isnan() & expect.isnan())).all())
        row.copy_(kept)
    torch.cuda.synchronize()
    wrong = [t for t, o in zip(at, torch.stack(ok).tolist()) if not o]
    assert not wrong, f"positions {wrong[:20]} of {len(wrong)}"


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40, 200])
@pytest.mark.parametrize("new,kv", [(40, 40), (64, 64), (100, 100), (33, 150), (64, 190), (70, 700)])
def test_pieces_of_prompt(rf, dev, d, window, new, kv):
    check(Case([new], [kv], window=window, d=d))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40, 200])
@pytest.mark.parametrize("new,kv", [(1, 77), (4, 64), (3, 190), (4, 600)])
def test_few_rows(rf, dev, d, window, new, kv):
    check(Case([new], [kv], window=window, d=d))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1500])
@pytest.mark.parametrize("new,kv", [(2, 3000), (90, 5000)])
def test_requests_in_parts(rf, dev, d, window, new, kv):
    check(Case([new], [kv], nh=4, nkv=1, window=window, d=d))


@pytest.mark.parametrize("hint", [0, 1, 1 << 30])
def test_whatever_the_hint(rf, dev, hint):
    c = Case([4], [150], window=90)
    c.args.max_new = hint
    check(c)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (5, 1), (28, 4)])
def test_head_layouts(rf, dev, nh, nkv):
    check(Case([60], [130], nh, nkv, window=50))
