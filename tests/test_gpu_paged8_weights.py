"""The weights of the attention over 8-bit pages: a row of one key, and far more small weights than one step of fp16
holds beside a large one."""
import math

import pytest
import torch

from . import paged_util as P
from .test_gpu_paged8_attn import Case


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("out_f32", [0, 1])
@pytest.mark.parametrize("new,kv", [(1, 1), (1, 300), (3, 40), (5, 5), (40, 700), (200, 200)])
def test_a_row_of_one_key_is_its_value(rf, dev, d, out_f32, new, kv):
    # o / l with o = w v exact: a reciprocal and a product, 2^-24 each; v itself is one of fp16's values
    c = Case([new], [kv], window=1, d=d, out_f32=out_f32, sizes=8.0)
    got = c.run()
    t = torch.arange(kv - new, kv, device=P.DEV)
    v = c.v[c.tab[0].long()[t // 16], t % 16].double().repeat_interleave(c.nh // c.v.shape[2], 1)
    assert bool(((got - v).abs() <= (v.abs() * 2.0 ** -23 if out_f32 else 0.0)).all())
    # the first row of a prompt sees one key without a window too
    c.args.window = 0
    if new == kv:
        assert bool(((c.run()[0] - v[0]).abs() <= (v[0].abs() * 2.0 ** -23 if out_f32 else 0.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("at", [0, 40000])
@pytest.mark.parametrize("lead", [14.0, 17.5, 19.0])
@pytest.mark.parametrize("new,nh", [(1, 8), (40, 8), (900, 64)])
def test_a_hundred_thousand_small_weights(rf, dev, d, at, lead, new, nh):
    """One key leads (an attention sink), and what the others hold together still is some thousandths: e^-17.5 is
    below half of fp16's smallest step."""
    kv = 100000
    c = Case([new], [kv], nh=nh, nkv=1, d=d, out_f32=1)
    c.p.k.fill_(0)
    c.p.ks.fill_(127)
    c.p.k[c.at(0, at)][0, 0] = 0x38                    # 1
    c.p.v &= 0x7f
    c.p.v.masked_fill_(c.p.v == 0x7f, 0)
    c.p.v[c.at(0, at)] = 0                             # the sink's own value
    c.take()
    c.q.zero_()
    c.q.view(-1, nh, d)[:, :, 0] = lead / c.scale
    got = c.run()
    leads = float(c.q[0, 0].double()) * c.scale
    t = torch.arange(kv, device=P.DEV)
    v = c.v[c.tab[0].long()[t // 16], t % 16][:, 0].double()
    sums = v.cumsum(0)[kv - new:]
    seen = torch.arange(kv - new, kv, device=P.DEV).double()[:, None]    # keys beside the one that leads
    want = sums / (math.exp(leads) + seen)
    # weights are off by 2^-11 of themselves, the one that leads (in the sum) and the others (in both), or by 2^-25, where a
    # row's largest is 2^6 at least; scores below 32 in fp32 by 2^-18, weights by as much; the sums of 100000 are
    # of 16 or more at once, 6250 times 2^-24 at most
    off = (2.0 ** -10 + 2.0 ** -11) * want + 2.0 ** -31 * sums
    assert bool(((got - want[:, None]).abs() <= off[:, None]).all()), ((got - want[:, None]).abs() / off[:, None]).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("jump", [20.0, 26.0, 30.0])
@pytest.mark.parametrize("half", [0, 1])
def test_a_maximum_that_leaps_within_a_tile(rf, dev, jump, half):
    """Heads of 256: one half of a tile of 64 positions leads the other by more than a weight's bits, whose weights are
    8 binary orders above the row's maximum so far."""
    c = Case([40], [840], nh=2, nkv=1, d=256, out_f32=1)
    c.p.k.fill_(0)
    c.p.ks.fill_(127)
    t = torch.arange(840, device=P.DEV)
    pg, row = c.tab[0].long()[t // 16], t % 16
    tile = 64 * 5 + 32 * torch.arange(2, device=P.DEV)
    score = torch.zeros(840, device=P.DEV)
    score[tile[1 - half]:tile[1 - half] + 32] = 5.0    # natural units: 2^7.2
    score[tile[half] + 9] = 5.0 + jump * math.log(2)
    codes = (score.view(-1, 1) * torch.tensor([[1.0, 0.0]], device=P.DEV)).half()
    # a score is q . k with q = 1 / scale in two dims: an e4m3 value and what it leaves
    first = codes[:, 0].to(torch.float8_e4m3fn)
    rest = (score - first.float()).to(torch.float8_e4m3fn)
    c.p.k[pg, row, 0, 0], c.p.k[pg, row, 0, 1] = first.view(torch.uint8), rest.view(torch.uint8)
    c.p.v &= 0x7f
    c.p.v.masked_fill_(c.p.v == 0x7f, 0)
    c.p.v[pg[tile[half] + 9], row[tile[half] + 9]] = 0           # what leads holds nothing
    c.take()
    c.q.zero_()
    c.q.view(-1, 2, 256)[:, :, :2] = 1 / c.scale
    got = c.run()
    x = c.k[pg, row][:, 0, :2].double().sum(1)
    v = c.v[pg, row][:, 0].double()
    w = (x - x.max()).exp()
    for i in (0, 39):
        n = 800 + i + 1
        want = (w[:n] @ v[:n]) / w[:n].sum()
        # as above: 2^-31 of the largest for each weight (the 32 of 2^-jump below it, and 2^-7 of these for the others)
        off = (2.0 ** -10 + 2.0 ** -11) * want + 2.0 ** -31 * v[:n].sum(0)
        assert bool(((got[i] - want).abs() <= off).all()), ((got[i] - want).abs() / off).max().item()


BEHIND = [(4, 498), (3, 130), (6, 34), (100, 120), (64, 708), (300, 2004), (130, 300)]


def first_of_the_last_block(new, kv):
    """Position, and how many of the new rows see it or one behind it."""
    block = 16 * ((kv - 1) // 16)
    return block, kv - block


def test_some_rows_are_in_front_of_the_last_block():
    for new, kv in BEHIND:
        assert 0 < first_of_the_last_block(new, kv)[1] < new


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("new,kv", BEHIND)
def test_large_keys_behind_some_rows(rf, dev, d, window, new, kv):
    """Codes and exponents that only the last rows see: all others keep their bits."""
    c = Case([new], [kv], window=window, d=d)
    block, seen = first_of_the_last_block(new, kv)
    want = c.run().half().view(torch.int16).clone()
    pg, _ = c.at(0, block)
    for t in range(block, kv):
        c.p.k[c.at(0, t)] = 0x7e
        c.p.v[c.at(0, t)] = 0xfe
    c.p.ks[pg], c.p.vs[pg] = 127 + 3, 134
    got = c.run().half().view(torch.int16)
    assert torch.equal(got[:new - seen], want[:new - seen])
    assert bool((got[new - seen:] != want[new - seen:]).flatten(1).any(1).all())
