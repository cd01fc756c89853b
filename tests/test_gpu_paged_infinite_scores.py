"""Scores of -inf and +inf (rf_paged_attention_launch): as the softmax of them has it.
A row that sees keys but has only -inf for them is NaN; one that sees none is zero."""
import math

import pytest
import torch

from . import paged_util as P
from .test_gpu_paged_attn import Case

pytestmark = pytest.mark.gpu


def case(new, kv, d, window=0, scale=None, out_f32=0):
    """Dim 0 of q is 1, of K 0: K's dim 0 is the score's infinity."""
    c = Case([new, 2], [kv, 90], nh=8, nkv=2, d=d, window=window, scale=scale, out_f32=out_f32)
    c.q[:, ::d] = 1.0
    c.k[..., 0] = 0.0
    return c


def poison(c, to, value=-math.inf):
    for t in to:
        c.k[c.tab[0, t // 16].long(), t % 16, :, 0] = value


CASES = [(1, 60), (3, 700), (1, 9000), (40, 40), (100, 300), (33, 5000), (6, 3)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("new,kv", CASES)
def test_rows_of_nothing_but_minus_infinity(rf, dev, new, kv, d, window):
    c = case(new, kv, d, window)
    want = c.run().clone()
    poison(c, range(kv))
    got = c.run()
    empty = max(new - kv, 0)                             # rows in front of position 0
    assert bool((got[:empty] == 0).all()) and bool(got[empty:new].isnan().all())
    assert torch.equal(got[new:], want[new:])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv", [(2, 60), (3, 700), (2, 9000), (40, 100), (100, 300), (33, 5000)])
def test_some_keys_of_minus_infinity(rf, dev, new, kv, d):
    # half of the keys, whole tiles of them among these; every row keeps some
    c = case(new, kv, d)
    poison(c, [t for t in range(kv) if t % 2 or 64 <= t < 256])
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv", [(1, 60), (3, 700), (40, 100), (100, 300)])
def test_a_key_of_plus_infinity(rf, dev, new, kv, d):
    c = case(new, kv, d)
    want = c.run().clone()
    t = kv - new // 2 - 1
    poison(c, [t], math.inf)
    got = c.run()
    pos = torch.arange(kv - new, kv, device=P.DEV)
    assert bool(got[:new][pos >= t].isnan().all()) and torch.equal(got[:new][pos < t], want[:new][pos < t])
    assert torch.equal(got[new:], want[new:])


def test_fp32_outputs(rf, dev):
    c = case(2, 300, 128, out_f32=1)
    poison(c, range(300))
    got = c.run()
    assert bool(got[:2].isnan().all()) and bool(got[2:].isfinite().all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv", [(1, 60), (3, 700), (40, 100), (33, 5000)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_a_scale_of_zero(rf, dev, new, kv, d, value):
    # 0 times an infinite product is NaN; 0 times a finite one is 0
    c = case(new, kv, d, scale=0.0)
    c.check()
    poison(c, [kv // 2 - new // 2], value)
    got = c.run()
    pos = torch.arange(kv - new, kv, device=P.DEV)
    sees = pos >= kv // 2 - new // 2
    assert bool(sees.any()) and bool(got[:new][sees].isnan().all()) and bool(got[:new][~sees].isfinite().all())
    assert bool(got[new:].isfinite().all())
