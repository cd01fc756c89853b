"""What lies behind a row's position, or in front of its window, changes none of the
row's bits (rf_paged_attention_launch): large finite K and V there, seen by other
rows of its tile."""
import pytest
import torch

from . import paged_util as P
from .test_gpu_paged_attn import Case

pytestmark = pytest.mark.gpu


def bits(c):
    return c.run().half().view(torch.int16).clone()      # (live() is of fp16 values)


def lead(c, t, size):
    """K and V of request 0's position t: K along one of the query rows that see it."""
    row, group = min(t - (c.kv[0] - c.new[0]), c.new[0] - 1), c.nh // c.k.shape[2]
    at = c.tab[0, t // 16].long(), t % 16
    q = c.q[max(row, 0)].reshape(-1, group, c.d)[:, 0]
    c.k[at] = (size * q.float()).half()
    c.v[at] = 60000.0


CASES = [(4, 500, 0), (3, 130, 0), (100, 100, 0), (128, 128, 0), (64, 700, 0), (300, 2000, 0), (130, 300, 60)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv,window", CASES)
@pytest.mark.parametrize("size", [0.3, 1.0, 3.0, 40.0])
def test_keys_behind_a_row(rf, dev, new, kv, window, d, size):
    for back in sorted({1, new // 2, new - 1}):          # the last `back` rows see it
        c = Case([new], [kv], window=window, d=d)
        want = bits(c)
        lead(c, kv - back, size)
        got = bits(c)
        assert torch.equal(got[:new - back], want[:new - back]), back
        assert not torch.equal(got[new - back:], want[new - back:])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,kv,window", [(4, 500, 90), (128, 500, 100), (200, 200, 70), (64, 1000, 300)])
@pytest.mark.parametrize("size", [0.3, 1.0, 3.0, 40.0])
def test_keys_in_front_of_a_window(rf, dev, new, kv, window, d, size):
    for row in sorted({0, new // 2, new - 2}):           # the last row whose window has it
        t = kv - new + row - window + 1
        if t < 0:
            continue
        c = Case([new], [kv], window=window, d=d)
        want = bits(c)
        lead(c, t, size)
        got = bits(c)
        assert torch.equal(got[row + 1:], want[row + 1:]), row
        assert not torch.equal(got[:row + 1], want[:row + 1])
