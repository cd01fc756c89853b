"""fp32 rows of any size through the adapters (rf_lora_add_launch), in tiles of few rows and of many: on a base of
zeros, so that nothing but the adapter's share is looked at."""
import pytest
import torch

from . import paged_util as P
from .test_gpu_lora import Case as Base

pytestmark = pytest.mark.gpu

# rows of a request each: dot products, tiles of 16, 32 and 64 rows
NEW = [[1], [4, 3], [5], [40], [1, 17, 2], [800], [2600]]


class Case(Base):
    def __init__(self, new, ranks=(16, 5, 11), max_rank=16, **kw):
        super().__init__(new, list(range(len(new))), list(ranks)[:len(new)], max_rank, **kw)
        for b in self.base:
            b.zero_()

    def check(self):
        super().check()
        live = slice(0, sum(self.new))
        for y in self.y:                                   # no row is lost: its values are of x's size
            top, x = y[live].double().abs().amax(1), self.x[live].double().abs().amax(1)
            assert bool((top > 0.01 * x).all())


@pytest.mark.parametrize("size", [1e-36, 1e-30, 1e-12, 1e-9, 1e-7, 1e-5, 1.0, 1e5, 1e9, 1e30, 1e36])
@pytest.mark.parametrize("new", NEW)
def test_sizes(rf, dev, new, size):
    Case(new, size=size).check()


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("max_rank,k", [(8, 264), (32, 2000), (64, 1000), (128, 520)])
def test_rows_of_many_sizes(rf, dev, new, max_rank, k):
    # from 1e-34 to 1e34, one behind the other
    c = Case(new, (max_rank, max_rank - 3, 7), max_rank, k=k, widths=(72,))
    c.x *= torch.pow(10.0, (torch.arange(c.x.shape[0], device=P.DEV) * 29 % 69 - 34).double()).float()[:, None]
    c.check()


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("at", [0, 100, 1023])
@pytest.mark.parametrize("outlier", [1e5, 1e7])
def test_outliers_that_an_adapter_does_not_look_at(rf, dev, new, at, outlier):
    # what is small beside the row's largest counts as it does alone: the smallest step is 2^-42 of that one or less, off by
    # 1.2e-6 of 1e7 at most, 2^-20 of most values: half of what the bound has for the sums
    c = Case(new, k=1024)
    c.x[:, at] = outlier
    c.a[0][:, :, at] = 0.0
    c.run()
    want, bound = c.want(0)
    n = sum(c.new)
    assert bool(((c.y[0].double() - want).abs() <= bound)[:n].all())
    assert bool((c.y[0][:n].abs().amax(1) > 0.01).all())


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("by", [10, 14])
def test_rows_that_climb(rf, dev, new, up, by):
    # x 2^0 .. 2^by along k and A as much smaller, so that all products count alike
    c = Case(new, k=2048)
    climb = torch.exp2(torch.linspace(0, by, 2048, device=P.DEV).round() * (1 if up else -1) + (0 if up else by))
    c.x *= climb
    c.a[0] /= climb.half()
    c.x[0, :700] = 0.0                                     # nothing at first
    c.run()
    want, bound = c.want(0)
    assert bool(((c.y[0].double() - want).abs() <= bound)[:sum(c.new)].all())


def test_a_row_is_the_same_size_in_any_company(rf, dev):
    # alone and among 39 others of its adapter: both finite, and both within their bounds
    c = Case([40], size=3e5)
    c.check()
    alone = Case([1], size=3e5)
    alone.x.copy_(c.x[7:8])
    alone.a[0].copy_(c.a[0])
    alone.b[0].copy_(c.b[0])
    alone.check()
    want, bound = alone.want(0)
    assert bool(((c.y[0][7:8].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("new", [[5], [40], [17, 30, 6], [800], [2600]])
@pytest.mark.parametrize("max_rank", [16, 32, 64, 128])
@pytest.mark.parametrize("looked_at", [False, True])
def test_values_that_do_not_fit_the_first_ones(rf, dev, new, max_rank, looked_at):
    # 10^3 to 10^30 times the others, in some rows, far behind where a wave begins; rows without one keep their bits
    c = Case(new, (max_rank, max_rank - 9, 7), max_rank, k=12288, widths=(72,))
    n, dims = sum(new), torch.arange(700, 12288, 1333, device=P.DEV)
    if not looked_at:
        c.a[0][:, :, dims] = 0.0
    c.run()
    want = c.y[0][:n].clone()
    rows = torch.arange(1, n, 3, device=P.DEV)
    size = torch.pow(10.0, 3 + (rows * 7 % 28 if looked_at else rows % 4).double()).float()
    c.x[rows, dims[rows % len(dims)]] = size
    c.run()
    value, bound = c.want(0)
    assert bool(((c.y[0].double() - value).abs() <= bound)[:n].all())
    others = torch.ones(n, dtype=torch.bool, device=P.DEV)
    others[rows] = False
    assert torch.equal(c.y[0][:n][others], want[others])
