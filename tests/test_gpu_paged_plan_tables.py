"""Entries of a block table that name no page: the plan's slots of rows there lie
outside the cache, never in another request's page."""
import pytest
import torch

from .test_gpu_paged_plan import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [0, 9000])              # (padding rows: the second launch writes them)
@pytest.mark.parametrize("page", [8, 16, 1024])
def test_entries_that_name_no_page(rf, dev, page, rows):
    wrap = 2 ** 32 // page                               # entry * page is a multiple of 2^32 more or less
    entries = [wrap, wrap + 1, -wrap, 1 - wrap, 2 ** 31 - 1, -2 ** 31, -1, 1000, 2 ** 31 // page, -2 ** 31 // page]
    entries = [e for e in entries if -2 ** 31 <= e < 2 ** 31]
    s = Step([1] * len(entries), [3] * len(entries), page, free=0, max_rows=len(entries) + rows)
    width = s.args.max_blocks
    tab = s.t["tab"].view(-1, width)
    tab[:, 0] = torch.tensor(entries, dtype=torch.int32)
    for r, e in enumerate(entries):
        slot = e * page + 3
        s.host["slot"][r] = slot if -2 ** 31 <= slot < 2 ** 31 else -1
        s.host["tab"][r][0] = e
    s.check()
    cache = s.num_pages * page
    assert not any(0 <= v < cache for v in s.t["slot"].tolist())
