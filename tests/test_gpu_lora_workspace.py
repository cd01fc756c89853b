"""One workspace, of a server's largest step, for all of its steps (rf_lora_add_launch)."""
import math

import pytest
import torch

from rocmforge_amd import lora

from . import paged_util as P
from .test_gpu_lora import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x16", [False, True])
def test_the_largest_step_s_workspace(rf, dev, x16):
    make = lambda new, seed=0: Case(new, [i % 3 for i in range(len(new))], [30, 9, 16], 32, k=2048, widths=(128, 64),
                                    x16=x16, seed=seed)
    most = make([1500, 1] + [700] * 3)
    n = lora.workspace_bytes(most.step, most.t)
    ws = torch.full((n // 4 + 64,), math.nan, device=P.DEV)
    for new in ([1], [5], [1] * 64, [1, 1, 40], [700, 60], [760, 20], [1400, 900, 300], [1500, 1] + [700] * 3):
        c = make(new, seed=len(new))
        assert lora.workspace_bytes(c.step, c.t) <= n
        c.step.workspace, c.step.workspace_bytes = ws, n
        c.check()
        assert bool(ws[n // 4:].isnan().all())


def test_as_many_adapters_as_an_integer_counts(rf, dev):
    # (the requests name the first ones; no others are looked at)
    c = Case([3, 40, 1, 2], [0, 1, -1, 2], [16, 5, 9])
    c.step.num_adapters = (1 << 31) - 1
    c.check()
