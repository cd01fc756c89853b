"""The current stream's handle where torch has no call that gives it without an object around it (no GPU needed:
stand-ins)."""
from types import SimpleNamespace

import pytest
import torch

from rocmforge_amd import paged
from rocmforge_amd.ops import HipApiError

from .test_paged_tensors import LAUNCHES

HERE = 0


@pytest.fixture(autouse=True)
def devices(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: HERE)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: SimpleNamespace(cuda_stream=77, device_index=HERE))
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)


def test_the_handle():
    assert paged._stream(None, None) == 77 and paged._stream(None, HERE) == 77
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        paged._stream(None, 1)


@pytest.mark.parametrize("kind", LAUNCHES)
def test_launches(rf, kind):
    fn, make, beside = LAUNCHES[kind]
    block = make()
    setattr(block, "num_seqs" if kind == "plan" else "rows", -1)         # (refused before any launch)
    with pytest.raises(HipApiError):
        fn(*([block] if beside is None else [block, beside()]))
