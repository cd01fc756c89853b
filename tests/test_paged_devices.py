"""paged.py refuses tensors and streams of another device than the current one, whose
kernels could not reach them (no GPU needed: stand-ins)."""
from types import SimpleNamespace

import pytest
import torch

from rocmforge_amd import paged
from rocmforge_amd.ops import HipApiError

from .test_paged_tensors import LAUNCHES, OnGpu, gpu, i32

HERE = 1                             # the current device


@pytest.fixture(autouse=True)
def devices(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: HERE)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=0, device_index=HERE))


def on(block, index):
    for name, t in list(block._kept.items()):
        setattr(block, name, OnGpu(t.t, index))
    return block


def launch(kind, at=HERE, beside_at=HERE, stream=None, **fields):
    fn, make, beside = LAUNCHES[kind]
    block = on(make(), at)
    for n, v in fields.items():
        setattr(block, n, v)
    fn(*([block] if beside is None else [block, on(beside(), beside_at)]), stream=stream)


def nothing(kind):
    """A number that the library refuses."""
    return {"num_seqs" if kind == "plan" else "rows": -1}


@pytest.mark.parametrize("stream", [None, 0, SimpleNamespace(cuda_stream=0, device_index=HERE)])
@pytest.mark.parametrize("kind", LAUNCHES)
def test_another_device_than_the_current_one(rf, kind, stream):
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        launch(kind, at=0, beside_at=0, stream=stream)
    with pytest.raises(HipApiError):
        launch(kind, stream=stream, **nothing(kind))


@pytest.mark.parametrize("kind", LAUNCHES)
def test_a_stream_of_another_device(rf, kind):
    with pytest.raises(ValueError, match="stream of cuda:0"):
        launch(kind, stream=SimpleNamespace(cuda_stream=0, device_index=0))


@pytest.mark.parametrize("kind", LAUNCHES)
def test_tensors_of_two_devices(rf, kind):
    fn, make, beside = LAUNCHES[kind]
    for name in make()._kept:
        with pytest.raises(ValueError, match="cuda:1 and cuda:2"):
            launch(kind, **{name: OnGpu(make()._kept[name].t, 2)})
    if beside is not None:
        with pytest.raises(ValueError, match="cuda:1 and cuda:2"):
            launch(kind, beside_at=2)


def test_release_and_tables(rf):
    t = lambda index: [OnGpu(x.t, index) for x in (i32(2), i32(2), i32(2, 4), i32(8), i32(1))]
    with pytest.raises(ValueError):
        paged.release(*t(0), 2, 4, 16, 8)
    with pytest.raises(ValueError):
        paged.release(*t(HERE)[:4], OnGpu(i32(1).t, 2), 2, 4, 16, 8)
    with pytest.raises(HipApiError):
        paged.release(*t(HERE), -1, 4, 16, 8)
    with pytest.raises(ValueError):
        paged.rope_turns_table(gpu(64, dtype=torch.float64), 128, 1e6)
    with pytest.raises(HipApiError):
        paged.rope_turns_table(gpu(64, dtype=torch.float64, index=HERE), 7, 1e6)
