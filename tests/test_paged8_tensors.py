"""paged.py and lora.py look at the tensors of 8-bit pages and of adapters before they
launch on them (no GPU needed: stand-ins with a GPU tensor's properties)."""
from types import SimpleNamespace

import pytest
import torch

from rocmforge_amd import lora, paged
from rocmforge_amd.ops import HipApiError

from .test_paged_tensors import OnGpu, attn, f16, f32, gpu, i32, pointers, rope, wrong

u8 = lambda *s: gpu(*s, dtype=torch.uint8)


def cache8(**kw):
    f = dict(k=u8(4, 16, 2, 128), v=u8(4, 16, 2, 128), k_scale=u8(4, 1, 2), v_scale=u8(4, 1, 2), page_stride=4096,
             row_stride=256, head_stride=128, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128)
    return paged.PagedCache8(**{**f, **kw})


def read(**kw):
    f = dict(k=f16(8, 256), v=f16(8, 256), block_tables=i32(2, 4), row_start=i32(3), first=i32(2), ld_out=256,
             num_seqs=2, max_blocks=4, rows=8)
    return paged.PagedRead(**{**f, **kw})


def step(**kw):
    f = dict(x=f32(2, 256), adapters=i32(2), q_start=i32(3), ranks=i32(3), scales=f32(3), ld_x=256, rows=2, num_seqs=2,
             num_adapters=3, max_rank=16, in_dim=256, x_f16=0)
    return lora.LoraStep(**{**f, **kw})


def target(**kw):
    f = dict(a=f16(3, 16, 256), b=f16(3, 512, 16), base=f32(2, 512), y=f32(2, 512), a_stride=4096, b_stride=8192,
             ld_base=512, ld_y=512, out_dim=512)
    return lora.LoraTarget(**{**f, **kw})


@pytest.fixture(autouse=True)
def no_device_calls(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


CALLS = {"rope": lambda **kw: paged.rope_write8(rope(), cache8(**kw), stream=0),
         "attn": lambda **kw: paged.attention8(attn(), cache8(**kw), stream=0),
         "read": lambda **kw: paged.read8(read(), cache8(**kw), stream=0)}


@pytest.mark.parametrize("call", CALLS)
def test_types_of_pages(rf, call):
    for name in ("k", "v", "k_scale", "v_scale"):
        for t in wrong(cache8()._kept[name]):
            with pytest.raises(ValueError, match=name):
                CALLS[call](**{name: t})
    with pytest.raises(HipApiError):
        CALLS[call](num_pages=-1)


def test_types_that_pass(rf):
    for t in (torch.float8_e4m3fn, torch.int8):
        with pytest.raises(HipApiError):
            CALLS["read"](k=gpu(4, 16, 2, 128, dtype=t), num_pages=-1)
    with pytest.raises(HipApiError):
        CALLS["read"](k_scale=gpu(4, 1, 2, dtype=torch.float8_e8m0fnu), num_pages=-1)
    for t in (torch.float8_e5m2, torch.float8_e4m3fnuz):
        with pytest.raises(ValueError, match="k"):
            CALLS["read"](k=gpu(4, 16, 2, 128, dtype=t))


def test_strides_of_pages(rf):
    by_head = OnGpu(torch.zeros(4, 2, 16, 128, dtype=torch.uint8).transpose(1, 2))
    with pytest.raises(ValueError, match="PagedCache8.v"):
        CALLS["attn"](v=by_head)
    with pytest.raises(ValueError, match="k_scale"):
        CALLS["attn"](k_scale=OnGpu(torch.zeros(2, 1, 4, dtype=torch.uint8).permute(2, 1, 0)))


@pytest.mark.parametrize("make,call", [(read, lambda b: paged.read8(b, cache8(), stream=0)),
                                       (step, lambda b: lora.add(b, target(), stream=0)),
                                       (target, lambda b: lora.add(step(), b, stream=0))])
def test_types_and_strides(rf, make, call):
    for name in pointers(make()):
        if name == "workspace":                      # (of any type)
            continue
        good = make()._kept[name]
        for t in wrong(good):
            with pytest.raises(ValueError, match=name):
                call(make(**{name: t}))
        every_other = torch.zeros(*good.shape[:-1], 2 * good.shape[-1], dtype=good.dtype)[..., ::2]
        with pytest.raises(ValueError, match=name):
            call(make(**{name: OnGpu(every_other)}))
        with pytest.raises(ValueError, match="not on a GPU"):
            make(**{name: torch.zeros(good.shape, dtype=good.dtype)})


def test_x_has_the_type_that_is_said(rf):
    with pytest.raises(ValueError, match="x"):
        lora.add(step(x=f16(2, 256)), target(), stream=0)
    with pytest.raises(ValueError, match="x"):
        lora.add(step(x_f16=1), target(), stream=0)
    with pytest.raises(HipApiError):
        lora.add(step(x=f16(2, 256), x_f16=1, rows=-1), target(), stream=0)


def test_devices(rf, monkeypatch):
    for call in CALLS.values():
        with pytest.raises(ValueError, match="cuda:0 and cuda:1"):
            call(v_scale=gpu(4, 1, 2, dtype=torch.uint8, index=1))
    with pytest.raises(ValueError, match="cuda:0 and cuda:1"):
        lora.add(step(), [target(), target(y=gpu(2, 512, index=1))], stream=0)
    with pytest.raises(ValueError, match="stream of cuda:1"):
        lora.add(step(), target(), stream=SimpleNamespace(cuda_stream=0, device_index=1))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        lora.add(step(), target(), stream=0)
    for call in CALLS.values():
        with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
            call()
