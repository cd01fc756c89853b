"""paged.py looks at the tensors that it is given before it launches on them: types,
strides and pointers (no GPU needed: stand-ins with a GPU tensor's properties)."""
import ctypes
import math

import pytest
import torch

from rocmforge_amd import paged
from rocmforge_amd.ops import HipApiError

A = 0x100000                         # never dereferenced


class OnGpu:
    """What paged.py asks of a tensor, of a host tensor's shape, strides and type."""
    is_cuda = True

    def __init__(self, t, index=0):
        self.t, self.device = t, torch.device("cuda", index)
        self.dtype, self.shape = t.dtype, t.shape

    def data_ptr(self):
        return A

    def stride(self):
        return self.t.stride()


def gpu(*shape, dtype=torch.float32, index=0):
    return OnGpu(torch.zeros(*shape, dtype=dtype), index)


i32 = lambda *s: gpu(*s, dtype=torch.int32)
f16 = lambda *s: gpu(*s, dtype=torch.float16)
f32 = lambda *s: gpu(*s)


def cache(**kw):
    f = dict(k=f16(4, 16, 2, 128), v=f16(4, 16, 2, 128), page_stride=4096, row_stride=256, head_stride=128,
             num_pages=4, page_size=16, num_kv_heads=2, head_dim=128)
    return paged.PagedCache(**{**f, **kw})


def plan(**kw):
    f = dict(new_lens=i32(2), ctx_in=i32(2), ctx_out=i32(2), free_pages=i32(8), free_in=i32(1), free_out=i32(1),
             block_tables=i32(2, 4), q_start=i32(3), kv_lens=i32(2), positions=i32(8), slots=i32(8), num_seqs=2,
             max_blocks=4, page_size=16, max_rows=8, num_pages=8)
    return paged.PagedPlan(**{**f, **kw})


def rope(**kw):
    f = dict(q=f32(2, 512), k=f32(2, 256), v=f32(2, 256), q_norm=f32(128), k_norm=f32(128), q16=f16(2, 512),
             positions=i32(2), slots=i32(2), turns=gpu(64, dtype=torch.float64), ld_q=512, ld_k=256, ld_v=256,
             ld_q16=512, rows=2, num_heads=4, rot_dim=128, neox=1, eps=1e-6, attn_factor=1.0)
    return paged.PagedRope(**{**f, **kw})


def attn(**kw):
    f = dict(q=f16(2, 512), out=f16(2, 512), block_tables=i32(2, 4), q_start=i32(3), kv_lens=i32(2),
             workspace=gpu(1 << 20, dtype=torch.uint8), workspace_bytes=1 << 30, ld_q=512, ld_out=512, num_seqs=2,
             max_blocks=4, rows=2, num_heads=4, max_new=1, window=0, out_f32=0, scale=0.1)
    return paged.PagedAttention(**{**f, **kw})


def rules(**kw):
    f = dict(logits=f32(2, 1000), out=f32(2, 1000), history=i32(2, 10), prompt_lens=i32(2), total_lens=i32(2),
             repetition=f32(2), frequency=f32(2), presence=f32(2), bias_start=i32(3), bias_ids=i32(5),
             bias_values=f32(5), allowed=i32(2, 32), ld_logits=1000, ld_out=1000, ld_history=10, ld_allowed=32, rows=2,
             vocab=1000)
    return paged.LogitsRules(**{**f, **kw})


# each launch, its own block and the one beside it
LAUNCHES = {"plan": (paged.plan, plan, None), "rope": (paged.rope_write, rope, cache),
            "attn": (paged.attention, attn, cache), "rules": (paged.logits_rules, rules, None)}


def launch(kind, block):
    fn, _, beside = LAUNCHES[kind]
    fn(*([block] if beside is None else [block, beside()]), stream=0)


@pytest.fixture(autouse=True)
def no_device_calls(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def pointers(block):
    return [n for n, t in block._fields_ if t is ctypes.c_void_p]


def wrong(t):
    """Tensors of the same shape and other types."""
    for dtype in (torch.int64, torch.bfloat16, torch.float32, torch.float16, torch.int32, torch.float64):
        if dtype != t.dtype:
            yield OnGpu(torch.zeros(t.shape, dtype=dtype))


@pytest.mark.parametrize("kind", LAUNCHES)
def test_types(rf, kind):
    make = LAUNCHES[kind][1]
    for name in pointers(make()):
        if name == "workspace":
            continue
        good = make()._kept[name]
        for t in wrong(good):
            with pytest.raises(ValueError, match=name):
                launch(kind, make(**{name: t}))


@pytest.mark.parametrize("name", ["k", "v"])
def test_types_of_pages(rf, name):
    for t in wrong(f16(4, 16, 2, 128)):
        for kind, step in (("rope", rope), ("attn", attn)):
            with pytest.raises(ValueError, match=name):
                LAUNCHES[kind][0](step(), cache(**{name: t}), stream=0)


def good_ones_reach_the_library(kind, **kw):
    # (refused there, before any launch: a negative number of rows or requests)
    fn, make, beside = LAUNCHES[kind]
    block = make(**kw)
    block.__setattr__("num_seqs" if kind == "plan" else "rows", -1)
    with pytest.raises(HipApiError):
        launch(kind, block)


@pytest.mark.parametrize("kind", LAUNCHES)
def test_right_tensors(rf, kind):
    good_ones_reach_the_library(kind)


def test_bits_of_fp16_and_masks(rf):
    bits = lambda *s: gpu(*s, dtype=torch.int16)
    good_ones_reach_the_library("attn", q=bits(2, 512), out=bits(2, 512))
    good_ones_reach_the_library("rope", q16=gpu(2, 512, dtype=torch.uint16))
    good_ones_reach_the_library("rules", allowed=gpu(2, 32, dtype=torch.uint32))


def test_the_output_has_the_type_that_is_asked_for(rf):
    good_ones_reach_the_library("attn", out=f32(2, 512), out_f32=1)
    with pytest.raises(ValueError, match="out"):
        launch("attn", attn(out_f32=1))
    a = attn()
    good_ones_reach_the_library("attn")
    a.out_f32 = 1                                        # (looked at again after a change)
    with pytest.raises(ValueError, match="out"):
        launch("attn", a)


@pytest.mark.parametrize("kind", LAUNCHES)
def test_strides(rf, kind):
    make = LAUNCHES[kind][1]
    for name in pointers(make()):
        good = make()._kept[name].t
        every_other = torch.zeros(*good.shape[:-1], 2 * good.shape[-1], dtype=good.dtype)[..., ::2]
        if good.shape[-1] == 1:                          # (one element lies anywhere)
            good_ones_reach_the_library(kind, **{name: OnGpu(every_other)})
            continue
        with pytest.raises(ValueError, match=name):
            launch(kind, make(**{name: OnGpu(every_other)}))
        if good.dim() == 2:
            wide = torch.zeros(good.shape[0], good.shape[1] + 8, dtype=good.dtype)[:, :good.shape[1]]
            turned = torch.zeros(good.shape[1], good.shape[0], dtype=good.dtype).t()
            for t in (wide, turned):
                with pytest.raises(ValueError, match=name):
                    launch(kind, make(**{name: OnGpu(t)}))


def test_rows_further_apart(rf):
    wide = lambda dtype: OnGpu(torch.zeros(2, 640, dtype=dtype)[:, :512])
    good_ones_reach_the_library("rope", q=wide(torch.float32), ld_q=640, q16=wide(torch.float16), ld_q16=640)
    good_ones_reach_the_library("attn", q=wide(torch.float16), ld_q=640)
    heads = OnGpu(torch.zeros(2, 5, 128, dtype=torch.float16)[:, :4])
    good_ones_reach_the_library("attn", q=heads, ld_q=640)
    with pytest.raises(ValueError):
        launch("attn", attn(q=OnGpu(torch.zeros(2, 4, 160, dtype=torch.float16)[..., :128]), ld_q=640))
    one = OnGpu(torch.zeros(1, 700, dtype=torch.float16)[:, :512])
    good_ones_reach_the_library("attn", q=one)           # one row is no distance away from another
    good_ones_reach_the_library("plan", block_tables=i32(8))


def test_pages_in_either_order(rf):
    by_head = OnGpu(torch.zeros(4, 2, 16, 128, dtype=torch.float16).transpose(1, 2))
    ok = cache(k=by_head, v=by_head, row_stride=128, head_stride=2048)
    with pytest.raises(HipApiError):
        paged.attention(attn(rows=-1), ok, stream=0)
    with pytest.raises(ValueError, match="v"):
        paged.attention(attn(), cache(v=by_head), stream=0)
    one_page = OnGpu(torch.zeros(9, 16, 2, 128, dtype=torch.float16)[::9])
    with pytest.raises(HipApiError):
        paged.attention(attn(rows=-1), cache(k=f16(1, 16, 2, 128), v=one_page, num_pages=1), stream=0)
    dims_apart = OnGpu(torch.zeros(4, 16, 128, 2, dtype=torch.float16).transpose(2, 3))
    with pytest.raises(ValueError):
        paged.attention(attn(), cache(k=dims_apart, v=dims_apart), stream=0)


def test_numbers_are_no_tensors(rf):
    with pytest.raises(ValueError):
        plan(num_seqs=i32(1))
    a = attn()
    with pytest.raises(ValueError):
        a.scale = f32(1)
    assert math.isclose(a.scale, 0.1, rel_tol=1e-6)


def test_a_refused_tensor_changes_nothing(rf):
    p = plan()
    kept = p._kept["kv_lens"]
    with pytest.raises(ValueError):
        p.kv_lens = torch.zeros(2, dtype=torch.int32)    # of the host
    assert p.kv_lens == A and p._kept["kv_lens"] is kept


def test_a_replaced_tensor_is_let_go(rf):
    p = plan(new_lens=gpu(2, dtype=torch.int64))
    p.new_lens = 2 * A
    assert "new_lens" not in p._kept and p.new_lens == 2 * A
    p.num_seqs = -1
    with pytest.raises(HipApiError):
        launch("plan", p)


def test_release(rf):
    good = [i32(2), i32(2), i32(2, 4), i32(8), i32(1)]
    for i in range(5):
        bad = list(good)
        for t in wrong(good[i]):
            bad[i] = t
            with pytest.raises(ValueError):
                paged.release(*bad, 2, 4, 16, 8, stream=0)
    with pytest.raises(ValueError):
        paged.release(good[0], good[1], i32(2, 5), good[3], good[4], 2, 4, 16, 8, stream=0)
    with pytest.raises(HipApiError):
        paged.release(*good, -1, 4, 16, 8, stream=0)


def test_tables_of_turns(rf):
    with pytest.raises(ValueError):
        paged.rope_turns_table(f32(64), 128, 1e6, stream=0)
    with pytest.raises(ValueError):
        paged.rope_turns_table(gpu(64, dtype=torch.float64), 128, 1e6, freq_scale=gpu(64, dtype=torch.float64), stream=0)
    with pytest.raises(HipApiError):
        paged.rope_turns_table(gpu(64, dtype=torch.float64), 7, 1e6, freq_scale=f32(64), stream=0)
