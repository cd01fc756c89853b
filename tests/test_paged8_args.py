"""The launchers of 8-bit pages and of low-rank adapters refuse what their declarations
exclude, before any HIP call (no GPU needed)."""
import ctypes

import pytest

from rocmforge_amd import lora, paged

from .test_paged_args import A, ODD, attn, cache, refused, rope


def cache8(**kw):
    f = dict(k=A, v=A, k_scale=A + 1, v_scale=A + 3, page_stride=16 * 256, row_stride=256, head_stride=128, num_pages=4,
             page_size=16, num_kv_heads=2, head_dim=128)
    return paged.PagedCache8(**{**f, **kw})


def read(**kw):
    f = dict(k=A, v=A, block_tables=A, row_start=A, first=A, ld_out=256, num_seqs=2, max_blocks=4, rows=2)
    return paged.PagedRead(**{**f, **kw})


def step(**kw):
    f = dict(x=A, adapters=A, q_start=A, ranks=A, scales=A, ld_x=256, rows=2, num_seqs=2, num_adapters=3, max_rank=16,
             in_dim=256, x_f16=0)
    return lora.LoraStep(**{**f, **kw})


def target(**kw):
    f = dict(a=A, b=A, base=A, y=2 * A, a_stride=16 * 256, b_stride=16 * 512, ld_base=512, ld_y=512, out_dim=512)
    return lora.LoraTarget(**{**f, **kw})


BAD_CACHE = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=ODD), dict(v=ODD),
             dict(page_stride=4104), dict(row_stride=0), dict(row_stride=(1 << 27) + 16), dict(head_stride=-128),
             dict(head_stride=136), dict(num_pages=0), dict(num_pages=1 << 28), dict(page_size=24), dict(page_size=4),
             dict(page_size=2048), dict(num_kv_heads=0), dict(head_dim=96)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_caches(rf, bad):
    refused(paged.rope_write8, rope(), cache8(**bad))
    refused(paged.attention8, attn(), cache8(**bad))
    refused(paged.read8, read(), cache8(**bad))


@pytest.mark.parametrize("bad", [{n: None} for n in ("q", "k", "v", "q16", "positions", "slots", "turns")] + [
    dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(q16=ODD), dict(q_norm=ODD), dict(k_norm=ODD), dict(ld_q=514),
    dict(ld_k=-4), dict(ld_v=255), dict(ld_q16=516), dict(ld_q16=504), dict(rows=-1), dict(rows=(1 << 23) + 1),
    dict(num_heads=0), dict(rot_dim=136), dict(rot_dim=12), dict(rot_dim=-8)])
def test_rotary_steps(rf, bad):
    refused(paged.rope_write8, rope(**bad), cache8())


@pytest.mark.parametrize("bad", [{n: None} for n in ("q", "out", "block_tables", "q_start", "kv_lens", "workspace")] + [
    dict(q=ODD), dict(out=ODD), dict(workspace=ODD), dict(ld_q=516), dict(ld_q=504), dict(ld_out=504), dict(rows=-1),
    dict(rows=(1 << 23) + 1), dict(num_seqs=-1), dict(max_blocks=-1), dict(max_blocks=1 << 27), dict(num_heads=0),
    dict(num_heads=3), dict(num_heads=256, ld_q=256 * 128, ld_out=256 * 128), dict(window=-1),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace_bytes=0),
    dict(rows=1 << 23, num_heads=32, ld_q=4096, ld_out=4096)])
def test_attentions(rf, bad):
    refused(paged.attention8, attn(**bad), cache8())


@pytest.mark.parametrize("bad", [dict(block_tables=None), dict(row_start=None), dict(k=ODD), dict(v=ODD), dict(ld_out=252),
                                 dict(ld_out=260), dict(rows=-1), dict(rows=(1 << 27) + 1), dict(num_seqs=-1),
                                 dict(max_blocks=-1)])
def test_reads(rf, bad):
    refused(paged.read8, read(**bad), cache8())


@pytest.mark.parametrize("bad", [{n: None} for n in ("x", "adapters", "q_start", "ranks", "scales")] + [
    dict(x=ODD), dict(ld_x=252), dict(ld_x=258), dict(x_f16=1, ld_x=260), dict(rows=-1), dict(rows=(1 << 23) + 1),
    dict(num_seqs=-1), dict(num_adapters=-1), dict(max_rank=0), dict(max_rank=12), dict(max_rank=136), dict(in_dim=0),
    dict(in_dim=252), dict(in_dim=(1 << 20) + 8)])
def test_adapter_steps(rf, bad):
    refused(lora.add, step(**bad), target())


@pytest.mark.parametrize("bad", [{n: None} for n in ("a", "b", "base", "y")] + [
    dict(a=ODD), dict(b=ODD), dict(base=ODD), dict(y=ODD), dict(a_stride=16 * 256 - 8), dict(a_stride=16 * 256 + 4),
    dict(b_stride=16 * 512 - 8), dict(b_stride=16 * 512 + 4), dict(ld_base=508), dict(ld_y=508), dict(ld_base=514),
    dict(ld_y=514), dict(out_dim=0), dict(out_dim=510), dict(out_dim=(1 << 20) + 4), dict(y=A, ld_y=516)])
def test_adapter_targets(rf, bad):
    refused(lora.add, step(), target(**bad))
    refused(lora.add, step(), [target(), target(**bad)])


def test_workspaces(rf):
    big = dict(rows=100, ld_x=256)
    n = lora.workspace_bytes(step(**big), target())
    assert n > 0 and lora.workspace_bytes(step(**big), [target()] * 3) > n
    assert lora.workspace_bytes(step(), target()) == 0                   # few rows: one launch
    for bad in (dict(), dict(workspace=A), dict(workspace=A, workspace_bytes=n - 1), dict(workspace=ODD, workspace_bytes=n)):
        assert rf.rf_lora_add_launch(ctypes.byref(step(**big, **bad)), ctypes.byref(target()), 1, None) == 1
    assert lora.workspace_bytes(step(rows=-1), target()) == 0
    assert lora.workspace_bytes(step(**big), []) == 0


def test_numbers_of_targets(rf):
    refused(lora.add, step(), [])
    refused(lora.add, step(), [target()] * 4)


def test_null_blocks(rf):
    c8, st, t = cache8(), step(), target()
    for f, block in (("rf_paged_rope_write8_launch", rope()), ("rf_paged_attention8_launch", attn()),
                     ("rf_paged_read8_launch", read())):
        assert getattr(rf, f)(None, ctypes.byref(c8), None) == 1
        assert getattr(rf, f)(ctypes.byref(block), None, None) == 1
    assert rf.rf_lora_add_launch(None, ctypes.byref(t), 1, None) == 1
    assert rf.rf_lora_add_launch(ctypes.byref(st), None, 1, None) == 1


def test_nothing_to_do_is_no_error(rf):
    paged.rope_write8(rope(rows=0, q=None), cache8(), 0)
    paged.attention8(attn(rows=0, q=None), cache8(), 0)
    paged.attention8(attn(num_seqs=0, q=None), cache8(), 0)
    paged.read8(read(rows=0, row_start=None), cache8(), 0)
    paged.read8(read(num_seqs=0, row_start=None), cache8(), 0)
    paged.read8(read(k=None, v=None, row_start=None), cache8(), 0)
    lora.add(step(rows=0, x=None), target(y=None), 0)
    lora.add(step(num_seqs=0, x=None), target(y=None), 0)


def test_pages_of_the_other_kind(rf):
    for fn, block, other in ((paged.rope_write, rope(), cache8()), (paged.attention, attn(), cache8()),
                             (paged.rope_write8, rope(), cache()), (paged.attention8, attn(), cache()),
                             (paged.read8, read(), cache())):
        with pytest.raises(TypeError):
            fn(block, other, 0)
