"""The paged-cache launchers refuse what their declarations exclude, before any
HIP call (no GPU needed)."""
import ctypes

import pytest

from rocmforge_amd import paged
from rocmforge_amd.ops import HipApiError

A, ODD = 0x100000, 0x100008          # never dereferenced: validation rejects first


def cache(**kw):
    f = dict(k=A, v=A, page_stride=16 * 256, row_stride=256, head_stride=128, num_pages=4, page_size=16,
             num_kv_heads=2, head_dim=128)
    return paged.PagedCache(**{**f, **kw})


def plan(**kw):
    f = {n: A for n, t in paged.PagedPlan._fields_ if t is ctypes.c_void_p}
    f.update(num_seqs=2, max_blocks=4, page_size=16, max_rows=8, num_pages=8)
    return paged.PagedPlan(**{**f, **kw})


def rope(**kw):
    f = {n: A for n, t in paged.PagedRope._fields_ if t is ctypes.c_void_p}
    f.update(ld_q=512, ld_k=256, ld_v=256, ld_q16=512, rows=2, num_heads=4, rot_dim=128, neox=1, eps=1e-6,
             attn_factor=1.0)
    return paged.PagedRope(**{**f, **kw})


def attn(**kw):
    f = {n: A for n, t in paged.PagedAttention._fields_ if t is ctypes.c_void_p}
    f.update(workspace_bytes=1 << 30, ld_q=512, ld_out=512, num_seqs=2, max_blocks=4, rows=2, num_heads=4, max_new=1,
             window=0, out_f32=0, scale=0.1)
    return paged.PagedAttention(**{**f, **kw})


def rules(**kw):
    f = {n: A for n, t in paged.LogitsRules._fields_ if t is ctypes.c_void_p}
    f.update(out=2 * A, ld_logits=1000, ld_out=1000, ld_history=10, ld_allowed=32, rows=2, vocab=1000)
    return paged.LogitsRules(**{**f, **kw})


def refused(fn, *args):
    with pytest.raises(HipApiError) as e:
        fn(*args, 0)
    assert e.value.code == 1


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=ODD), dict(v=ODD), dict(page_stride=4100), dict(row_stride=0), dict(row_stride=(1 << 26) + 8),
             dict(head_stride=-128), dict(num_pages=0), dict(num_pages=1 << 28), dict(page_size=24), dict(page_size=4),
             dict(page_size=2048), dict(num_kv_heads=0), dict(head_dim=96)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_caches(rf, bad):
    refused(paged.rope_write, rope(), cache(**bad))
    refused(paged.attention, attn(), cache(**bad))


@pytest.mark.parametrize("bad", [{n: None} for n, t in paged.PagedPlan._fields_ if t is ctypes.c_void_p] + [
    dict(num_seqs=-1), dict(max_blocks=-1), dict(max_rows=-1), dict(page_size=0), dict(page_size=12),
    dict(num_pages=-1), dict(num_pages=1 << 27)])
def test_plans(rf, bad):
    refused(paged.plan, plan(**bad))


@pytest.mark.parametrize("bad", [{n: None} for n in ("q", "k", "v", "q16", "positions", "slots", "turns")] + [
    dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(q16=ODD), dict(q_norm=ODD), dict(k_norm=ODD), dict(ld_q=514),
    dict(ld_k=-4), dict(ld_v=255), dict(ld_q16=516), dict(ld_q16=504), dict(rows=-1), dict(rows=(1 << 23) + 1),
    dict(num_heads=0), dict(rot_dim=136), dict(rot_dim=12), dict(rot_dim=-8)])
def test_rotary_steps(rf, bad):
    refused(paged.rope_write, rope(**bad), cache())


@pytest.mark.parametrize("bad", [{n: None} for n in ("q", "out", "block_tables", "q_start", "kv_lens", "workspace")] + [
    dict(q=ODD), dict(out=ODD), dict(workspace=ODD), dict(ld_q=516), dict(ld_q=504), dict(ld_out=504), dict(rows=-1),
    dict(rows=(1 << 23) + 1), dict(num_seqs=-1), dict(max_blocks=-1), dict(max_blocks=1 << 27), dict(num_heads=0), dict(num_heads=3),
    dict(num_heads=256, ld_q=256 * 128, ld_out=256 * 128), dict(window=-1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(workspace_bytes=0)])
def test_attentions(rf, bad):
    refused(paged.attention, attn(**bad), cache())


def test_more_rows_and_heads_than_a_launch_counts(rf):
    refused(paged.attention, attn(rows=1 << 23, num_heads=32, ld_q=4096, ld_out=4096), cache())


@pytest.mark.parametrize("bad", [dict(logits=None), dict(out=None), dict(ld_logits=999), dict(ld_out=999),
                                 dict(rows=-1), dict(rows=65536), dict(vocab=-1), dict(bias_ids=None),
                                 dict(bias_start=None), dict(history=None), dict(prompt_lens=None),
                                 dict(total_lens=None), dict(ld_history=-1), dict(ld_allowed=31),
                                 dict(out=A, ld_out=1004)])
def test_rules(rf, bad):
    refused(paged.logits_rules, rules(**bad))


@pytest.mark.parametrize("args", [
    (None, 128, 1e6), (A, 0, 1e6), (A, 7, 1e6), (A, 258, 1e6), (A, 128, 1.0), (A, 128, float("nan")),
    (A, 128, 1e6, 3), (A, 128, 1e6, -1), (A, 128, 1e6, 1, 0.0), (A, 128, 1e6, 2, 4.0, 0.0),
    (A, 128, 1e6, 2, 4.0, 4096.0, 1.0, 32.0), (A, 128, 1e6, 2, 4.0, 4096.0, 32.0, 0.0)])
def test_turns_tables(rf, args):
    with pytest.raises(HipApiError):
        paged.rope_turns_table(*args, stream=0)


@pytest.mark.parametrize("i", range(5))
def test_releases(rf, i):
    args = [A] * 5
    args[i] = None
    refused(paged.release, *args, 2, 4, 16, 8)
    refused(paged.release, *[A] * 5, 2, 4, 20, 8)
    refused(paged.release, *[A] * 5, -1, 4, 16, 8)
    refused(paged.release, *[A] * 5, 2, -1, 16, 8)
    refused(paged.release, *[A] * 5, 2, 4, 16, -1)


def test_null_blocks(rf):
    assert rf.rf_paged_plan_launch(None, None) == 1
    assert rf.rf_paged_rope_write_launch(None, ctypes.byref(cache()), None) == 1
    assert rf.rf_paged_rope_write_launch(ctypes.byref(rope()), None, None) == 1
    assert rf.rf_paged_attention_launch(None, ctypes.byref(cache()), None) == 1
    assert rf.rf_paged_attention_launch(ctypes.byref(attn()), None, None) == 1
    assert rf.rf_logits_rules_launch(None, None) == 1


def test_nothing_to_do_is_no_error(rf):
    none = dict.fromkeys(n for n, t in paged.PagedPlan._fields_ if t is ctypes.c_void_p)
    paged.plan(plan(**none, num_seqs=0, max_rows=0), 0)
    paged.rope_write(rope(rows=0, q=None), cache(), 0)
    paged.attention(attn(rows=0, q=None), cache(), 0)
    paged.attention(attn(num_seqs=0, q=None), cache(), 0)
    paged.logits_rules(rules(rows=0, logits=None), 0)
    paged.logits_rules(rules(vocab=0, logits=None), 0)
    paged.release(None, None, None, None, None, 0, 4, 16, 8, 0)


@pytest.mark.parametrize("args", [(0, 1, 128), (4, 0, 128), (4, 3, 128), (4, 2, 96)])
def test_workspaces_of_no_launch(rf, args):
    assert paged.attention_workspace_bytes(*args) == 0


def test_tensors_of_the_host(rf):
    import torch
    t = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        plan(new_lens=t)
    p = plan()
    with pytest.raises(ValueError):
        p.kv_lens = t
    with pytest.raises(ValueError):
        paged.release(t, A, A, A, A, 1, 4, 16, 8, 0)
    with pytest.raises(ValueError):
        paged.rope_turns_table(t, 8, 1e4, stream=0)


def test_unknown_fields(rf):
    with pytest.raises(TypeError):
        paged.PagedCache(pages=3)
