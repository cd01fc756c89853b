"""Several requests on a paged cache -- the Python face of the rf_paged_* and
rf_logits_rules launchers in include/rocmforge_cdna4.h, which state what each
computes and which arguments it takes.

A server keeps, per layer, a PagedCache on its K and V pages and the argument
blocks on its buffers, and runs a step of a batch as

    plan(p)                       pages, block tables, row ranges, positions and slots
    per layer:
        rope_write(r, cache)      norms, RoPE, fp16 q, k and v into their slots
        attention(a, cache)       the new rows over their requests' pages
    logits_rules(l)               before a token is picked

with release() for requests that ended.  The argument blocks are the C
structs; pointer fields take device addresses, torch tensors of the GPU (kept
alive by the block) or None.  Launches go to the given stream, else to torch's current
one, and raise ops.HipApiError where the library refuses the arguments.
"""
from __future__ import annotations

import ctypes

from ._lib import load
from .ops import HipApiError

ROPE_PLAIN, ROPE_LINEAR, ROPE_YARN = 0, 1, 2

_vp, _i32, _i64, _f, _sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class _Block(ctypes.Structure):
    def __init__(self, **fields):
        super().__init__()
        types = dict(self._fields_)
        unknown = sorted(set(fields) - set(types))
        if unknown:
            raise TypeError(f"{type(self).__name__} has no field {', '.join(unknown)}")
        for name, value in fields.items():
            setattr(self, name, value)

    def __setattr__(self, name, value):
        if hasattr(value, "data_ptr"):
            self.__dict__.setdefault("_kept", {})[name] = value
            value = _addr(value)
        super().__setattr__(name, value)


class PagedCache(_Block):
    """K and V pages of one layer (rf_paged_cache)."""
    _fields_ = [("k", _vp), ("v", _vp), ("page_stride", _i64), ("row_stride", _i64), ("head_stride", _i64),
                ("num_pages", _i32), ("page_size", _i32), ("num_kv_heads", _i32), ("head_dim", _i32)]


class PagedPlan(_Block):
    """The plan of a step (rf_paged_plan)."""
    _fields_ = [(n, _vp) for n in ("new_lens", "ctx_in", "ctx_out", "free_pages", "free_in", "free_out",
                                   "block_tables", "q_start", "kv_lens", "positions", "slots")] + \
               [(n, _i32) for n in ("num_seqs", "max_blocks", "page_size", "max_rows", "num_pages")]


class PagedRope(_Block):
    """The rotary step into the pages (rf_paged_rope)."""
    _fields_ = [(n, _vp) for n in ("q", "k", "v", "q_norm", "k_norm", "q16", "positions", "slots", "turns")] + \
               [(n, _i64) for n in ("ld_q", "ld_k", "ld_v", "ld_q16")] + \
               [(n, _i32) for n in ("rows", "num_heads", "rot_dim", "neox")] + [("eps", _f), ("attn_factor", _f)]


class PagedAttention(_Block):
    """Attention of the new rows over the pages (rf_paged_attention)."""
    _fields_ = [(n, _vp) for n in ("q", "out", "block_tables", "q_start", "kv_lens", "workspace")] + \
               [("workspace_bytes", _sz), ("ld_q", _i64), ("ld_out", _i64)] + \
               [(n, _i32) for n in ("num_seqs", "max_blocks", "rows", "num_heads", "max_new", "window", "out_f32")] + \
               [("scale", _f)]


class LogitsRules(_Block):
    """Rules on a batch of logits (rf_logits_rules)."""
    _fields_ = [("logits", _vp), ("out", _vp), ("ld_logits", _i64), ("ld_out", _i64), ("history", _vp),
                ("ld_history", _i64), ("prompt_lens", _vp), ("total_lens", _vp), ("repetition", _vp),
                ("frequency", _vp), ("presence", _vp), ("bias_start", _vp), ("bias_ids", _vp), ("bias_values", _vp),
                ("allowed", _vp), ("ld_allowed", _i64), ("rows", _i32), ("vocab", _i32)]


def _addr(p):
    if not hasattr(p, "data_ptr"):
        return p
    if not p.is_cuda:
        raise ValueError("a tensor that is not on a GPU")
    return p.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise HipApiError(rc, what)


def plan(step: PagedPlan, stream=None) -> None:
    _check(load().rf_paged_plan_launch(ctypes.byref(step), _stream(stream)), "rf_paged_plan_launch")


def release(ended, ctx_lens, block_tables, free_pages, free_count, num_seqs: int, max_blocks: int, page_size: int,
            num_pages: int, stream=None) -> None:
    _check(load().rf_paged_release_launch(_addr(ended), _addr(ctx_lens), _addr(block_tables), _addr(free_pages),
                                          _addr(free_count), num_seqs, max_blocks, page_size, num_pages,
                                          _stream(stream)), "rf_paged_release_launch")


def rope_turns_table(turns, rot_dim: int, theta_base: float, mode: int = ROPE_PLAIN, factor: float = 1.0,
                     orig_positions: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, freq_scale=None,
                     stream=None) -> None:
    _check(load().rf_rope_turns_table(_addr(turns), rot_dim, theta_base, mode, factor, orig_positions, beta_fast,
                                      beta_slow, _addr(freq_scale), _stream(stream)), "rf_rope_turns_table")


def rope_write(step: PagedRope, cache: PagedCache, stream=None) -> None:
    _check(load().rf_paged_rope_write_launch(ctypes.byref(step), ctypes.byref(cache), _stream(stream)),
           "rf_paged_rope_write_launch")


def attention_workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int) -> int:
    return int(load().rf_paged_attention_workspace_bytes(num_heads, num_kv_heads, head_dim))


def attention(step: PagedAttention, cache: PagedCache, stream=None) -> None:
    _check(load().rf_paged_attention_launch(ctypes.byref(step), ctypes.byref(cache), _stream(stream)),
           "rf_paged_attention_launch")


def logits_rules(rules: LogitsRules, stream=None) -> None:
    _check(load().rf_logits_rules_launch(ctypes.byref(rules), _stream(stream)), "rf_logits_rules_launch")
