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

Tensors are looked at before they are launched on, once after each change of a
block: a ValueError where a type is not the field's (16-bit integers pass for fp16
bits, the workspace is of any type), where elements do not lie as the field's
strides say (rows one ld_.. apart and dense in themselves, all else contiguous), or
where a tensor or the stream is not of the current device.  Addresses are taken as
they are, and so are sizes.
"""
from __future__ import annotations

import ctypes

from ._lib import load
from .ops import HipApiError

ROPE_PLAIN, ROPE_LINEAR, ROPE_YARN = 0, 1, 2

_vp, _i32, _i64, _f, _sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


# What a pointer field takes: types of elements, and where these lie ("dense", "last": the last
# dim is dense, or the field that holds the distance of rows).
_I32 = (("int32",), "dense")
_F32 = (("float32",), "dense")
_HALF = ("float16", "int16", "uint16")


def _dense(shape, strides) -> bool:
    n = 1
    for size, stride in zip(reversed(shape), reversed(strides)):
        if size == 0:
            return True
        if size > 1 and stride != n:
            return False
        n *= size
    return True


def _look(what: str, t, types, layout, ld=None) -> None:
    kind = str(t.dtype).replace("torch.", "")
    if types is not None and kind not in types:
        raise ValueError(f"{what} is {kind}, not {' or '.join(types)}")
    shape, strides = tuple(t.shape), tuple(t.stride())
    if layout == "last":
        ok = not shape or shape[-1] <= 1 or strides[-1] == 1
    elif layout == "dense" or len(shape) < 2:
        ok = _dense(shape, strides)
    else:
        ok = _dense(shape[1:], strides[1:]) and (shape[0] <= 1 or strides[0] == ld)
    if not ok:
        where = f"rows {ld} apart ({layout})" if ld is not None else "dense"
        raise ValueError(f"{what} has strides {strides}, not {where}")


class _Block(ctypes.Structure):
    _tensors = {}

    def __init__(self, **fields):
        super().__init__()
        types = dict(self._fields_)
        unknown = sorted(set(fields) - set(types))
        if unknown:
            raise TypeError(f"{type(self).__name__} has no field {', '.join(unknown)}")
        for name, value in fields.items():
            setattr(self, name, value)

    def __setattr__(self, name, value):
        tensor = hasattr(value, "data_ptr")
        if tensor and name not in self._tensors:
            raise ValueError(f"{type(self).__name__}.{name} is not a pointer")
        super().__setattr__(name, _addr(value))
        kept = self.__dict__.setdefault("_kept", {})
        kept.pop(name, None)
        if tensor:
            kept[name] = value
        self.__dict__.pop("_on", None)

    def _types(self, name):
        return self._tensors[name][0]

    def _device(self):
        """Index of the device of the block's tensors, None without any; they are looked at before."""
        kept = self.__dict__.get("_kept", {})
        for name, t in kept.items():
            layout = self._tensors[name][1]
            _look(f"{type(self).__name__}.{name}", t, self._types(name), layout, getattr(self, layout, None))
        on = self.__dict__["_on"] = _one_device([t.device.index for t in kept.values()])
        return on


class PagedCache(_Block):
    """K and V pages of one layer (rf_paged_cache)."""
    _fields_ = [("k", _vp), ("v", _vp), ("page_stride", _i64), ("row_stride", _i64), ("head_stride", _i64),
                ("num_pages", _i32), ("page_size", _i32), ("num_kv_heads", _i32), ("head_dim", _i32)]
    _tensors = {"k": (_HALF, "last"), "v": (_HALF, "last")}

    def _device(self):
        k, v = [self.__dict__.get("_kept", {}).get(n) for n in "kv"]
        if k is not None and v is not None and len(k.shape) == len(v.shape) and any(
                m > 1 and n > 1 and a != b for m, n, a, b in zip(k.shape, v.shape, k.stride(), v.stride())):
            raise ValueError(f"PagedCache.v has strides {v.stride()}, k {k.stride()}")
        return super()._device()


class PagedPlan(_Block):
    """The plan of a step (rf_paged_plan)."""
    _fields_ = [(n, _vp) for n in ("new_lens", "ctx_in", "ctx_out", "free_pages", "free_in", "free_out",
                                   "block_tables", "q_start", "kv_lens", "positions", "slots")] + \
               [(n, _i32) for n in ("num_seqs", "max_blocks", "page_size", "max_rows", "num_pages")]
    _tensors = {n: _I32 for n, t in _fields_ if t is _vp} | {"block_tables": (("int32",), "max_blocks")}


class PagedRope(_Block):
    """The rotary step into the pages (rf_paged_rope)."""
    _fields_ = [(n, _vp) for n in ("q", "k", "v", "q_norm", "k_norm", "q16", "positions", "slots", "turns")] + \
               [(n, _i64) for n in ("ld_q", "ld_k", "ld_v", "ld_q16")] + \
               [(n, _i32) for n in ("rows", "num_heads", "rot_dim", "neox")] + [("eps", _f), ("attn_factor", _f)]
    _tensors = {n: (("float32",), f"ld_{n}") for n in "qkv"} | {
        "q_norm": _F32, "k_norm": _F32, "q16": (_HALF, "ld_q16"), "positions": _I32, "slots": _I32,
        "turns": (("float64",), "dense")}


class PagedAttention(_Block):
    """Attention of the new rows over the pages (rf_paged_attention)."""
    _fields_ = [(n, _vp) for n in ("q", "out", "block_tables", "q_start", "kv_lens", "workspace")] + \
               [("workspace_bytes", _sz), ("ld_q", _i64), ("ld_out", _i64)] + \
               [(n, _i32) for n in ("num_seqs", "max_blocks", "rows", "num_heads", "max_new", "window", "out_f32")] + \
               [("scale", _f)]
    _tensors = {"q": (_HALF, "ld_q"), "out": (None, "ld_out"), "block_tables": (("int32",), "max_blocks"),
                "q_start": _I32, "kv_lens": _I32, "workspace": (None, "dense")}

    def _types(self, name):
        return ((("float32",) if self.out_f32 else _HALF) if name == "out" else super()._types(name))


class LogitsRules(_Block):
    """Rules on a batch of logits (rf_logits_rules)."""
    _fields_ = [("logits", _vp), ("out", _vp), ("ld_logits", _i64), ("ld_out", _i64), ("history", _vp),
                ("ld_history", _i64), ("prompt_lens", _vp), ("total_lens", _vp), ("repetition", _vp),
                ("frequency", _vp), ("presence", _vp), ("bias_start", _vp), ("bias_ids", _vp), ("bias_values", _vp),
                ("allowed", _vp), ("ld_allowed", _i64), ("rows", _i32), ("vocab", _i32)]
    _tensors = {"logits": (("float32",), "ld_logits"), "out": (("float32",), "ld_out"),
                "history": (("int32",), "ld_history"), "prompt_lens": _I32, "total_lens": _I32, "repetition": _F32,
                "frequency": _F32, "presence": _F32, "bias_start": _I32, "bias_ids": _I32, "bias_values": _F32,
                "allowed": (("int32", "uint32"), "ld_allowed")}


def _addr(p):
    if not hasattr(p, "data_ptr"):
        return p
    if not p.is_cuda:
        raise ValueError("a tensor that is not on a GPU")
    return p.data_ptr()


def _one_device(indexes):
    on = sorted(set(i for i in indexes if i is not None))
    if len(on) > 1:
        raise ValueError("tensors of cuda:" + " and cuda:".join(map(str, on)) + " in one launch")
    return on[0] if on else None


def _stream(stream, on):
    """The stream's handle.  on: the tensors' device, None where there are addresses only."""
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
        current = stream.device_index
    elif on is None and not hasattr(stream, "cuda_stream"):
        return stream
    else:
        current = torch.cuda.current_device()
        if getattr(stream, "device_index", current) != current:
            raise ValueError(f"a stream of cuda:{stream.device_index}, the current device is cuda:{current}")
    if on is not None and on != current:
        raise ValueError(f"tensors of cuda:{on}, the current device is cuda:{current}")
    return getattr(stream, "cuda_stream", stream)


def _launch(name: str, stream, step, cache=None) -> None:
    on = step.__dict__["_on"] if "_on" in step.__dict__ else step._device()
    if cache is None:
        _check(getattr(load(), name)(ctypes.byref(step), _stream(stream, on)), name)
        return
    cache_on = cache.__dict__["_on"] if "_on" in cache.__dict__ else cache._device()
    if on != cache_on:
        on = _one_device([on, cache_on])
    _check(getattr(load(), name)(ctypes.byref(step), ctypes.byref(cache), _stream(stream, on)), name)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise HipApiError(rc, what)


def _addrs(stream, tensors):
    """Addresses of (name, value, types, layout, rows' distance), and the stream's handle."""
    out, on = [], []
    for name, value, types, layout, ld in tensors:
        out.append(_addr(value))
        if hasattr(value, "data_ptr"):
            _look(name, value, types, layout, ld)
            on.append(value.device.index)
    return out, _stream(stream, _one_device(on))


def plan(step: PagedPlan, stream=None) -> None:
    _launch("rf_paged_plan_launch", stream, step)


def release(ended, ctx_lens, block_tables, free_pages, free_count, num_seqs: int, max_blocks: int, page_size: int,
            num_pages: int, stream=None) -> None:
    at, handle = _addrs(stream, [("ended", ended, *_I32, None), ("ctx_lens", ctx_lens, *_I32, None),
                                 ("block_tables", block_tables, ("int32",), "max_blocks", max_blocks),
                                 ("free_pages", free_pages, *_I32, None), ("free_count", free_count, *_I32, None)])
    _check(load().rf_paged_release_launch(*at, num_seqs, max_blocks, page_size, num_pages, handle),
           "rf_paged_release_launch")


def rope_turns_table(turns, rot_dim: int, theta_base: float, mode: int = ROPE_PLAIN, factor: float = 1.0,
                     orig_positions: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, freq_scale=None,
                     stream=None) -> None:
    at, handle = _addrs(stream, [("turns", turns, ("float64",), "dense", None), ("freq_scale", freq_scale, *_F32, None)])
    _check(load().rf_rope_turns_table(at[0], rot_dim, theta_base, mode, factor, orig_positions, beta_fast, beta_slow,
                                      at[1], handle), "rf_rope_turns_table")


def rope_write(step: PagedRope, cache: PagedCache, stream=None) -> None:
    _launch("rf_paged_rope_write_launch", stream, step, cache)


def attention_workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int) -> int:
    return int(load().rf_paged_attention_workspace_bytes(num_heads, num_kv_heads, head_dim))


def attention(step: PagedAttention, cache: PagedCache, stream=None) -> None:
    _launch("rf_paged_attention_launch", stream, step, cache)


def logits_rules(rules: LogitsRules, stream=None) -> None:
    _launch("rf_logits_rules_launch", stream, rules)
