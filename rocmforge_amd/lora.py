"""Low-rank adapters of many requests beside a shared projection -- the Python face
of rf_lora_add_launch in include/rocmforge_cdna4.h, which states what it computes and
which arguments it takes.

A projection's weights stay shared and quantised; each request of a batch's step (the
rows' order is paged.py's) names the adapter whose B A x is added to its rows:

    add(step, [target_q, target_k, target_v])      targets that share x: up to three

The blocks are the C structs, and tensors are looked at as paged.py does.  A step
without a workspace gets one from torch's allocator for the call, on its stream (a graph
that is not torch's needs one of its own: workspace_bytes).
"""
from __future__ import annotations

import ctypes

from ._lib import load
from .paged import _F32, _HALF, _I32, _Block, _check, _i32, _i64, _one_device, _stream, _sz, _vp


class LoraStep(_Block):
    """A step's rows and the requests' adapters (rf_lora)."""
    _fields_ = [(n, _vp) for n in ("x", "adapters", "q_start", "ranks", "scales", "workspace")] + \
               [("workspace_bytes", _sz), ("ld_x", _i64)] + \
               [(n, _i32) for n in ("rows", "num_seqs", "num_adapters", "max_rank", "in_dim", "x_f16")]
    _tensors = {"x": (None, "ld_x"), "adapters": _I32, "q_start": _I32, "ranks": _I32, "scales": _F32,
                "workspace": (None, "dense")}

    def _types(self, name):
        return ((_HALF if self.x_f16 else ("float32",)) if name == "x" else super()._types(name))


class LoraTarget(_Block):
    """One projection's adapters and output (rf_lora_target): a [adapters][max_rank][in_dim], b
    [adapters][out_dim][max_rank]."""
    _fields_ = [(n, _vp) for n in ("a", "b", "base", "y")] + \
               [(n, _i64) for n in ("a_stride", "b_stride", "ld_base", "ld_y")] + [("out_dim", _i32)]
    _tensors = {"a": (_HALF, "a_stride"), "b": (_HALF, "b_stride"), "base": (("float32",), "ld_base"),
                "y": (("float32",), "ld_y")}


def _targets(targets):
    targets = [targets] if isinstance(targets, LoraTarget) else list(targets)
    return targets, (LoraTarget * max(len(targets), 1))(*targets)


def workspace_bytes(step: LoraStep, targets) -> int:
    """Bytes of a launch's workspace; 0 where it needs none (or is refused).  A server's largest step (rows, requests,
    targets, ranks, widths) needs the most."""
    targets, block = _targets(targets)
    return int(load().rf_lora_workspace_bytes(ctypes.byref(step), block, len(targets)))


def _memory(n: int, stream):
    """n bytes for work on the stream: they go back to the allocator as the call ends, and to that stream's work alone."""
    import torch
    if stream is None:
        return torch.empty(n, dtype=torch.uint8, device="cuda")
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        return torch.empty(n, dtype=torch.uint8, device="cuda")


def add(step: LoraStep, targets, stream=None) -> None:
    """y = base + scale B (A x) for each target (a LoraTarget, or up to three of them)."""
    targets, block = _targets(targets)
    on = {b.__dict__["_on"] if "_on" in b.__dict__ else b._device() for b in (step, *targets)}
    handle = _stream(stream, _one_device(on) if len(on) > 1 else on.pop())
    lib = load()
    memory = None
    if not step.workspace:
        n = lib.rf_lora_workspace_bytes(ctypes.byref(step), block, len(targets))
        if n:
            memory = _memory(n, stream)
            step = LoraStep.from_buffer_copy(step)
            # (past the block's own: a copy keeps no tensors)
            ctypes.Structure.__setattr__(step, "workspace", memory.data_ptr())
            ctypes.Structure.__setattr__(step, "workspace_bytes", n)
    _check(lib.rf_lora_add_launch(ctypes.byref(step), block, len(targets), handle), "rf_lora_add_launch")
