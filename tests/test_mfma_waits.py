"""Wait states between a matrix instruction and the reads of its result in the built kernels, over branches too
(the compiler inserts them, and has left too few where a branch skips what stands between the two)."""
import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from rocmforge_amd import build as B

OBJDUMP = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm/bin/llvm-objdump"
# wait states from the instruction to a read of its result that is no matrix instruction: of 4 passes, and of 8 (those of
# 32 rows)
NEED = {"v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_32x32x16_f16": 12}
OTHER = 8
BLOCK = re.compile(r"^[0-9a-f]+ <(\S+)>:$")


def kernels(obj, tmp):
    """(name, instructions) of an object's kernels; an instruction is (name, operands), a label (None, name)."""
    shutil.copy(obj, tmp / obj.name)
    subprocess.run([OBJDUMP, "--offloading", obj.name], cwd=tmp, check=True, capture_output=True)
    for code in sorted(tmp.glob(f"{obj.name}*gfx950*")):
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", code], check=True,
                              capture_output=True, text=True).stdout
        name, body = None, []
        for line in text.splitlines():
            line = line.split("//")[0].strip()
            block = BLOCK.match(line)
            if block and not re.fullmatch(r"L\d+", block[1]):
                if name:
                    yield name, body
                name, body = block[1], []
            elif block or re.fullmatch(r"<L\d+>:", line):
                body.append((None, block[1] if block else line[1:-2]))
            elif line and name:
                op, _, rest = line.partition(" ")
                body.append((op, [t.strip() for t in re.split(r",(?![^\[]*\])", rest)] if rest.strip() else []))
        if name:
            yield name, body


def registers(operand):
    m = re.match(r"[-|]*([av])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    lo, hi = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(lo), int(hi) + 1)}


def reads(op, operands):
    """Registers that an instruction reads, its result's among them."""
    if op.startswith(("v_mfma", "v_smfma")) or not op.startswith(("v_", "ds_", "global_", "flat_", "scratch_", "buffer_")):
        return set()
    return set().union(*map(registers, operands)) if operands else set()


def too_close(body):
    """(matrix instruction, read, wait states between, needed), the nearest read of each."""
    at = {name: i for i, (op, name) in enumerate(body) if op is None}
    for i, (op, operands) in enumerate(body):
        if not op or not op.startswith("v_mfma"):
            continue
        need, result = NEED.get(op, OTHER), registers(operands[0])
        todo, seen = [(i + 1, 0)], set()
        while todo:
            j, waited = todo.pop()
            if j >= len(body) or waited >= need or (j, waited) in seen:
                continue
            seen.add((j, waited))
            name, args = body[j]
            if name is None:
                todo.append((j + 1, waited))
            elif name == "s_nop":
                todo.append((j + 1, waited + 1 + int(args[0], 0)))
            elif name.startswith(("s_cbranch", "s_branch")):
                todo.append((at[args[0]], waited + 1))
                if name != "s_branch":
                    todo.append((j + 1, waited + 1))
            elif name == "s_endpgm":
                continue
            elif reads(name, args) & result:
                yield f"{op} {operands[0]}", f"{name} {', '.join(args)}", waited, need
            else:
                todo.append((j + 1, waited + 1))


@pytest.mark.parametrize("source", ["lora.hip", "paged_attn.hip", "paged8_attn.hip"])
def test_results_are_read_late_enough(tmp_path, source):
    obj = B.BUILD / (Path(source).stem + ".o")
    if not obj.exists() or not OBJDUMP.exists():
        pytest.skip("no built object, or nothing to disassemble it with")
    wrong, seen = [], 0
    for name, body in kernels(obj, tmp_path):
        seen += sum(op is not None and op.startswith("v_mfma") for op, _ in body)
        wrong += [f"{name}: {mfma} -> {read}: {waited} of {need}" for mfma, read, waited, need in too_close(body)]
    assert seen > 20                                       # (it has looked at the kernels)
    assert not wrong, "\n".join(wrong[:10])


def test_what_is_too_close():
    # a read behind a branch that skips the instructions in between, and the same with enough of them
    mfma = ("v_mfma_f32_16x16x32_f16", ["a[0:3]", "v[0:3]", "v[4:7]", "a[0:3]"])
    body = lambda n: [mfma, ("s_cbranch_vccnz", ["L1"])] + [("v_mov_b32_e32", ["v9", "v8"])] * 9 + [(None, "L1")] + \
                     [("s_nop", [str(n)]), ("v_accvgpr_read_b32", ["v1", "a2"]), ("s_endpgm", [])]
    assert [w[2:] for w in too_close(body(2))] == [(4, 8)]
    assert not list(too_close(body(6)))
