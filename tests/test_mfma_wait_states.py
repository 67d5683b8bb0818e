"""Codegen guard (CPU only: the files are cross-compiled to assembly): between a matrix instruction and the first other instruction
that reads its result there are 8 wait states on EVERY path, not only on straight lines.

The compiler (ROCm 7.2) places these waits itself, but where a branch skips other matrix instructions it counted along the long
path only: the short path then read a result before it was there - wrong values without an error, and only in tiles that took the
branch.  mfma16.h says how the kernels avoid such branches; this test finds one if it comes back."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "transformer_engine_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
WAIT_STATES = 8     # 16x16x32, eight passes; the smallest distance on the compiler's own straight lines is the same

pytestmark = pytest.mark.skipif(shutil.which(HIPCC) is None and not os.path.exists(HIPCC), reason="hipcc not available")


def _registers(operand):
    m = re.fullmatch(r"([av])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.fullmatch(r"([av])(\d+)", operand)
    return {(m[1], int(m[2]))} if m else set()


def _split(instruction):
    name, _, rest = instruction.partition(" ")
    return name, [o.strip() for o in rest.split(",")] if rest else []


def _kernels(asm):
    """{kernel: [(label, [instruction, ...]), ...]} in layout order."""
    found, blocks = {}, None
    for line in asm.split("\n"):
        m = re.match(r"(_ZN2te\w+):", line)
        if m:
            blocks = found.setdefault(m[1], [("entry", [])])
        elif line.startswith(".Lfunc_end"):
            blocks = None
        elif blocks is not None:
            m = re.match(r"(\.LBB\w+):", line)
            text = line.split(";")[0].strip()
            if m:
                blocks.append((m[1], []))
            elif text and not text.startswith("."):
                blocks[-1][1].append(re.sub(r"\s+", " ", text))
    return found


def _early_reads(blocks):
    place = {label: i for i, (label, _) in enumerate(blocks)}
    found = []

    def follow(block, start, pending, distance, jumps, origin):
        while block < len(blocks):
            for text in blocks[block][1][start:]:
                name, ops = _split(text)
                stores = name.startswith(("global_store", "ds_write", "scratch_store"))
                if not name.startswith("s_"):
                    # a matrix instruction may take the result as its accumulator at once
                    sources = ops[1:3] if name.startswith("v_mfma") else ops if stores else ops[1:]
                    read = set().union(*(_registers(o) for o in sources)) if sources else set()
                    if read & pending:
                        if distance < WAIT_STATES:
                            found.append((distance, origin, text))
                        pending = pending - read
                    if ops and not stores:
                        pending = pending - _registers(ops[0])
                distance += int(ops[0]) + 1 if name == "s_nop" else 1
                if not pending or distance >= WAIT_STATES or name in ("s_endpgm", "s_setpc_b64"):
                    return
                if name in ("s_branch",) or name.startswith("s_cbranch"):
                    if jumps < 6 and ops[-1] in place:
                        follow(place[ops[-1]], 0, pending, distance, jumps + 1, origin)
                    if name == "s_branch":
                        return
            block, start = block + 1, 0

    for i, (_, instructions) in enumerate(blocks):
        for j, text in enumerate(instructions):
            if text.startswith("v_mfma"):
                follow(i, j + 1, _registers(_split(text)[1][0]), 0, 0, text)
    return found


def test_the_check_sees_the_short_path():
    blocks = [("entry", ["v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]", "s_cbranch_scc1 .LBB0_2"]),
              (".LBB0_1", ["v_mfma_f32_16x16x32_bf16 a[4:7], v[0:3], v[4:7], a[4:7]"] + ["v_mov_b32 v9, v8"] * 9),
              (".LBB0_2", ["v_accvgpr_read_b32 v8, a0"])]
    assert [d for d, _, _ in _early_reads(blocks)] == [1]
    blocks[0][1].insert(1, "s_nop 7")
    assert not _early_reads(blocks)


@pytest.mark.parametrize("source", ["lora.hip", "moe_decode.hip"])
def test_no_result_is_read_early(source, tmp_path):
    out = os.path.join(str(tmp_path), "k.s")
    subprocess.run([HIPCC, "-std=c++17", "-O3", "-fPIC", "--offload-arch=gfx950", "-I../../include", "-I.", "-fno-gpu-rdc",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", source, "-o", out],
                   cwd=CSRC, check=True, capture_output=True, timeout=900)
    with open(out) as fh:
        kernels = _kernels(fh.read())
    assert sum("v_mfma" in t for blocks in kernels.values() for _, ins in blocks for t in ins) > 1000
    early = {k: _early_reads(blocks) for k, blocks in kernels.items()}
    assert not any(early.values()), {k: v[:3] for k, v in early.items() if v}
