"""CPU: where lanes that a branch had switched off come back - `s_or_b64 exec, exec, ...` at the head of a block - nothing may have been done to vector registers before: the
lanes would go without it. Where this compiler puts a scalar register that it spills at the head of such a block (v_writelane), copies and spills of vector registers have come behind it,
and before the lanes (in builds of policy_rows_kernel that kept 96 registers and spilled both kinds: garbage in the lanes' addresses behind the block). Looked up in the
code that the compiler makes of ws_loss.hip with the library's flags; the built kernels have to spill no vector register either."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

import wo
from test_lds_budget import READELF
from test_meeting_order import LIB, code_objects

KERNELS = r"score_rows_kernel|grad_rows_kernel|policy_rows_kernel|policy_kernel|preference_kernel"
N_KERNELS = 16 + 8 + 36 + 6 + 2  # scores, gradients, policy rows of three builds and of a fourth for fp32, the two losses over log-probabilities
VECTOR = re.compile(r"v_(?!writelane|readlane|readfirstlane)|scratch_|global_|ds_|flat_|buffer_")
ENDS = re.compile(r"s_cbranch|s_branch|s_and_saveexec|s_mov_b64 exec|s_and_b64 exec|s_xor_b64 exec|s_andn2_b64 exec")


def blocks(text):
    """(kernel, instructions) of every basic block of a listing: they begin at a label or at the compiler's remark that one begins."""
    kernel, block = None, []
    for line in text.splitlines():
        name = re.match(r"^(_Z\w+):", line)
        if name or re.match(r"^\.LBB", line) or "; %bb." in line:
            if block:
                yield kernel, block
            kernel, block = (name.group(1) if name else kernel), []
            continue
        op = line.split(";")[0].strip()
        if op and not op.startswith("."):
            block.append(op)
    if block:
        yield kernel, block


def before_the_lanes_come_back(block):
    """The vector instructions at a block's head, scalar spills among them, before its lanes come back; None where they do not at its head."""
    before, spilled = [], False
    for op in block:
        spilled = spilled or op.startswith("v_writelane")
        if op.startswith("s_or_b64 exec, exec"):
            return before if spilled else []
        if ENDS.match(op):
            return None
        if VECTOR.match(op):
            before.append(op)
    return None


def test_nothing_vector_stands_before_the_lanes_come_back(tmp_path):
    spec = importlib.util.spec_from_file_location("ws_build", os.path.join(wo.ROOT, "whirl-llm_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    out = tmp_path / "loss.s"
    subprocess.run([hipcc, *build.FLAGS, "-S", "--cuda-device-only", "-o", str(out), build.SRC_LOSS], check=True, capture_output=True)
    seen, restores = set(), 0
    for kernel, block in blocks(out.read_text()):
        seen.add(kernel)
        before = before_the_lanes_come_back(block)
        if before is not None:
            restores += 1
            assert not before, (kernel, before)
    assert len([k for k in seen if k and re.search(KERNELS, k)]) == N_KERNELS and restores > 1000


def test_a_copy_before_the_lanes_come_back_is_seen():
    text = "_Z1k:\n\ts_and_saveexec_b64 s[0:1], vcc\n\ts_cbranch_execz .LBB0_2\n; %bb.1:\n\tv_mov_b32_e32 v1, 0\n.LBB0_2:\n\tv_writelane_b32 v9, s1, 0\n\tv_mov_b32_e32 v2, v1\n\ts_or_b64 exec, exec, s[0:1]\n"
    assert [before_the_lanes_come_back(b) for _, b in blocks(text)] == [None, None, ["v_mov_b32_e32 v2, v1"]]


def test_loss_kernels_keep_their_registers(tmp_path):
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    found = 0
    for i, blob in enumerate(code_objects(LIB)):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(blob)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for block in re.split(r"(?=\.agpr_count)", notes):
            name = re.search(r"\.name: +(\S+)", block)
            if name and re.search(KERNELS, name.group(1)):
                found += 1
                assert re.search(r"\.vgpr_spill_count: 0\b", block) and re.search(r"\.private_segment_fixed_size: 0\b", block), name.group(1)
    assert found == N_KERNELS
