"""CPU: the code that the compiler makes of the kernels of a cycle with trees. Nothing may be done to vector registers before the lanes that a branch has switched off come back
(test_exec_restore.py says why); and the builds of attention that load straight into LDS wait for all their loads right before the meetings behind which LDS is read."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

import wo
from test_exec_restore import before_the_lanes_come_back, blocks
from test_lds_budget import READELF
from test_meeting_order import LIB, code_objects


def listing(tmp_path, source):
    spec = importlib.util.spec_from_file_location("ws_build", os.path.join(wo.ROOT, "whirl-llm_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    out = tmp_path / "code.s"
    subprocess.run([hipcc, *build.FLAGS, "-S", "--cuda-device-only", "-o", str(out), getattr(build, source)], check=True, capture_output=True)
    return out.read_text()


@pytest.mark.parametrize("source,kernels,number", [("SRC_TREE", r"tree_(stage|rows|draw)_kernel", 1 + 4 + 8), ("SRC_ATTEND", r"attend_(join_)?kernel", 2 * 12),
                                                   ("SRC_CACHE", r"cache_(reserve|fork|copy|release|keep)_kernel", 5)])
def test_nothing_vector_stands_before_the_lanes_come_back(tmp_path, source, kernels, number):
    seen, staged = set(), 0
    text = listing(tmp_path, source)
    for kernel, block in blocks(text):
        seen.add(kernel)
        before = before_the_lanes_come_back(block)
        assert not before, (kernel, before)
    assert len([k for k in seen if k and re.search(kernels, k)]) == number
    if source != "SRC_ATTEND":
        return
    for name, body in re.findall(r"^(_Z\w*attend_kernel\w*):(.*?)^\.Lfunc_end", text, re.S | re.M):
        if "global_load_lds" not in body:
            continue
        staged += 1
        ops = [line.split(";")[0].strip() for line in body.splitlines()]
        last = max(i for i, op in enumerate(ops) if op.startswith("global_load_lds"))
        waits = [i for i, op in enumerate(ops) if re.match(r"s_waitcnt vmcnt\(0\)", op)]
        meetings = [i for i, op in enumerate(ops) if op.startswith("s_barrier")]
        assert any(b > last for b in meetings), name
        first = min(i for i, op in enumerate(ops) if op.startswith("global_load_lds"))
        heads = [b for b in meetings if b > first and any(b - 8 < w < b for w in waits)]  # each half of the loop over two buffers begins with one
        assert len(heads) >= 2, name
    assert staged == 9


def test_verification_kernels_keep_their_registers(tmp_path):
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    found = 0
    for i, blob in enumerate(code_objects(LIB)):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(blob)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for block in re.split(r"(?=\.agpr_count)", notes):
            name = re.search(r"\.name: +(\S+)", block)
            if name and re.search(r"tree_(stage|rows|draw)_kernel", name.group(1)):
                found += 1
                assert re.search(r"\.vgpr_spill_count: 0\b", block) and re.search(r"\.private_segment_fixed_size: 0\b", block), name.group(1)
    assert found == 1 + 4 + 8


def flow(function):
    """{block: (instructions, the blocks behind)} of a function in the compiler's intermediate form."""
    out, name = {}, "entry"
    for line in function.splitlines()[1:]:
        label = re.match(r"^(\d+):", line)
        if label:
            name = label.group(1)
        ops, behind = out.setdefault(name, ([], []))
        op = line.strip()
        if line.startswith("  "):
            ops.append(op)
            if op.startswith("br ") or op.startswith("switch ") or op.startswith("]") or re.match(r"i\d+ \S+, label", op):
                behind.extend(re.findall(r"label %(\d+)", op))
    return out


def reached_without_meeting(blocks_, first, second):
    """Whether an instruction of `second` can come behind one of `first` with no meeting of the workgroup between them."""
    seen, left = set(), [(name, i + 1) for name, (ops, _) in blocks_.items() for i, op in enumerate(ops) if first(op)]
    assert left
    while left:
        name, i = left.pop()
        ops, behind = blocks_[name]
        for op in ops[i:]:
            if "@llvm.amdgcn.s.barrier()" in op:
                break
            if second(op):
                return True
        else:
            for to in behind:
                if to not in seen:
                    seen.add(to)
                    left.append((to, 0))
    return False


def test_attention_clears_a_flag_before_a_meeting(tmp_path):
    """A workgroup's flag for infinities and NaN in the V of nodes (s_odd): between the store that clears it and one of another wave that sets it the waves meet, on every way through the kernel. Else
    a wave that is late would clear what another one has found."""
    spec = importlib.util.spec_from_file_location("ws_build", os.path.join(wo.ROOT, "whirl-llm_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    out = tmp_path / "code.ll"
    subprocess.run([hipcc, *build.FLAGS, "-S", "-emit-llvm", "--cuda-device-only", "-o", str(out), build.SRC_ATTEND], check=True, capture_output=True)
    found = 0
    for function in re.findall(r"^define [^\n]*attend_kernel.*?^}", out.read_text(), re.S | re.M):
        flag = r"@\w*s_odd\b"
        places = re.findall(rf"(%\d+) = getelementptr [^\n]*{flag}", function)
        at = rf"(?:{flag}|{'|'.join(re.escape(p) for p in places)})" if places else flag
        clears, sets = re.compile(rf"store i32 0, ptr addrspace\(3\) {at}(?:,|$)"), re.compile(rf"store i32 1, ptr addrspace\(3\) {at}(?:,|$)")
        blocks_ = flow(function)
        assert sum(bool(sets.match(op)) for ops, _ in blocks_.values() for op in ops) >= 1
        assert not reached_without_meeting(blocks_, clears.match, sets.match), function[:120]
        found += 1
    assert found == 12
