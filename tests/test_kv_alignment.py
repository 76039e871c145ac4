"""The alignment that the key-value cache's kernels promise the compiler, from
the LLVM IR that hipcc makes of them (no GPU): a cache's tensors are aligned to
16 bytes and no more, three words of a 4-bit row to 4."""
import collections
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vram-compression_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


def accesses(source, tmp_path):
    """{(load or store, vector type): alignments} of a file's global accesses."""
    out = tmp_path / "ir.ll"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-emit-llvm", "-S", "-o", str(out),
                    os.path.join(CSRC, source)], check=True, capture_output=True)
    found = collections.defaultdict(set)
    for kind, type_, align in re.findall(r"(load|store) (<\d+ x \w+>)[^\n]*?ptr addrspace\(1\)[^\n]*?align (\d+)",
                                         out.read_text()):
        found[kind, type_].add(int(align))
    return found


def test_three_words_of_a_row(tmp_path):
    found = accesses("kv_attend.hip", tmp_path)
    assert found["load", "<3 x i32>"] == {4}
    assert found["load", "<2 x i32>"] == {8}
    assert found["load", "<4 x i32>"] <= {16}


def test_rows_of_f32(tmp_path):
    """Reads of new keys and values and writes of outputs may promise 32 bytes
    (the host checks them); reads and writes of a cache may not."""
    found = accesses("kv_append.hip", tmp_path)
    assert found["load", "<8 x float>"] == {16, 32}
    assert found["store", "<8 x float>"] <= {32} and found["store", "<4 x i32>"] <= {16}
    text = (tmp_path / "ir.ll").read_text()
    bodies = {name: body for name, body in re.findall(r"define [^\n]*@(\w*kernelI\w+)\((.*?)\n}", text, re.S)}
    appends = [b for n, b in bodies.items() if "kv_append_kernelIfLb0" in n]
    reads = [b for n, b in bodies.items() if "kv_read_kernelIf" in n]
    assert len(appends) == 2 and len(reads) == 1
    for b in appends:
        assert not re.search(r"store <8 x float>", b)
    for b in reads:
        assert set(re.findall(r"load <8 x float>[^\n]*align (\d+)", b)) == {"16"}
