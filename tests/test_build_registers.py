"""Kernels whose loops have no register to spare: what ptxas said of them when the library was built."""
import glob
import os
import re
import subprocess

from attention_kernel_triton_b200 import build


def kernels(src, tmp_path):
    """(mangled name, registers, bytes of spill stores, bytes of spill loads) of every kernel of a source file."""
    path = os.path.join(build.CSRC, src)
    log, obj = build.log_of(path), os.path.join(build.BUILD, src[:-3] + ".o")
    deps = [path, *glob.glob(os.path.join(build.CSRC, "*.cuh")), *glob.glob(os.path.join(build.CSRC, "*.h"))]
    if os.path.exists(log) and not build._needs(obj, deps):
        with open(log) as f:
            text = f.read()
    else:  # the library here is not built of these sources
        cmd = [build.nvcc(), *build.flags_for(path), "-c", path, "-o", str(tmp_path / "k.o")]
        text = subprocess.run(cmd, check=True, capture_output=True, text=True).stderr
    return [(m[1], int(m[4]), int(m[2]), int(m[3])) for m in re.finditer(
        r"Compiling entry function '(\w+)'.*?(\d+) bytes spill stores, (\d+) bytes spill loads.*?Used (\d+) registers",
        text, re.S)]


def test_the_chunk_attention_spills_nothing(tmp_path):
    forms = [k for k in kernels("chunk.cu", tmp_path) if "chunk_fwd_kernel" in k[0]]
    assert len(forms) == 16  # type, head dim, loader, shared prefixes or not
    assert {k[1:] for k in forms} == {(168, 0, 0)}


def test_the_attention_weights_spill_nothing(tmp_path):
    forms = [k for k in kernels("weights.cu", tmp_path) if "weights_kernel" in k[0]]
    assert len(forms) == 8
    assert {k[2:] for k in forms} == {(0, 0)}
