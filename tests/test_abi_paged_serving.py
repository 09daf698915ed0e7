"""The argument structs of the rotary and page entry points: the ctypes layout against the C layout that gcc computes."""
import ctypes
import os
import subprocess

from attention_kernel_triton_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {
    "akt_chunk_paged_args": _lib.ChunkPagedArgs,
    "akt_rotary_args": _lib.RotaryArgs,
    "akt_append_rotary_args": _lib.AppendRotaryArgs,
    "akt_page_pool": _lib.PagePool,
    "akt_fork_paged_args": _lib.ForkPagedArgs,
    "akt_compact_paged_args": _lib.CompactPagedArgs,
}


def test_ctypes_structs_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "akt.h"', "int main(void){"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    lines.append("return 0;}")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    seen = 0
    for line in filter(None, out):
        cname, field, val = line.split()
        py = STRUCTS[cname]
        assert (ctypes.sizeof(py) if field == "size" else getattr(py, field).offset) == int(val), (cname, field)
        seen += 1
    assert seen == sum(len(s._fields_) + 1 for s in STRUCTS.values())
