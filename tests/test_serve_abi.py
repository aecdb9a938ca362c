"""The third part of the C ABI (include/flux_hip_serve.h): every function is exported and bound, and the ctypes structures and constants are the header's (no GPU needed)."""
import ctypes
import os
import re
import subprocess

from triton_kernels import _native as nv
from triton_kernels.kernels import attention, quantization

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "flux_hip_serve.h")
STRUCTS = {"flux_w4": nv.W4, "flux_linear_w4_args": nv.LinearW4Args, "flux_select_blocks_args": nv.SelectBlocksArgs, "flux_sparse_attention_args": nv.SparseAttentionArgs}


def text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_every_declared_function_is_exported_and_bound():
    names = set(re.findall(r"\b(flux_[a-z0-9_]+)\s*\(", text()))
    assert names == set(nv.SERVE_SIGNATURES)
    assert not names & (set(nv.SIGNATURES) | set(nv.TUNE_SIGNATURES))
    version = int(re.search(r"#define FLUX_SERVE_ABI_VERSION (\d+)", text()).group(1))
    assert nv.lib().flux_serve_abi_version() == nv.SERVE_ABI_VERSION == version


def test_struct_layouts_match_the_header(tmp_path):
    assert set(re.findall(r"typedef struct (\w+)", text())) == set(STRUCTS)
    lines, want = [], []
    for name, struct in STRUCTS.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        want.append(ctypes.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append(f'printf("%zu ", offsetof({name}, {field}));')
            want.append(getattr(struct, field).offset)
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flux_hip_serve.h"\nint main(void){' + "\n".join(lines)
                   + 'printf("%d %d", FLUX_QUERY_BLOCK, FLUX_KEY_BLOCK);return 0;}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(t) for t in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want + [attention.QUERY_BLOCK, attention.KEY_BLOCK]


def test_the_layout_that_python_writes_is_the_one_of_the_header():
    comment = open(HEADER).read()
    assert quantization.GROUPS == (32, 64, 128) and "group 32, 64 or 128" in comment
    assert f"tiles of {quantization._TILE} rows x {quantization._CHUNK} columns" in comment
