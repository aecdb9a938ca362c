"""The second part of the C ABI (include/flux_hip_tune.h): every function is exported and bound, the ctypes structures have the
layout of the header's, and bad arguments are refused before anything is launched (no GPU needed)."""
import ctypes
import os
import re
import subprocess

import pytest

from triton_kernels import _native as nv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "flux_hip_tune.h")
STRUCTS = {"flux_layer_norm_fwd_args": nv.LayerNormFwdArgs, "flux_layer_norm_bwd_args": nv.LayerNormBwdArgs, "flux_rope_ids": nv.RopeIds,
           "flux_rope_nd_args": nv.RopeNdArgs, "flux_linear_lora_args": nv.LinearLoraArgs}


def text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_every_declared_function_is_exported_and_bound():
    names = set(re.findall(r"\b(flux_[a-z0-9_]+)\s*\(", text()))
    assert names == set(nv.TUNE_SIGNATURES)
    assert not names & set(nv.SIGNATURES)
    version = int(re.search(r"#define FLUX_TUNE_ABI_VERSION (\d+)", text()).group(1))
    assert nv.lib().flux_tune_abi_version() == nv.TUNE_ABI_VERSION == version


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
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flux_hip_tune.h"\nint main(void){' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    assert [int(t) for t in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()] == want


BUF = ctypes.create_string_buffer(256)
P = ctypes.addressof(BUF)


def layer_norm_args(**kw):
    return nv.LayerNormFwdArgs(**{**dict(x=P, w=P, b=P, y=P, batch=2, seq=3, x_sb=24, x_sl=8, groups=1, n=8, x_dtype=0, w_dtype=0, eps=1e-5), **kw})


@pytest.mark.parametrize("change,rc", [(dict(x=None), -1), (dict(y=None), -1), (dict(mean=P), -1), (dict(batch=-1), -2), (dict(seq=-1), -2), (dict(n=0), -2), (dict(groups=3), -2),
                                       (dict(n=65537), -5), (dict(batch=2**20, seq=2**20), -2), (dict(x_dtype=2), -3), (dict(x_dtype=1), -3), (dict(batch=0, x=None), 0)])
def test_layer_norm_refusals(change, rc):
    assert nv.lib().flux_layer_norm(ctypes.byref(layer_norm_args(**change)), None) == rc
    assert nv.lib().flux_layer_norm(None, None) == -1


@pytest.mark.parametrize("change,ws,rc", [(dict(dy=None), 1 << 20, -1), (dict(mean=None), 1 << 20, -1), (dict(groups=3), 1 << 20, -2), (dict(seq=300), 0, -1), (dict(n=70000), 1 << 20, -5),
                                          (dict(x_dtype=1), 1 << 20, -3), (dict(dx=None, dw=None, db=None), 0, 0), (dict(batch=0), 1 << 20, -2), (dict(batch=0, dw=None, db=None), 0, 0)])
def test_layer_norm_bwd_refusals(change, ws, rc):
    a = nv.LayerNormBwdArgs(**{**dict(dy=P, x=P, w=P, mean=P, rstd=P, dx=P, dw=P, db=P, batch=2, seq=3, dy_sb=24, dy_sl=8, x_sb=24, x_sl=8, groups=1, n=8, x_dtype=0, w_dtype=0), **change})
    assert nv.lib().flux_layer_norm_bwd(ctypes.byref(a), P if ws else None, ws, None) == rc


def test_layer_norm_bwd_workspace():
    a = nv.LayerNormBwdArgs(dy=P, x=P, w=P, mean=P, rstd=P, dx=P, dw=P, db=P, batch=4, seq=1000, dy_sb=8000, dy_sl=8, x_sb=8000, x_sl=8, groups=4, n=8, x_dtype=0, w_dtype=0)
    need = nv.lib().flux_layer_norm_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0 and need % (2 * 4 * 8 * 4) == 0
    assert nv.lib().flux_layer_norm_bwd(ctypes.byref(a), P, need - 1, None) == -2      # too small
    assert nv.lib().flux_layer_norm_bwd(ctypes.byref(a), P + 2, need, None) == -1      # not aligned
    a.seq = 128                                                                        # few rows: one launch, without parts
    assert nv.lib().flux_layer_norm_bwd_workspace_bytes(ctypes.byref(a)) == 0
    a.seq, a.dw, a.db = 1000, None, None
    assert nv.lib().flux_layer_norm_bwd_workspace_bytes(ctypes.byref(a)) == 0


def rope_ids(**kw):
    axes = kw.pop("axes", (16, 24, 24))
    return nv.RopeIds(**{**dict(ids=P, sb=0, sl=3, sa=1, theta=10000.0, dtype=0, n_axes=len(axes), axes_dim=(ctypes.c_int32 * 8)(*axes[:8])), **kw})


IDS_REFUSALS = [(dict(ids=None), -1), (dict(dtype=4), -3), (dict(dtype=-1), -3), (dict(n_axes=0), -2), (dict(n_axes=9), -2), (dict(axes=(16, 23, 25)), -2), (dict(axes=(64, 0)), -2),
                (dict(axes=(-2, 66)), -2), (dict(axes=(256, 258)), -2), (dict(theta=0.0), -2), (dict(theta=float("inf")), -2), (dict(theta=float("nan")), -2)]


@pytest.mark.parametrize("change,rc", IDS_REFUSALS)
def test_rope_ids_refusals(change, rc):
    at = rope_ids(**change)
    src = nv.Src4(P, 0, 0, 0)
    a = nv.RopeNdArgs(q=src, k=src, q_out=P, k_out=P, at=at, B=1, Hq=1, Hk=1, L=1, D=64)
    assert nv.lib().flux_rope_nd(ctypes.byref(a), None) == rc
    assert nv.lib().flux_rope_table(ctypes.byref(at), P, 1, 1, None) == rc


@pytest.mark.parametrize("change,rc", [(dict(D=62), -2), (dict(B=-1), -2), (dict(L=-1), -2), (dict(Hq=-1), -2), (dict(L=2**31), -2), (dict(B=65536), -2), (dict(q_out=None), -1), (dict(k=nv.Src4()), -1),
                                       (dict(dtype=2), -3), (dict(L=0), 0), (dict(B=0), 0), (dict(Hq=0, Hk=0), 0)])
def test_rope_nd_refusals(change, rc):
    src = nv.Src4(P, 0, 0, 0)
    a = nv.RopeNdArgs(**{**dict(q=src, k=src, q_out=P, k_out=P, at=rope_ids(), B=1, Hq=1, Hk=1, L=1, D=64), **change})
    assert nv.lib().flux_rope_nd(ctypes.byref(a), None) == rc
    assert nv.lib().flux_rope_nd(None, None) == -1


def test_rope_table_refusals():
    at, call = ctypes.byref(rope_ids()), nv.lib().flux_rope_table
    assert call(at, None, 1, 1, None) == -1 and call(None, P, 1, 1, None) == -1 and call(at, P, -1, 1, None) == -2 and call(at, P, 1, 2**31, None) == -2
    assert call(at, P + 4, 1, 1, None) == -4 and call(at, P, 2**20, 2**20, None) == -2 and call(at, P, 0, 5, None) == 0


def lora_args(**kw):
    return nv.LinearLoraArgs(**{**dict(x=P, w=P, bias=P, y=P, lora_a=P, lora_b=P, adapter=P, scaling=P, M=4, N=16, K=8, ldx=8, ldw=8, ldy=16, requests=2, adapters=3, rank=4), **kw})


WS = ctypes.create_string_buffer(1 << 16)
WS_AT = (ctypes.addressof(WS) + 255) // 256 * 256


@pytest.mark.parametrize("change,rc", [(dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1), (dict(lora_a=None), -1), (dict(lora_b=None), -1), (dict(adapter=None), -1), (dict(M=-1), -2),
                                       (dict(N=2**31), -2), (dict(ldx=7), -2), (dict(ldw=7), -2), (dict(ldy=15), -2), (dict(adapters=0), -2), (dict(rank=0), -2), (dict(rank=257), -2),
                                       (dict(requests=3), -2), (dict(requests=0), -2), (dict(requests=-4), -2), (dict(act=2), -6), (dict(M=2**28, requests=1), -2),
                                       (dict(M=2**20, N=2**14, K=7, ldx=7, ldw=7, ldy=2**14), -2), (dict(N=2**28, ldy=2**28), -2), (dict(M=0), 0), (dict(N=0), 0)])
def test_linear_lora_refusals(change, rc):
    a = ctypes.byref(lora_args(**change))
    assert nv.lib().flux_linear_lora_bf16(a, WS_AT, 1 << 15, None) == rc
    if rc:
        assert nv.lib().flux_linear_lora_workspace_bytes(a) == nv.lib().flux_linear_lora_least_bytes(a) == 0


def test_linear_lora_workspace():
    call, a = nv.lib().flux_linear_lora_bf16, lora_args()
    least = nv.lib().flux_linear_lora_least_bytes(ctypes.byref(a))
    assert least == nv.lib().flux_linear_lora_workspace_bytes(ctypes.byref(a)) == 512                # 4 rows of 32 values, 4 adapters' numbers
    assert call(ctypes.byref(a), None, 1 << 15, None) == -1 and call(ctypes.byref(a), WS_AT + 16, 1 << 15, None) == -1
    assert call(ctypes.byref(a), WS_AT, least - 1, None) == -2 and call(None, WS_AT, least, None) == -1
    cut = lora_args(M=64, N=2048, K=16384, ldx=16384, ldw=16384, ldy=2048, rank=40)
    assert nv.lib().flux_linear_lora_least_bytes(ctypes.byref(cut)) == 64 * 64 * 2 + 256
    assert nv.lib().flux_linear_lora_workspace_bytes(ctypes.byref(cut)) > 64 * 64 * 2 + 256            # K in parts
