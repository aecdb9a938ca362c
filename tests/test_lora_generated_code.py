"""The generated code of linear_lora's kernels: nothing goes to scratch memory, and in the 256-wide tile nothing in its loop over K."""
import importlib.util
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-kernels_amd", "csrc")
spec = importlib.util.spec_from_file_location("check_no_scratch", os.path.join(CSRC, "check_no_scratch.py"))
chk = importlib.util.module_from_spec(spec)
spec.loader.exec_module(chk)

SPILL = "\tscratch_store_dword off, v1, off ; 4-byte Folded Spill\n"


def kernel(in_front="", inside="", behind="", branch="s_cbranch_scc1"):
    return (f"_ZN4flux16lora_ring_kernelE:\n{in_front}.LBB0_1:\n\tv_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]\n\ts_barrier\n{inside}\t{branch} .LBB0_1\n"
            f"{behind}\ts_cbranch_vccz .LBB0_2\n.LBB0_2:\n\ts_endpgm\n.Lfunc_end0:\n")


def test_the_check_finds_what_is_in_the_loop_alone(tmp_path):
    f = tmp_path / "g.s"
    for text, inside, anywhere in ((kernel(), 0, 0), (kernel(in_front=SPILL), 0, 1), (kernel(behind=SPILL), 0, 1), (kernel(inside=SPILL), 1, 1), (kernel(inside=SPILL, branch="s_branch"), 1, 1),
                                   ("_ZN4flux16lora_ring_kernelE:\n\ts_endpgm\n.Lfunc_end0:\n", 1, 0)):
        f.write_text(text)
        assert len(chk.check(str(f), "lora_ring_kernel", loop=True)) == inside and len(chk.check(str(f), "lora_ring_kernel")) == anywhere


def test_the_built_kernels():
    unit = os.path.join(CSRC, "..", "..", "build", "csrc", "%s-hip-amdgcn-amd-amdhsa-gfx950.s")
    if not os.path.exists(unit % "gemm_lora"):
        pytest.skip("library not built in this tree")
    for name in ("lora_rect_kernel", "lora_low_kernel", "lora_rows_kernel"):
        assert chk.check(unit % "gemm_lora", name) == [], name
    for name in ("gemm_nt_pair_kernel", "gemm_reduce_kernel"):
        assert chk.check(unit % "gemm_lora_pair", name) == [], name
    assert chk.check(unit % "gemm_lora", "lora_ring_kernel", loop=True) == []
    for name, lines in chk.kernels(unit % "gemm_lora", "lora_ring_kernel").items():
        loops = chk.loops_over_k(lines)
        assert loops and max(sum("v_mfma" in l for l in loop) for loop in loops) >= 128, name    # a slab: two steps of 8 x 8 fragments
