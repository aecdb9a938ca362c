"""The generated code of attention over listed blocks and of products with 4-bit weights: nothing goes to scratch memory, and the build looks at every kernel of theirs that loops over tiles."""
import os
import re

import pytest

from test_lora_generated_code import CSRC, chk

KERNELS = {"attention_blocks": ("attn_blocks_kernel", "attn_blocks_parts_kernel"), "linear_w4": ("w4_rows_kernel", "w4_tiles_kernel", "w4_product_kernel")}


@pytest.mark.parametrize("unit", KERNELS)
def test_the_build_checks_every_kernel(unit):
    make = open(os.path.join(CSRC, "Makefile")).read()
    source = open(os.path.join(CSRC, unit + ".hip")).read()
    assert set(re.findall(r"check_no_scratch\.py \S*/%s-hip-\S+ (\w+)" % unit, make)) == set(KERNELS[unit])
    assert all(re.search(r"void %s\(" % name, source) for name in KERNELS[unit])


@pytest.mark.parametrize("unit", KERNELS)
def test_the_built_kernels(unit):
    text = os.path.join(CSRC, "..", "..", "build", "csrc", "%s-hip-amdgcn-amd-amdhsa-gfx950.s")
    if not os.path.exists(text % "gemm_lora"):
        pytest.skip("library not built in this tree")
    for name in KERNELS[unit]:
        assert chk.check(text % unit, name) == [], name
