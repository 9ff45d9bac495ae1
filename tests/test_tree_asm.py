"""The drafted-tree attention's LDS tile copies (CPU: compiles gfx950 assembly, runs nothing).

Every copy has the wait states that gfx950 asks for after the scalar writes it reads, M0 is written by scalar
instructions only, and the few-row kernel, whose waves wait for their copies by count, has no scratch: a spilled
register's store or reload would be counted among them."""

from __future__ import annotations

import re
import subprocess

import pytest

from tests import test_asm_hazards as hazards

FEW = [f"tree_attn_kernel<mt::{e}, {d}>" for e in ("BF16", "FP16") for d in (32, 64, 128)]
MANY = [f"tree_attn_rows_kernel<mt::{e}, {d}, {rw}>" for e, d in (("BF16", 64), ("FP16", 128), ("BF16", 32)) for rw in (2, 4, 8)]


@pytest.mark.parametrize("kernels", [FEW, MANY], ids=["few_rows", "many_rows"])
def test_copies_of_the_tree_attention(tmp_path, kernels):
    hipcc = hazards._hipcc()
    if hipcc is None:
        pytest.skip("hipcc not available")
    src, out = tmp_path / "tu.hip", tmp_path / "tu.s"
    src.write_text('#include "tree_kernels.h"\n' + "".join(f"template __global__ void mt::{k}(mt::TreeAttnParams);\n" for k in kernels))
    proc = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "--cuda-device-only", "-S",
                           "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-pass-failed",
                           "-I", hazards.CSRC, str(src), "-o", str(out)], capture_output=True, text=True, timeout=900)
    assert proc.returncode == 0, proc.stderr[-2000:]
    asm = out.read_text()
    ins = hazards._instructions(asm)
    hazards.test_every_lds_copy_has_its_wait_states(ins)
    assert not [x for x in ins if x.startswith("v_") and hazards._writes(x, {"m0"})]
    sizes = [int(x) for x in re.findall(r"; ScratchSize: (\d+)", asm)]
    assert len(sizes) == len(kernels)
    if kernels is FEW:
        assert set(sizes) == {0}
