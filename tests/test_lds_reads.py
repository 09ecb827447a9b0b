"""The matrix kernels read LDS by inline assembly and wait later, and the largest tile's matrix instructions are assembly: the built
code is checked for a touch of such a register before the wait and for the distances (tools/lds_reads.py), and the check itself
on small listings with a mistake in them."""
import os
import shutil

import pytest

from tools import lds_reads
from tools.kernel_resources import LLVM


def _code(text):
    lines = [ln.strip() for ln in text.strip().splitlines()]
    return [(4 * i, ln.split(None, 1)[0], ln.split(None, 1)[1] if " " in ln else "") for i, ln in enumerate(lines)]


GOOD = ["""
    ds_read_b128 v[4:7], v1
    ds_read_b64_tr_b16 v[8:9], v2 offset:512
    v_add_u32 v1, v1, v3
    s_waitcnt lgkmcnt(1)
    v_mov_b32 v10, v5
    s_waitcnt lgkmcnt(0)
    v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]
    s_endpgm
""", """
    ds_read_b32 v4, v1
    s_cbranch_scc1 1
    ds_write_b32 v2, v3
    s_waitcnt vmcnt(2) lgkmcnt(0)
    v_mov_b32 v5, v4
    s_endpgm
"""]
BAD = [("""
    ds_read_b128 v[4:7], v1
    v_mov_b32 v8, v6
    s_waitcnt lgkmcnt(0)
    s_endpgm
""", 1), ("""
    ds_read_b128 v[4:7], v1
    v_mov_b32 v5, 0
    s_waitcnt lgkmcnt(0)
    s_endpgm
""", 1), ("""
    ds_read_b32 v4, v1
    ds_read_b32 v5, v1 offset:4
    s_waitcnt vmcnt(0) lgkmcnt(1)
    v_add_f32 v6, v4, v5
    s_endpgm
""", 3), ("""
    s_nop 0
    v_mov_b32 v2, v4
    ds_read_b32 v4, v1
    s_cbranch_scc1 65533
    s_waitcnt lgkmcnt(0)
    s_endpgm
""", (1, 2)), ("""
    ds_read_b32 v4, v1
    s_cbranch_scc1 1
    ds_write_b32 v2, v3
    s_waitcnt lgkmcnt(1)
    v_mov_b32 v5, v4
    s_endpgm
""", 4), ("""
    ds_read_b32 a4, v1
    v_accvgpr_read_b32 v5, a4
    s_endpgm
""", 1)]


@pytest.mark.parametrize("text", GOOD)
def test_waited_reads_pass(text):
    bad, reads = lds_reads.check(_code(text))
    assert not bad and reads


@pytest.mark.parametrize("text,at", BAD)
def test_early_touches_are_found(text, at):
    bad, _ = lds_reads.check(_code(text))
    assert [b[0] // 4 for b in bad] == list(at if isinstance(at, tuple) else (at,))


M = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]"
FILL = ["v_mfma_f32_16x16x32_bf16 a[%d:%d], v[4:7], v[8:11], a[%d:%d]" % (r, r + 3, r, r + 3) for r in (4, 8, 12)]


@pytest.mark.parametrize("lines,at", [
    ((M, M, "s_endpgm"), ()),                                                                        # accumulation in place
    ((M, *FILL, "v_accvgpr_read_b32 v0, a1", "s_endpgm"), ()),
    ((M, *FILL[:2], "v_accvgpr_read_b32 v0, a1", "s_endpgm"), (3,)),
    ((M, "s_nop 10", "v_accvgpr_read_b32 v0, a1", "s_endpgm"), ()),
    ((M, "s_nop 9", "v_accvgpr_read_b32 v0, a1", "s_endpgm"), (2,)),
    ((M, "v_mfma_f32_16x16x32_bf16 a[4:7], a[0:3], v[8:11], a[4:7]", "s_endpgm"), (1,)),
    (("v_mov_b32 v6, 0", "s_nop 0", M, "s_endpgm"), (2,)),
    (("v_mov_b32 v6, 0", "s_nop 1", M, "s_endpgm"), ()),
    (("v_accvgpr_write_b32 a3, v0", "ds_read_b32 v20, v21", "ds_read_b32 v22, v21", M, "s_endpgm"), ()),
    ((M, "s_nop 1", "s_cbranch_scc1 65533", "v_accvgpr_read_b32 v0, a1", "s_endpgm"), (3,)),
    (("s_nop 0", M, "s_cbranch_scc1 1", "s_nop 12", "ds_write_b32 v30, a2", "s_endpgm"), (4,)),
])
def test_distances_of_matrix_instructions(lines, at):
    assert [b[0] // 4 for b in lds_reads.check_distances(_code("\n".join(lines)))] == list(at)


def test_built_matrix_kernels_wait_for_their_lds_reads():
    from diffusionmodel_amd import _lib
    if not os.path.exists(f"{LLVM}/llvm-objdump") or not shutil.which("objcopy"):
        pytest.skip("no disassembler")
    found = lds_reads.check_library(_lib.lib_path(), r"gemm_|attention|tapconv|resfuse|upfuse|ws1x1")
    # 3 operand orders x (bf16: 5 tiles, f32: 4) and 2 orders of the few-rows kernel in both types
    assert sum("gemm_kernel" in k for k in found) == 27 and sum("gemm_few_kernel" in k for k in found) == 4
    assert all(reads >= 8 for k, (_, reads) in found.items() if "gemm_kernel" in k or "gemm_few_kernel" in k)
    assert sum(bool(lds_reads.ASM_MFMA.search(k)) for k in found) == 3
    assert not {k: bad for k, (bad, _) in found.items() if bad}
