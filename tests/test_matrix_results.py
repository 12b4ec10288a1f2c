"""No kernel reads the result of a matrix product before it is there (see build.early_reads), or has lost what a narrowed lane mask was for."""
import importlib

import pytest

build = importlib.import_module("mojo-rl_amd.build")

EARLY = """
_Zkernel:
\tv_mfma_f32_16x16x4_f32 v[0:3], v8, v9, v[0:3]
\ts_cbranch_vccnz .LBB0_2
; %bb.1:
\ts_nop 9
\tv_add_f32_e32 v4, v0, v5
.LBB0_2:
\tv_mul_f32_e32 v6, v1, v5
\ts_endpgm
"""


def test_a_read_behind_a_branch_is_found():
    products, faults = build.early_reads(EARLY.splitlines())
    assert products == 1 and len(faults) == 1
    kernel, product, reader, waited = faults[0]
    assert kernel == "_Zkernel" and reader.startswith("v_mul_f32_e32 v6, v1") and waited == 1


@pytest.mark.parametrize("old,new", [("s_cbranch_vccnz .LBB0_2", "s_nop 9"),          # waits ahead of both
                                     ("\ts_cbranch", "\ts_nop 8\n\ts_cbranch"),        # ahead of the branch
                                     ("v6, v1, v5", "v6, v4, v5"),                      # another register
                                     ("v_mul_f32_e32 v6, v1, v5", "v_mfma_f32_16x16x4_f32 v[0:3], v8, v9, v[0:3]")])
def test_what_waits_is_not_found(old, new):
    assert build.early_reads(EARLY.replace(old, new).splitlines()) == (1 + ("mfma" in new), [])


def test_a_product_of_a_result_and_a_store_are_reads():
    for reader in ("v_mfma_f32_16x16x4_f32 v[4:7], v1, v9, v[4:7]", "global_store_dword v7, v1, s[0:1]", "ds_write_b32 v7, v1", "v_mov_b32_e32 v1, 0"):
        assert len(build.early_reads(EARLY.replace("v_mul_f32_e32 v6, v1, v5", reader).splitlines())[1]) == 1


def test_accumulation_registers_are_registers_of_their_own():
    apart = EARLY.replace("v_mfma_f32_16x16x4_f32 v[0:3], v8, v9, v[0:3]", "v_mfma_f32_16x16x4_f32 a[0:3], v8, v9, a[0:3]")
    assert build.early_reads(apart.splitlines()) == (1, [])
    faults = build.early_reads(apart.replace("v_mul_f32_e32 v6, v1, v5", "v_accvgpr_read_b32 v6, a1").splitlines())[1]
    assert len(faults) == 1 and faults[0][2].startswith("v_accvgpr_read_b32 v6, a1") and faults[0][3] == 1


def test_an_empty_mask_is_found():
    kept = "_Zkernel:\n\ts_and_saveexec_b64 s[10:11], s[6:7]\n\tv_mov_b32_e32 v17, v0\n\ts_or_b64 exec, exec, s[10:11]\n"
    assert build.empty_masks(kept.splitlines()) == []
    assert build.empty_masks(kept.replace("\tv_mov_b32_e32 v17, v0\n", "").splitlines()) == ["_Zkernel"]


def test_no_unit_reads_a_result_early():
    found = build.check_matrix_results()
    assert {"mrl_delta.hip", "mrl_delta_back.hip", "mrl_glu.hip", "mrl_muon.hip"} <= set(found)
    for unit, (products, faults, empty) in found.items():
        assert products > 0 and faults == [] and empty == [], (unit, faults[:4], empty[:4])
