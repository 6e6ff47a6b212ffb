"""CPU tests of the FP8 products' tile plan for every kind of operand and C."""
import pytest

import gemm_sm100 as gs

N, T, VEC, BLK = gs.OP_N, gs.OP_T, gs.SCALE_VEC128, gs.SCALE_BLK128


def test_defaults_are_the_other_calls():
    for args, kw in (((T, N, 8192, 8192, 8192), {}), ((T, N, 4096, 16, 4096), {}), ((T, N, 2048, 128, 2048), dict(groups=64)),
                     ((N, T, 2880, 2880, 4096), dict(groups=16, ragged=gs.GROUP_K))):
        assert gs.plan_gemm_fp8(*args, **kw) == gs.plan_gemm_fp8(*args, a_mode=BLK, b_mode=VEC, ctype=gs.R_16BF, c_aligned=True, **kw)


def test_scales_of_rows_and_columns_cost_the_wide_tile_more():
    """1358 against 776 cycles a K block: 16 experts' weight gradients take 128 x 128 tiles where blocks take pairs."""
    args, kw = (N, T, 2048, 2048, 16384), dict(groups=16, ragged=gs.GROUP_K, ctype=gs.R_32F)
    assert gs.plan_gemm_fp8(*args, a_mode=VEC, **kw)[1:3] == (128, 1)
    assert gs.plan_gemm_fp8(*args, a_mode=BLK, **kw)[1:3] == (256, 2)


def test_a_wide_tile_needs_an_aligned_c_to_be_cheap():
    args = (T, N, 4096, 4096, 512)
    assert gs.plan_gemm_fp8(*args)[1] == 256
    assert gs.plan_gemm_fp8(*args, c_aligned=False)[1] < 256
    assert gs.plan_gemm_fp8(T, N, 8192, 8192, 32768, c_aligned=False)[1] == 256  # long sums: the store matters less


@pytest.mark.parametrize("bad", [dict(a_mode=3), dict(b_mode=0), dict(ctype=gs.R_8I), dict(ctype=gs.R_64F)])
def test_refusals(bad):
    assert gs.plan_gemm_fp8(T, N, 256, 256, 256, **bad)[0] == gs.STATUS_INVALID_VALUE


@pytest.mark.parametrize("m,k,a_mode,ctype", [(2880, 4096, VEC, gs.R_16BF), (2880, 1024, BLK, gs.R_16BF),
                                              (2208, 8192, BLK, gs.R_32F), (2272, 8192, BLK, gs.R_32F)])
def test_weight_gradients_whose_last_tile_is_part(m, k, a_mode, ctype):
    """The cases of tests/test_gpu_fp8_staging.py that are there for the pair tile."""
    assert gs.plan_gemm_fp8(N, T, m, 2880, k, groups=16, ragged=gs.GROUP_K, a_mode=a_mode, ctype=ctype) == (0, 256, 2, 1)


@pytest.mark.parametrize("m,k,groups", [(2208, 256, 0), (2272, 256, 0), (2208, 512, 8)])
def test_f32_products_whose_last_tile_is_part(m, k, groups):
    assert gs.plan_gemm_fp8(T, N, m, 24576, k, groups=groups, ctype=gs.R_32F) == (0, 256, 2, 1)
