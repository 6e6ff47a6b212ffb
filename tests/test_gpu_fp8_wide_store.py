"""GPU tests of the ways C leaves the wide FP8 tile other than whole TMA stores: added to what was there (beta), with
rows that are not multiples of 16 bytes, and at the ends of ragged groups. Whole numbers are exact: bits are compared,
and what lies behind C's rows stays."""
import pytest
import torch

import gemm_sm100 as gs
from fp8_util import FLOAT, Operand

pytestmark = pytest.mark.gpu
E4, VEC, BLK, N, T = gs.R_8F_E4M3, gs.SCALE_VEC128, gs.SCALE_BLK128, gs.OP_N, gs.OP_T
F32, BF16, F16 = gs.R_32F, gs.R_16BF, gs.R_16F


@pytest.mark.parametrize("beta", [0.0, 1.0])
@pytest.mark.parametrize("m,n,k,pad,groups,ct", [
    (2880, 3000, 640, 0, 0, BF16), (2880, 3000, 640, 0, 0, F32), (2880, 3000, 640, 0, 5, F16),   # aligned rows
    (2001, 2003, 8192, 1, 0, BF16), (2001, 2003, 8192, 0, 0, F32), (2303, 2305, 16384, 2, 3, F16),
    # aligned rows that end between 16-byte steps: a TMA store would write on to the next one
    (2303, 2305, 16384, 1, 3, F32), (2875, 3000, 640, 5, 0, BF16), (2881, 3000, 640, 15, 5, F16), (2878, 3000, 640, 2, 0, F32),
    (2817, 3000, 640, 63, 0, BF16), (2820, 3000, 640, 4, 0, F16),
])
def test_store(handle, m, n, k, pad, groups, ct, beta):
    ldc = m + pad
    assert gs.plan_gemm_fp8(T, N, m, n, k, groups=groups, ctype=ct, c_aligned=ldc * FLOAT[ct].itemsize % 16 == 0)[1] == 256
    gen = torch.Generator().manual_seed(m + n + ct)
    a, b = Operand(gen, k, m, E4, BLK, True, True, batch=max(groups, 1)), Operand(gen, k, n, E4, VEC, True, True)
    off = [0, n] if not groups else [5, *(n * g // groups + 3 * g for g in range(1, groups)), n - 7]
    c0 = torch.randint(-3, 4, (n, ldc), generator=gen).to(FLOAT[ct]).cuda()
    want, bv = c0.clone(), b.values()
    for g, (lo, hi) in enumerate(zip(off, off[1:])):
        full = 0.125 * (bv[lo:hi] @ a.values(g).t()) + beta * c0[lo:hi, :m].double()
        want[lo:hi, :m] = full.to(want.dtype)
    c = c0.clone()
    if groups:
        handle.gemm_fp8_grouped(gs.GROUP_N, T, N, m, n, k, groups, torch.tensor(off, dtype=torch.int32, device="cuda"), 0.125,
                                a.bytes, E4, a.ld, a.stride, a.scale, BLK, a.lds, a.stride_s, b.bytes, E4, b.ld, b.scale, VEC,
                                b.lds, beta, c, ct, ldc, 0)
    else:
        handle.gemm_fp8(T, N, m, n, k, 0.125, a.bytes, E4, a.ld, a.scale, BLK, a.lds, b.bytes, E4, b.ld, b.scale, VEC, b.lds, beta,
                        c, ct, ldc)
    torch.cuda.synchronize()
    assert handle.device_error() == 0
    assert torch.equal(c, want)


@pytest.mark.parametrize("m,ct", [(2873, BF16), (2886, F16), (2303, F32), (2880, BF16)])
def test_store_of_groups_into_a_wider_array(handle, m, ct):
    """Each group's C is a part of a larger matrix, whose other elements stay."""
    n, k, groups, ldc = 2880, 8192, 16, 3008
    assert gs.plan_gemm_fp8(N, T, m, n, k, groups=groups, ragged=gs.GROUP_K, ctype=ct)[1] == 256
    gen = torch.Generator().manual_seed(m)
    a, b = Operand(gen, m, k, E4, BLK, False, True), Operand(gen, n, k, E4, VEC, False, True)
    off = [512 * g for g in range(groups)] + [k]
    off[4] = off[5]
    c0 = torch.randint(-3, 4, (groups, n + 1, ldc), generator=gen).to(FLOAT[ct]).cuda()
    want, av, bv = c0.clone(), a.values(), b.values()
    for g, (lo, hi) in enumerate(zip(off, off[1:])):
        want[g, :n, :m] = (bv[:, lo:hi] @ av[:, lo:hi].t()).to(want.dtype)
    c = c0.clone()
    handle.gemm_fp8_grouped(gs.GROUP_K, N, T, m, n, k, groups, torch.tensor(off, dtype=torch.int32, device="cuda"), 1.0, a.bytes,
                            E4, a.ld, 0, a.scale, BLK, a.lds, 0, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c, ct, ldc,
                            (n + 1) * ldc)
    torch.cuda.synchronize()
    assert handle.device_error() == 0
    assert torch.equal(c, want)
