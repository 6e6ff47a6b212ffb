"""GPU tests of the wide FP8 tile's way out of shared memory: each promoter warp
sends its part of C through two staging buffers, and a tile at the edge of C
sends an odd number of blocks, so that one tile's last store and the next tile's
first may use the same buffer. Shapes whose last tile of features does that (m
mod 128 in 1..64 for 16-bit C, in 1..32 or 65..96 for f32), short K (little time
between tiles), empty groups (none), and ten tiles or more for each of the 74
CTA pairs. Whole numbers with power-of-two scales are exact: bits are compared."""
import pytest
import torch

import gemm_sm100 as gs
from fp8_util import FLOAT, Operand

pytestmark = pytest.mark.gpu
E4, VEC, BLK, N, T = gs.R_8F_E4M3, gs.SCALE_VEC128, gs.SCALE_BLK128, gs.OP_N, gs.OP_T
F32, BF16, F16 = gs.R_32F, gs.R_16BF, gs.R_16F


def _check(h, call, c, want, times=4):
    for _ in range(times):
        c.fill_(float("nan"))
        call()
        torch.cuda.synchronize()
        assert h.device_error() == 0
        bad = (c != want).sum().item()
        assert bad == 0, f"{bad} elements differ"


@pytest.mark.parametrize("m,k,ct", [(2880, 128, BF16), (2880, 256, BF16), (2880, 256, F16), (2208, 256, F32), (2272, 256, F32)])
def test_dense(handle, m, k, ct):
    n = 24576
    assert gs.plan_gemm_fp8(T, N, m, n, k, ctype=ct)[1] == 256
    gen = torch.Generator().manual_seed(m + k)
    a, b = Operand(gen, k, m, E4, BLK, True, True), Operand(gen, k, n, E4, VEC, True, True)
    c = torch.empty(n, m, dtype=FLOAT[ct], device="cuda")
    want = (b.values() @ a.values().t()).to(c.dtype)
    _check(handle, lambda: handle.gemm_fp8(T, N, m, n, k, 1.0, a.bytes, E4, a.ld, a.scale, BLK, a.lds, b.bytes, E4, b.ld, b.scale,
                                           VEC, b.lds, 0.0, c, ct, m), c, want)


@pytest.mark.parametrize("ta", [T, N])
@pytest.mark.parametrize("m,k,groups,ct", [(2880, 128, 32, BF16), (2880, 256, 32, BF16), (2208, 512, 8, F32)])
def test_ragged_columns(handle, ta, m, k, groups, ct):
    """Groups that end inside a tile, and empty ones."""
    n = 24576
    assert gs.plan_gemm_fp8(ta, N, m, n, k, groups=groups, ctype=ct)[1] == 256
    gen = torch.Generator().manual_seed(m + k + ta)
    a = Operand(gen, k if ta else m, m if ta else k, E4, BLK, bool(ta), True, batch=groups)
    b = Operand(gen, k, n, E4, VEC, True, True)
    cuts = torch.randint(0, n + 1, (groups - 1,), generator=gen).sort().values
    cuts[5] = cuts[6]
    off = [0, *cuts.tolist(), n]
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    c = torch.empty(n, m, dtype=FLOAT[ct], device="cuda")
    bv = b.values()
    want = torch.cat([bv[lo:hi] @ a.values(g).t() for g, (lo, hi) in enumerate(zip(off, off[1:]))]).to(c.dtype)
    _check(handle, lambda: handle.gemm_fp8_grouped(gs.GROUP_N, ta, N, m, n, k, groups, offsets, 1.0, a.bytes, E4, a.ld, a.stride,
                                                   a.scale, BLK, a.lds, a.stride_s, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0,
                                                   c, ct, m, 0), c, want)


@pytest.mark.parametrize("m,k,ma,ct", [(2880, 4096, VEC, BF16), (2880, 1024, BLK, BF16), (2208, 8192, BLK, F32),
                                       (2272, 8192, BLK, F32)])
def test_ragged_k_with_empty_groups(handle, m, k, ma, ct):
    """Every second group is empty: its tiles write zeros right behind a tile that may still be on its way out."""
    n, groups = 2880, 16
    assert gs.plan_gemm_fp8(N, T, m, n, k, groups=groups, ragged=gs.GROUP_K, a_mode=ma, ctype=ct)[1] == 256
    gen = torch.Generator().manual_seed(m + k)
    a, b = Operand(gen, m, k, E4, ma, False, True), Operand(gen, n, k, E4, VEC, False, True)
    step = k // (groups // 2)
    off = [(g + 1) // 2 * step for g in range(groups + 1)]
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    c = torch.empty(groups, n, m, dtype=FLOAT[ct], device="cuda")
    av, bv = a.values(), b.values()
    want = torch.stack([(bv[:, lo:hi] @ av[:, lo:hi].t()).to(c.dtype) for lo, hi in zip(off, off[1:])])
    _check(handle, lambda: handle.gemm_fp8_grouped(gs.GROUP_K, N, T, m, n, k, groups, offsets, 1.0, a.bytes, E4, a.ld, 0, a.scale,
                                                   ma, a.lds, 0, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c, ct, m, n * m),
           c, want)
