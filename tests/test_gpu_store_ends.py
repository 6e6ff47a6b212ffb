"""GPU tests of C's column ends in the tensor-core kernels (f16, bf16, int8, tf32): leading dimensions above m that TMA
can address, with m between its 16-byte steps. What lies behind a column belongs to the caller (padding, or another part of a
wider matrix) and has to stay. Whole numbers are exact: bits are compared, behind the columns too."""
import pytest
import torch

import gemm_sm100 as gs

pytestmark = pytest.mark.gpu
N, T = gs.OP_N, gs.OP_T
TORCH = {gs.R_32F: torch.float32, gs.R_16F: torch.float16, gs.R_16BF: torch.bfloat16, gs.R_8I: torch.int8, gs.R_32I: torch.int32}
TYPES = [(gs.R_16F, gs.R_32F), (gs.R_16F, gs.R_16F), (gs.R_16BF, gs.R_16BF), (gs.R_16BF, gs.R_32F), (gs.R_8I, gs.R_32I)]
SHAPES = [(297, 300, 64), (301, 520, 192), (511, 260, 128), (1, 40, 64), (2302, 1030, 256)]  # m, n, k


def problem(gen, batch, m, n, k, dt, ct, gap):
    """A (op T) and B (op N) of whole numbers, C in columns of ldc > m with `gap` more columns behind each matrix, and C
    as it has to be."""
    a, b = (torch.randint(-2, 3, (batch, x, k), generator=gen) for x in (m, n))
    ldc = (m + 15) // 16 * 16 + 16
    c0 = torch.randint(-3, 4, (batch, n + gap, ldc), generator=gen)
    want = c0.clone()
    want[:, :n, :m] = torch.bmm(b.double(), a.double().transpose(1, 2)).long()
    return a.to(TORCH[dt]).cuda(), b.to(TORCH[dt]).cuda(), c0.to(TORCH[ct]).cuda(), want.to(TORCH[ct]).cuda(), ldc


def compute(dt):
    return gs.COMPUTE_32I if dt == gs.R_8I else gs.COMPUTE_32F


@pytest.mark.parametrize("algo", [gs.GEMM_DEFAULT, 0, 1, 2])
@pytest.mark.parametrize("dt,ct", TYPES)
@pytest.mark.parametrize("batch", [1, 3])
def test_strided(handle, dt, ct, algo, batch):
    for m, n, k in SHAPES:
        a, b, c, want, ldc = problem(torch.Generator().manual_seed(m + dt), batch, m, n, k, dt, ct, 1)
        handle.gemm_strided_batched_ex(T, N, m, n, k, 1.0, a, dt, k, m * k, b, dt, k, n * k, 0.0, c, ct, ldc, (n + 1) * ldc, batch,
                                       compute(dt), algo=algo)
        torch.cuda.synchronize()
        assert handle.last_kernels() & (gs.KERNEL_TC_F16 | gs.KERNEL_TC_BF16 | gs.KERNEL_TC_I8)
        assert torch.equal(c, want), (m, n, k)


@pytest.mark.parametrize("dt,ct", TYPES)
@pytest.mark.parametrize("batch", [5, 70])  # maps built in the kernel, and by a kernel of their own
def test_pointer_arrays(handle, dt, ct, batch):
    m, n, k = 301, 130, 64
    a, b, c, want, ldc = problem(torch.Generator().manual_seed(batch), batch, m, n, k, dt, ct, 2)
    arrays = [torch.tensor([t[i].data_ptr() for i in range(batch)], dtype=torch.int64, device="cuda") for t in (a, b, c)]
    handle.gemm_batched_ex(T, N, m, n, k, 1.0, arrays[0], dt, k, arrays[1], dt, k, 0.0, arrays[2], ct, ldc, batch, compute(dt))
    torch.cuda.synchronize()
    assert torch.equal(c, want)


def test_fast_tf32(handle):
    m, n, k = 1021, 1000, 1024
    a, b, c, want, ldc = problem(torch.Generator().manual_seed(1), 1, m, n, k, gs.R_32F, gs.R_32F, 0)
    handle.gemm_ex(T, N, m, n, k, 1.0, a, gs.R_32F, k, b, gs.R_32F, k, 0.0, c, gs.R_32F, ldc, gs.COMPUTE_32F_FAST_TF32)
    torch.cuda.synchronize()
    assert handle.last_kernels() & gs.KERNEL_TC_TF32
    assert torch.equal(c, want)


def test_split_k(handle):
    m, n, k = 253, 256, 16384
    assert gs.plan_tile(T, N, m, n, k, gs.R_16F, gs.R_32F, gs.COMPUTE_32F)[2] > 1
    a, b, c, want, ldc = problem(torch.Generator().manual_seed(2), 1, m, n, k, gs.R_16F, gs.R_32F, 1)
    handle.gemm_ex(T, N, m, n, k, 1.0, a, gs.R_16F, k, b, gs.R_16F, k, 0.0, c, gs.R_32F, ldc, gs.COMPUTE_32F)
    torch.cuda.synchronize()
    assert torch.equal(c, want)
