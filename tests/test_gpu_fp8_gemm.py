"""GPU tests of the block-scaled FP8 products (gs_gemm_fp8, gs_gemm_fp8_grouped)
against float64. Small whole numbers with power-of-two scales make every sum
exact, so layout and masking mistakes show as unequal bits; random values with
arbitrary scales are held to a bound derived in fp8_util.bound."""
import pytest
import torch

import gemm_sm100 as gs
from fp8_util import FLOAT, Operand, blocks, bound, product

pytestmark = pytest.mark.gpu
E4, E5, VEC, BLK, N, T = gs.R_8F_E4M3, gs.R_8F_E5M2, gs.SCALE_VEC128, gs.SCALE_BLK128, gs.OP_N, gs.OP_T


def operands(gen, ta, tb, m, n, k, ma, mb, at=E4, bt=E4, integer=True, pad=0, batch=1):
    a = Operand(gen, k if ta else m, m if ta else k, at, ma, bool(ta), integer, pad, batch)
    b = Operand(gen, n if tb else k, k if tb else n, bt, mb, not tb, integer, pad)
    return a, b


def run_gemm(h, a, b, ta, tb, m, n, k, ct, alpha=1.0, beta=0.0, c0=None, ldc=None):
    ldc = ldc or m
    c = torch.full((n, ldc), float("nan"), dtype=FLOAT[ct], device="cuda") if c0 is None else c0.clone()
    h.gemm_fp8(ta, tb, m, n, k, alpha, a.bytes, a.type, a.ld, a.scale, a.mode, a.lds, b.bytes, b.type, b.ld, b.scale,
               b.mode, b.lds, beta, c, ct, ldc)
    torch.cuda.synchronize()
    assert h.device_error() == 0
    assert h.last_kernels() == gs.KERNEL_TC_F8
    return c


SHAPES = [(1, 1, 1), (128, 1, 128), (130, 3, 129), (256, 32, 256), (77, 33, 300), (300, 64, 1000), (129, 100, 640),
          (384, 128, 127), (257, 200, 513), (512, 300, 384), (640, 513, 1152), (100, 260, 40)]


@pytest.mark.parametrize("ta,tb", [(T, N), (N, N), (N, T), (T, T)])
@pytest.mark.parametrize("ma,mb", [(BLK, VEC), (VEC, VEC), (VEC, BLK), (BLK, BLK)])
def test_products_are_exact_on_whole_numbers(handle, ta, tb, ma, mb):
    gen = torch.Generator().manual_seed(ta * 31 + tb * 7 + ma * 3 + mb)
    for m, n, k in SHAPES:
        a, b = operands(gen, ta, tb, m, n, k, ma, mb, bt=E5 if (m + n) % 2 else E4, pad=m % 2)
        got = run_gemm(handle, a, b, ta, tb, m, n, k, gs.R_32F)
        ref, _ = product(a.values(), b.values())
        assert torch.equal(got.double(), ref), (m, n, k)


@pytest.mark.parametrize("ct", [gs.R_32F, gs.R_16F, gs.R_16BF])
@pytest.mark.parametrize("m,n,k,ta,tb,ma,mb", [
    (512, 512, 4096, T, N, BLK, VEC), (384, 7, 2048, T, N, BLK, VEC), (640, 384, 1500, N, T, VEC, VEC),
    (256, 100, 3000, N, N, BLK, VEC), (200, 260, 999, T, T, VEC, BLK), (4096, 16, 4096, T, N, BLK, VEC),
])
def test_random_values_and_scales(handle, ct, m, n, k, ta, tb, ma, mb):
    gen = torch.Generator().manual_seed(m + n + k)
    a, b = operands(gen, ta, tb, m, n, k, ma, mb, bt=E5 if tb else E4, integer=False, pad=1)
    b.scale.mul_(1e-4 if tb else 1e-2)  # f16 results stay in range
    alpha, beta = 0.75, 0.5
    c0 = torch.randn(n, m + 3, generator=gen).to(FLOAT[ct]).cuda()
    got = run_gemm(handle, a, b, ta, tb, m, n, k, ct, alpha, beta, c0, m + 3)
    ref, mag = product(a.values(), b.values())
    ref, mag = alpha * ref + beta * c0[:, :m].double(), alpha * mag + beta * c0[:, :m].double().abs()
    err = (got[:, :m].double() - ref).abs()
    assert bool((err <= bound(ref, mag, k, ct)).all()), float((err / bound(ref, mag, k, ct)).max())
    assert torch.equal(got[:, m:], c0[:, m:])  # the padding of C stays


@pytest.mark.parametrize("ct", [gs.R_32F, gs.R_16BF])
def test_k_zero_scales_c(handle, ct):
    c0 = torch.arange(12.0).view(3, 4).to(FLOAT[ct]).cuda()
    for beta, want in ((0.0, torch.zeros_like(c0)), (0.5, c0 * 0.5)):
        c = c0.clone() if beta else torch.full_like(c0, float("nan"))
        handle.gemm_fp8(T, N, 4, 3, 0, 1.0, None, E4, 16, None, BLK, 1, None, E4, 16, None, VEC, 3, beta, c, ct, 4)
        torch.cuda.synchronize()
        assert torch.equal(c, want)


def test_nan_and_zero_scales_stay_in_their_rows_and_columns(handle):
    gen = torch.Generator().manual_seed(5)
    m, n, k = 300, 70, 400
    a, b = operands(gen, T, N, m, n, k, VEC, VEC)
    a.scale[0, 1, 7] = float("nan")
    b.bytes.view(torch.uint8)[0, 9, 3] = 0x7F  # E4M3's NaN
    b.scale[0, :, 20] = 0.0
    got = run_gemm(handle, a, b, T, N, m, n, k, gs.R_32F)
    ref, _ = product(a.values(), b.values())
    assert torch.equal(got.isnan(), ref.isnan())
    assert int(ref.isnan().sum()) == n + m - 1
    assert torch.equal(got[~ref.isnan()].double(), ref[~ref.isnan()])


def _offsets(gen, groups, rows, align=1, first=0):
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=gen).sort().values.tolist()
    sizes = [y - x for x, y in zip([0] + cuts, cuts + [rows])]
    if groups > 2:
        sizes[1] = 0  # an empty group among them
    off = [first]
    for s in sizes:
        off.append(off[-1] + (s + align - 1) // align * align)
    return off


@pytest.mark.parametrize("ta", [T, N])
@pytest.mark.parametrize("groups,rows,m,k,ct", [(1, 40, 200, 256, gs.R_32F), (5, 7, 129, 300, gs.R_32F),
                                                (6, 1000, 384, 200, gs.R_32F), (64, 128, 256, 384, gs.R_16BF),
                                                (3, 2000, 300, 520, gs.R_16F), (200, 90, 128, 128, gs.R_32F)])
def test_ragged_columns(handle, ta, groups, rows, m, k, ct):
    gen = torch.Generator().manual_seed(groups + rows)
    off = _offsets(gen, groups, rows, first=3)
    n = off[-1] + 9  # columns behind the last group
    a, b = operands(gen, ta, N, m, n, k, BLK, VEC, batch=groups, pad=1)
    c = torch.full((n, m), 7.0, dtype=FLOAT[ct], device="cuda")
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    handle.gemm_fp8_grouped(gs.GROUP_N, ta, N, m, n, k, groups, offsets, 1.0, a.bytes, E4, a.ld, a.stride, a.scale, BLK, a.lds,
                            a.stride_s, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c, ct, m, 0)
    torch.cuda.synchronize()
    assert handle.device_error() == 0
    bv = b.values()
    assert bool((c[:off[0]] == 7).all()) and bool((c[off[-1]:] == 7).all())
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        ref, _ = product(a.values(g), bv[lo:hi])
        assert torch.equal(c[lo:hi], ref.to(c.dtype)), g


def test_ragged_columns_with_one_a_for_all_and_beta(handle):
    gen = torch.Generator().manual_seed(3)
    m, n, k, off = 160, 50, 128, [0, 20, 20, 50]
    a, b = operands(gen, T, N, m, n, k, VEC, VEC)
    c0 = torch.randint(-3, 4, (n, m), generator=gen).float().cuda()
    c = c0.clone()
    handle.gemm_fp8_grouped(gs.GROUP_N, T, N, m, n, k, 3, torch.tensor(off, dtype=torch.int32, device="cuda"), 2.0, a.bytes, E4,
                            a.ld, 0, a.scale, VEC, a.lds, 0, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 1.0, c, gs.R_32F, m, 0)
    torch.cuda.synchronize()
    ref, _ = product(a.values(), b.values())
    assert torch.equal(c.double(), 2 * ref + c0.double())


@pytest.mark.parametrize("off", [[0, 500, 20, -7, 30], [-5, -1, 10, 4000, 4000], [9, 3, 2, 1, 0]])
def test_ragged_columns_with_offsets_out_of_order_stay_in_bounds(handle, off):
    """Clamped to the operand and never decreasing: the documented reading of such offsets."""
    gen = torch.Generator().manual_seed(8)
    m, n, k, groups = 128, 40, 128, 4
    a, b = operands(gen, T, N, m, n, k, BLK, VEC, batch=groups)
    c = torch.full((n, m), 7.0, device="cuda")
    handle.gemm_fp8_grouped(gs.GROUP_N, T, N, m, n, k, groups, torch.tensor(off, dtype=torch.int32, device="cuda"), 1.0, a.bytes,
                            E4, a.ld, a.stride, a.scale, BLK, a.lds, a.stride_s, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c,
                            gs.R_32F, m, 0)
    torch.cuda.synchronize()
    fixed, top = [], 0
    for x in off:
        top = max(top, min(x, n))
        fixed.append(top)
    want = torch.full((n, m), 7.0, dtype=torch.float64, device="cuda")
    for g in range(groups):
        want[fixed[g]:fixed[g + 1]] = product(a.values(g), b.values()[fixed[g]:fixed[g + 1]])[0]
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("ta,tb,ma,mb", [(N, T, VEC, VEC), (T, N, VEC, VEC), (N, T, BLK, VEC), (N, N, BLK, BLK)])
def test_ragged_k(handle, ta, tb, ma, mb):
    gen = torch.Generator().manual_seed(ma + mb)
    m, n, groups = 200, 150, 5
    off = _offsets(gen, groups, 1500, 128, 128)
    k = off[-1] + 100           # the last group ends inside a block, where K ends
    off[-1] = k
    a, b = operands(gen, ta, tb, m, n, k, ma, mb)
    c0 = torch.randint(-3, 4, (groups, n, m), generator=gen).float().cuda()
    for beta in (0.0, 1.0):
        c = c0.clone()
        handle.gemm_fp8_grouped(gs.GROUP_K, ta, tb, m, n, k, groups, torch.tensor(off, dtype=torch.int32, device="cuda"), 1.0,
                                a.bytes, E4, a.ld, 0, a.scale, ma, a.lds, 0, b.bytes, E4, b.ld, b.scale, mb, b.lds, beta, c,
                                gs.R_32F, m, n * m)
        torch.cuda.synchronize()
        assert handle.device_error() == 0
        av, bv = a.values(), b.values()
        for g in range(groups):
            ref, _ = product(av[:, off[g]:off[g + 1]], bv[:, off[g]:off[g + 1]])
            assert torch.equal(c[g].double(), ref + beta * c0[g].double()), g


def test_ragged_k_reports_offsets_that_are_not_whole_blocks(cuda):
    gen = torch.Generator().manual_seed(1)
    m, n, k = 64, 64, 512
    a, b = operands(gen, N, T, m, n, k, VEC, VEC)
    with gs.Handle() as h:
        c = torch.full((2, n, m), 7.0, device="cuda")
        h.gemm_fp8_grouped(gs.GROUP_K, N, T, m, n, k, 2, torch.tensor([0, 100, 512], dtype=torch.int32, device="cuda"), 1.0,
                           a.bytes, E4, a.ld, 0, a.scale, VEC, a.lds, 0, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c,
                           gs.R_32F, m, n * m)
        assert h.device_error() == 2
        assert bool((c == 7).all())


def test_results_do_not_depend_on_the_run(handle):
    gen = torch.Generator().manual_seed(11)
    a, b = operands(gen, T, N, 512, 24, 4096, BLK, VEC, integer=False)
    first = run_gemm(handle, a, b, T, N, 512, 24, 4096, gs.R_32F)
    for _ in range(3):
        assert torch.equal(run_gemm(handle, a, b, T, N, 512, 24, 4096, gs.R_32F), first)


def test_two_graphs_of_one_handle_run_at_once(cuda):
    gen = torch.Generator().manual_seed(12)
    sets = [operands(gen, T, N, 256, 8 + 8 * i, 2048, BLK, VEC) for i in range(2)]
    with gs.Handle() as h:
        outs, graphs, streams = [], [], []
        for i, (a, b) in enumerate(sets):
            s = torch.cuda.Stream()
            n = 8 + 8 * i
            c = torch.zeros(n, 256, device="cuda")
            h.set_stream(s)

            def call():
                h.gemm_fp8(T, N, 256, n, 2048, 1.0, a.bytes, E4, a.ld, a.scale, BLK, a.lds, b.bytes, E4, b.ld, b.scale, VEC,
                           b.lds, 0.0, c, gs.R_32F, 256)

            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                call()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                call()
            c.zero_()
            outs.append(c)
            graphs.append(g)
            streams.append(s)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, (a, b) in zip(outs, sets):
            assert torch.equal(c.double(), product(a.values(), b.values())[0])
        assert h.device_error() == 0
        del graphs, g


@pytest.mark.parametrize("m,n,k,tb,mb", [(2048, 2048, 1024, N, VEC), (4096, 16, 4096, N, VEC), (1024, 512, 1024, N, BLK),
                                         (256, 4096, 1024, T, VEC)])
def test_wait_that_runs_out_ends_the_kernel_and_is_reported(cuda, m, n, k, tb, mb):
    """As test_gpu_wait_limit.py does for the other tensor-core kernels: the producer leaves a K block out (no copy, nothing
    issued after it), so the waits for it run out after a millisecond; the call is reported and the next one is right."""
    gen = torch.Generator().manual_seed(m)
    a, b = operands(gen, T, tb, m, n, k, BLK if tb == N else VEC, mb)
    with gs.Handle() as h:
        h.set_wait_limit(2_000_000)
        h.debug_skip_kblock(1)
        c = torch.empty(n, m, device="cuda")
        h.gemm_fp8(T, tb, m, n, k, 1.0, a.bytes, a.type, a.ld, a.scale, a.mode, a.lds, b.bytes, b.type, b.ld, b.scale, b.mode, b.lds,
                   0.0, c, gs.R_32F, m)
        word = h.device_error()
    assert word & 1 and (word >> 8) & 0xFF in (1, 2, 3, 4, 6, 7), hex(word)
    with gs.Handle() as h:
        h.set_wait_limit(2_000_000)  # healthy pipelines do not notice it
        assert torch.equal(run_gemm(h, a, b, T, tb, m, n, k, gs.R_32F).double(), product(a.values(), b.values())[0])


@pytest.mark.parametrize("bn,m,n,k,groups", [(32, 4096, 20, 2048, 0), (64, 1024, 1024, 640, 0), (128, 2048, 1024, 2048, 0),
                                             (256, 2048, 2048, 512, 0), (32, 512, 100, 512, 40), (256, 2048, 8000, 512, 4)])
def test_every_tile_kind(handle, bn, m, n, k, groups):
    """One product for each kind of tile, as the plan says, exact on whole numbers."""
    assert gs.plan_gemm_fp8(T, N, m, n, k, groups=groups)[1] == bn
    gen = torch.Generator().manual_seed(bn + groups)
    a, b = operands(gen, T, N, m, n, k, BLK, VEC, batch=max(groups, 1))
    if not groups:
        assert torch.equal(run_gemm(handle, a, b, T, N, m, n, k, gs.R_16BF), product(a.values(), b.values())[0].bfloat16())
        return
    off = _offsets(gen, groups, n)
    c = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
    handle.gemm_fp8_grouped(gs.GROUP_N, T, N, m, n, k, groups, torch.tensor(off, dtype=torch.int32, device="cuda"), 1.0, a.bytes, E4,
                            a.ld, a.stride, a.scale, BLK, a.lds, a.stride_s, b.bytes, E4, b.ld, b.scale, VEC, b.lds, 0.0, c,
                            gs.R_16BF, m, 0)
    torch.cuda.synchronize()
    bv = b.values()
    for g in range(groups):
        assert torch.equal(c[off[g]:off[g + 1]], product(a.values(g), bv[off[g]:off[g + 1]])[0].bfloat16())


def test_scale_matrix_shape_helper():
    assert [blocks(x) for x in (1, 127, 128, 129)] == [1, 1, 1, 2]
