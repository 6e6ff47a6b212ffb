"""GPU tests of gs_fp8_quantize against its definition in float64. Scales are
powers of two, so x / scale is exact and both outputs have to be equal bit for
bit: no tolerance."""
import math

import pytest
import torch

import gemm_sm100 as gs
from fp8_util import FLOAT, FP8, blocks

pytestmark = pytest.mark.gpu
E4, E5, VEC, BLK = gs.R_8F_E4M3, gs.R_8F_E5M2, gs.SCALE_VEC128, gs.SCALE_BLK128


def reference(x, mode, axis, fp8):
    """x [cols, rows] float64 -> (q values, scales in the call's layout)."""
    top, low, bits, emin = (448.0, -6, 3, 8) if fp8 == E4 else (57344.0, -14, 2, 15)
    c, r = x.shape
    a = torch.where(x.isfinite(), x.abs(), 0.0)
    a = torch.nn.functional.pad(a, (0, blocks(r) * 128 - r, 0, blocks(c) * 128 - c))
    if mode == BLK:
        amax = a.view(blocks(c), 128, blocks(r), 128).amax((1, 3))
    elif axis == 0:
        amax = a[:c].view(c, blocks(r), 128).amax(2).t()
    else:
        amax = a[:, :r].reshape(blocks(c), 128, r).amax(1)
    f, e = torch.frexp(amax)
    e = (e - 1 - emin + (f > 0.875).int()).clamp(min=-126)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), 1.0)
    if mode == BLK:
        full = scale.repeat_interleave(128, 0)[:c].repeat_interleave(128, 1)[:, :r]
    elif axis == 0:
        full = scale.t().repeat_interleave(128, 1)[:, :r]
    else:
        full = scale.repeat_interleave(128, 0)[:c]
    y = x / full
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp(min=2.0 ** low)).exponent - 1 - bits)
    q = torch.where(y.isfinite(), torch.round(y / step) * step, y)  # torch.round: ties to even
    if fp8 == E4:
        q = torch.where(y.isinf(), math.nan, q)
    assert bool((amax <= top * scale).all())
    return q, scale


def run(h, x, mode, axis, fp8, index=None, div=1, ld_pad=0, offset=0):
    """x: CPU [src_cols, rows] tensor of a float type."""
    st = {v: k for k, v in FLOAT.items()}[x.dtype]
    src_cols, rows = x.shape
    cols = src_cols if index is None else len(index)
    lds = rows + ld_pad
    buf = torch.full((src_cols * lds + offset,), math.nan, dtype=x.dtype, device="cuda")
    src = buf[offset:].view(src_cols, lds)
    src[:, :rows] = x.cuda()
    ldd = rows + ld_pad
    dst = torch.full((cols * ldd + offset,), 0x55, dtype=torch.uint8, device="cuda")
    d = dst[offset:].view(cols, ldd)
    shape = (blocks(cols), blocks(rows)) if mode == BLK else (blocks(rows), cols) if axis == 0 else (blocks(cols), rows)
    scale = torch.full((shape[0], shape[1] + ld_pad), -1.0, device="cuda")
    idx = None if index is None else torch.tensor(index, dtype=torch.int32, device="cuda")
    h.fp8_quantize(mode, axis, rows, cols, src, st, lds, d, fp8, ldd, scale, shape[1] + ld_pad, index=idx, index_div=div,
                   src_cols=src_cols)
    torch.cuda.synchronize()
    assert h.last_kernels() == gs.KERNEL_QUANTIZE
    assert bool((d[:, rows:] == 0x55).all()) and bool((scale[:, shape[1]:] == -1).all())  # padding stays
    return d[:, :rows].contiguous().view(FP8[fp8]).double().cpu(), scale[:, :shape[1]].double().cpu()


def check(got, want):
    (q, s), (rq, rs) = got, want
    assert torch.equal(s, rs)
    assert torch.equal(q.isnan(), rq.isnan())
    assert torch.equal(q[~rq.isnan()], rq[~rq.isnan()])


SHAPES = [(1, 1), (128, 128), (129, 5), (7, 300), (200, 130), (1024, 64), (130, 257), (64, 1), (1, 129), (2055, 131)]
MODES = [(VEC, 0), (VEC, 1), (BLK, 0)]


@pytest.mark.parametrize("fp8", [E4, E5])
@pytest.mark.parametrize("st", [gs.R_32F, gs.R_16F, gs.R_16BF])
@pytest.mark.parametrize("mode,axis", MODES)
def test_against_the_definition(handle, mode, axis, st, fp8):
    gen = torch.Generator().manual_seed(mode + axis + st + fp8)
    for rows, cols in SHAPES:
        x = (torch.randn(cols, rows, generator=gen) * torch.randn(cols, 1, generator=gen).exp()).to(FLOAT[st])
        # aligned rows take the 16-byte path, odd leading dimensions and addresses the other one
        pad, off = ((-rows) % 8, 0) if rows % 2 else (3, 1)
        check(run(handle, x, mode, axis, fp8, ld_pad=pad, offset=off), reference(x.double(), mode, axis, fp8))


@pytest.mark.parametrize("mode,axis", MODES)
@pytest.mark.parametrize("fp8", [E4, E5])
def test_special_values(handle, mode, axis, fp8):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(300, 300, generator=gen)
    x[0, 0], x[5, 140], x[200, 17] = math.inf, -math.inf, math.nan
    x[130:256, 128:256] = 0.0
    x[0:128, 256:] = 0.0                                   # a whole block of zeros
    x[256:, :128] = 1e-41                                  # subnormals: the scale stops at 2^-126
    x[256:, 128:256] = 3e38
    x[140, 140] = -0.0
    top = 448.0 if fp8 == E4 else 57344.0
    x[128, :128] = 0.0
    x[128, 0], x[129, 128], x[131, 130] = top, top * 2, top * 1.0001
    x[250, 0:16] = torch.arange(16.0) + 0.5                # ties
    check(run(handle, x, mode, axis, fp8), reference(x.double(), mode, axis, fp8))


@pytest.mark.parametrize("mode,axis", MODES)
@pytest.mark.parametrize("pad", [0, 1])
def test_gathered_columns(handle, mode, axis, pad):
    gen = torch.Generator().manual_seed(9)
    rows, src_cols, div = 264, 40, 3
    x = torch.randn(src_cols, rows, generator=gen).to(torch.bfloat16)
    index = torch.randint(0, src_cols * div, (333,), generator=gen).tolist()
    index[0], index[7], index[200], index[9], index[8] = -1, -5, src_cols * div, 5, 5
    full = torch.cat([x, torch.zeros(1, rows, dtype=x.dtype)]).double()
    pick = [i // div if 0 <= i < src_cols * div else src_cols for i in index]
    check(run(handle, x, mode, axis, E4, index, div, ld_pad=pad), reference(full[pick], mode, axis, E4))


def test_no_source_columns_give_zeros(handle):
    x = torch.empty(0, 128, dtype=torch.float32)
    q, s = run(handle, x, VEC, 0, E4, [3, -1, 0])
    assert bool((q == 0).all()) and bool((s == 1).all())


def test_more_columns_than_the_grid_holds_at_once(handle):
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(40000, 256, generator=gen).to(torch.bfloat16)
    for mode, axis in MODES:
        check(run(handle, x, mode, axis, E4), reference(x.double(), mode, axis, E4))
