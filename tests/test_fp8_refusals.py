"""CPU tests of the FP8 and routed-expert entry points' argument checks and of
their host-only planning calls. The checks come before the handle, so a call
with no handle answers a bad argument with its status and a good call with
GS_STATUS_NOT_INITIALIZED; nothing is launched here."""
import ctypes

import pytest

import gemm_sm100 as gs

OK, BAD, UNS = gs.STATUS_NOT_INITIALIZED, gs.STATUS_INVALID_VALUE, gs.STATUS_NOT_SUPPORTED
P = 1 << 20  # a 16-byte aligned address that nothing reads
ONE = ctypes.c_float(1.0)
F = ctypes.addressof(ONE)


def quantize(mode=gs.SCALE_VEC128, axis=0, rows=256, cols=128, src=P, st=gs.R_16BF, lds=256, index=None, div=1, src_cols=0,
             dst=P, dt=gs.R_8F_E4M3, ldd=256, scale=P, ldsc=None):
    if ldsc is None:
        ldsc = max(1, 2 if mode == gs.SCALE_BLK128 else cols if axis == 0 else rows)
    return gs.lib().gs_fp8_quantize(None, mode, axis, rows, cols, src, st, lds, index, div, src_cols, dst, dt, ldd, scale,
                                    ldsc)


@pytest.mark.parametrize("change,status", [
    ({}, OK), ({"axis": 1}, OK), ({"mode": gs.SCALE_BLK128}, OK), ({"index": P, "src_cols": 64, "div": 4}, OK),
    ({"index": P, "src_cols": 0, "src": None}, OK), ({"rows": 0, "src": None}, OK), ({"cols": 0, "dst": None}, OK),
    ({"mode": 3}, BAD), ({"axis": 2}, BAD), ({"mode": gs.SCALE_BLK128, "axis": 1}, BAD), ({"rows": -1}, BAD),
    ({"lds": 255}, BAD), ({"ldd": 255}, BAD), ({"ldsc": 127}, BAD), ({"axis": 1, "ldsc": 255}, BAD),
    ({"mode": gs.SCALE_BLK128, "ldsc": 1}, BAD), ({"index": P, "div": 0}, BAD), ({"index": P, "src_cols": -1}, BAD),
    ({"src": None}, BAD), ({"dst": None}, BAD), ({"scale": None}, BAD), ({"src": P + 1}, BAD), ({"scale": P + 2}, BAD),
    ({"index": P + 1, "src_cols": 4}, BAD), ({"st": gs.R_8I}, UNS), ({"dt": gs.R_16F}, UNS),
    ({"cols": 2**31 - 1, "ldsc": 2**31 - 1}, UNS), ({"rows": 2**30 + 1, "lds": 2**31 - 1, "ldd": 2**31 - 1}, UNS),
    ({"rows": 2**30, "lds": 2**30, "ldd": 2**30}, OK),
])
def test_quantize_checks(change, status):
    assert quantize(**change) == status


def gemm(grouped=False, ragged=gs.GROUP_N, ta=1, tb=0, m=256, n=96, k=512, groups=4, off=P, A=P, at=gs.R_8F_E4M3, lda=None,
         sta=256 * 512, sa=P, ma=gs.SCALE_BLK128, ldsa=None, stsa=8, B=P, bt=gs.R_8F_E5M2, ldb=None, sb=P,
         mb=gs.SCALE_VEC128, ldsb=None, C=P, ct=gs.R_16BF, ldc=None, stc=256 * 96, alpha=F, beta=F):
    up = lambda x: max(16, (x + 15) // 16 * 16)  # noqa: E731
    nb = lambda x: max(1, (x + 127) // 128)      # noqa: E731
    lda = up(k if ta else m) if lda is None else lda
    ldb = up(n if tb else k) if ldb is None else ldb
    ldsa = (max(m, 1) if ma == gs.SCALE_VEC128 else nb(k if ta else m)) if ldsa is None else ldsa
    ldsb = (max(n, 1) if mb == gs.SCALE_VEC128 else nb(n if tb else k)) if ldsb is None else ldsb
    ldc = max(m, 1) if ldc is None else ldc
    if grouped:
        return gs.lib().gs_gemm_fp8_grouped(None, ragged, ta, tb, m, n, k, groups, off, alpha, A, at, lda, sta, sa, ma, ldsa,
                                            stsa, B, bt, ldb, sb, mb, ldsb, beta, C, ct, ldc, stc)
    return gs.lib().gs_gemm_fp8(None, ta, tb, m, n, k, alpha, A, at, lda, sa, ma, ldsa, B, bt, ldb, sb, mb, ldsb, beta, C,
                                ct, ldc)


SHARED = [
    ({}, OK), ({"ta": 0}, OK), ({"m": 0, "C": None}, OK), ({"n": 0}, OK),
    ({"k": 0, "A": None, "B": None, "sa": None, "sb": None}, OK), ({"m": 255, "n": 33, "k": 77}, OK), ({"ct": gs.R_32F}, OK),
    ({"ta": 3}, BAD), ({"tb": -1}, BAD), ({"m": -1}, BAD), ({"k": -1}, BAD), ({"alpha": None}, BAD), ({"beta": None}, BAD),
    ({"ma": 0}, BAD), ({"mb": 2}, BAD), ({"lda": 496}, BAD), ({"ldb": 496}, BAD), ({"ldc": 255}, BAD), ({"ldsa": 3}, BAD),
    ({"ldsb": 95}, BAD), ({"ma": gs.SCALE_VEC128, "ldsa": 255}, BAD), ({"A": None}, BAD), ({"sa": None}, BAD),
    ({"sb": P + 2}, BAD), ({"C": None}, BAD), ({"C": P + 1}, BAD), ({"at": gs.R_8I}, UNS), ({"bt": gs.R_16F}, UNS),
    ({"ct": gs.R_8F_E4M3}, UNS), ({"A": P + 8}, UNS), ({"B": P + 4}, UNS), ({"lda": 520}, UNS), ({"ldb": 520}, UNS),
    ({"k": 2**31 - 1, "lda": 2**31 - 1, "ldb": 2**31 - 1, "ldsa": 2**24}, UNS),
]


@pytest.mark.parametrize("change,status", SHARED + [({"tb": 1}, OK), ({"mb": gs.SCALE_BLK128}, OK)])
def test_gemm_checks(change, status):
    assert gemm(**change) == status


@pytest.mark.parametrize("change,status", SHARED + [
    ({"ragged": gs.GROUP_K, "ta": 0, "tb": 1}, OK), ({"ragged": gs.GROUP_K, "mb": gs.SCALE_BLK128}, OK), ({"sta": 0}, OK),
    ({"groups": 0}, BAD), ({"ragged": 2}, BAD), ({"off": None}, BAD), ({"off": P + 2}, BAD), ({"sta": -16}, BAD),
    ({"stsa": -1}, BAD), ({"ragged": gs.GROUP_K, "stc": 256 * 96 - 1}, BAD), ({"groups": gs.FP8_MAX_GROUPS + 1}, UNS),
    ({"tb": 1}, UNS), ({"mb": gs.SCALE_BLK128}, UNS), ({"sta": 256 * 512 + 8}, UNS),
    ({"m": 2**31 - 2048, "ldc": 2**31 - 2048, "n": 2**20, "ldsb": 2**20}, UNS),
])
def test_grouped_gemm_checks(change, status):
    assert gemm(grouped=True, **change) == status


def route_desc(**kw):
    tokens, experts, top_k = kw.get("tokens", 2048), kw.get("experts", 64), kw.get("top_k", 4)
    d = dict(tokens=2048, experts=64, top_k=4, logits=P, logits_type=gs.R_32F, ld_logits=max(experts, 1),
             score=gs.ROUTE_SOFTMAX, groups=1, top_groups=1, scale=1.0, align=128, ids=P, weights=P, offsets=P, slot_row=P,
             row_slot=P, rows=tokens * top_k + 64 * 127, workspace=P, workspace_bytes=148 * max(experts, 1) * 4)
    d.update(kw)
    return gs.RouteDesc(**d)


@pytest.mark.parametrize("change,status", [
    ({}, OK), ({"offsets": None, "slot_row": None, "row_slot": None, "rows": 0, "workspace": None}, OK),
    ({"tokens": 0, "logits": None, "ids": None, "weights": None, "slot_row": None}, OK),
    ({"tokens": 16, "workspace": None, "workspace_bytes": 0}, OK), ({"groups": 8, "top_groups": 2}, OK),
    ({"experts": 1024, "top_k": 32, "rows": 2**20}, OK),
    ({"tokens": -1}, BAD), ({"experts": 0}, BAD), ({"top_k": 0}, BAD), ({"experts": 4, "top_k": 5}, BAD), ({"score": 2}, BAD),
    ({"ld_logits": 63}, BAD), ({"logits": None}, BAD), ({"logits": P + 2}, BAD), ({"ids": None}, BAD), ({"weights": P + 1}, BAD),
    ({"groups": 0}, BAD), ({"groups": 7}, BAD), ({"groups": 8, "top_groups": 9}, BAD), ({"groups": 32, "top_groups": 1}, BAD),
    ({"align": 0}, BAD), ({"rows": 2048 * 4}, BAD), ({"slot_row": None}, BAD), ({"row_slot": None}, BAD),
    ({"workspace": None}, BAD), ({"workspace_bytes": 64}, BAD), ({"workspace": P + 1}, BAD),
    ({"logits_type": gs.R_8I}, UNS), ({"experts": 1025}, UNS), ({"top_k": 33}, UNS), ({"groups": 64, "top_groups": 4}, UNS),
    ({"tokens": 2**30}, UNS),
])
def test_route_checks(change, status):
    assert gs.lib().gs_moe_route(None, ctypes.byref(route_desc(**change))) == status


def test_route_null_descriptor():
    assert gs.lib().gs_moe_route(None, None) == BAD
    assert gs.lib().gs_moe_route_backward(None, None, P, P, gs.R_32F, 64) == BAD


@pytest.mark.parametrize("change,dw,dl,dt,ld,status", [
    ({}, P, P, gs.R_32F, 64, OK), ({"logits_type": gs.R_16BF}, P, P, gs.R_16BF, 64, OK),
    ({"logits_type": gs.R_16BF}, P, P, gs.R_32F, 64, OK), ({"tokens": 0}, None, None, gs.R_32F, 64, OK),
    ({}, P, P, gs.R_32F, 63, BAD), ({}, None, P, gs.R_32F, 64, BAD), ({}, P, None, gs.R_32F, 64, BAD),
    ({"ids": None}, P, P, gs.R_32F, 64, BAD), ({}, P, P, gs.R_16BF, 64, UNS),
])
def test_route_backward_checks(change, dw, dl, dt, ld, status):
    assert gs.lib().gs_moe_route_backward(None, ctypes.byref(route_desc(**change)), dw, dl, dt, ld) == status


def combine(tokens=8, top_k=2, hidden=64, y=P, yt=gs.R_16BF, ldy=64, rows=16, slot=P, w=P, out=P, ot=gs.R_16BF, ldo=64):
    return gs.lib().gs_moe_combine(None, tokens, top_k, hidden, y, yt, ldy, rows, slot, w, out, ot, ldo)


@pytest.mark.parametrize("change,status", [
    ({}, OK), ({"w": None}, OK), ({"tokens": 0, "slot": None, "out": None}, OK), ({"rows": 0, "y": None}, OK),
    ({"tokens": -1}, BAD), ({"top_k": 0}, BAD), ({"hidden": -1}, BAD), ({"ldy": 63}, BAD), ({"ldo": 63}, BAD), ({"y": None}, BAD),
    ({"slot": None}, BAD), ({"out": None}, BAD), ({"y": P + 1}, BAD), ({"w": P + 2}, BAD), ({"out": P + 1}, BAD),
    ({"yt": gs.R_8I}, UNS), ({"ot": gs.R_8F_E4M3}, UNS), ({"tokens": 2**30, "top_k": 4}, UNS),
    ({"hidden": 2**30 + 1, "ldy": 2**31 - 1, "ldo": 2**31 - 1}, UNS),
])
def test_combine_checks(change, status):
    assert combine(**change) == status


def combine_backward(tokens=8, top_k=2, hidden=64, y=P, yt=gs.R_16BF, ldy=64, rows=16, slot=P, row=P, w=P, dout=P, ldo=64,
                     dy=P, lddy=64, dw=P):
    return gs.lib().gs_moe_combine_backward(None, tokens, top_k, hidden, y, yt, ldy, rows, slot, row, w, dout, ldo, dy, lddy,
                                            dw)


@pytest.mark.parametrize("change,status", [
    ({}, OK), ({"rows": 0, "y": None, "row": None, "dy": None}, OK), ({"ldo": 63}, BAD), ({"lddy": 63}, BAD), ({"row": None}, BAD),
    ({"w": None}, BAD), ({"dout": None}, BAD), ({"dy": None}, BAD), ({"dw": None}, BAD), ({"dout": P + 1}, BAD),
    ({"dw": P + 2}, BAD), ({"yt": gs.R_32I}, UNS),
])
def test_combine_backward_checks(change, status):
    assert combine_backward(**change) == status


@pytest.mark.parametrize("tokens,experts,top_k,align,rows", [
    (0, 8, 2, 128, 0), (1, 64, 4, 1, 4), (1, 64, 4, 128, 4 + 4 * 127), (1000, 16, 2, 128, 2000 + 16 * 127),
])
def test_plan_rows(tokens, experts, top_k, align, rows):
    assert gs.moe_rows(tokens, experts, top_k, align) == rows


def test_plan_rows_and_workspace_refusals():
    for bad in ((-1, 8, 2, 1), (1, 0, 2, 1), (1, 8, 0, 1), (1, 8, 2, 0), (2**30, 8, 2, 1)):
        with pytest.raises(gs.GemmError):
            gs.moe_rows(*bad)
    with pytest.raises(gs.GemmError):
        gs.moe_route_workspace(-1, 8, 2)
    assert gs.moe_route_workspace(16, 64, 4) == 0  # few slots: one block, no workspace
    assert gs.moe_route_workspace(65536, 256, 8) == 148 * 256 * 4


def test_plan_tile():
    s, bn, cg, parts = gs.plan_gemm_fp8(1, 0, 8192, 8192, 8192)
    assert (s, bn, cg, parts) == (0, 256, 2, 1)
    assert gs.plan_gemm_fp8(1, 0, 4096, 16, 4096) == (0, 32, 1, 4)      # few tokens: narrow tiles, K over clusters
    assert gs.plan_gemm_fp8(1, 0, 1024, 16, 8192) == (0, 32, 1, 8)
    assert gs.plan_gemm_fp8(1, 0, 1024, 1024, 1024) == (0, 64, 1, 1)    # 128 tiles for 148 SMs instead of 16 pair tiles
    assert gs.plan_gemm_fp8(0, 1, 4096, 16, 4096)[1] == 128  # op(B) = T is read in panels of 128 columns
    assert gs.plan_gemm_fp8(1, 0, 2048, 128, 2048, groups=64)[1:] == (32, 1, 1)
    for bad in (dict(m=0, n=1, k=1), dict(m=1, n=1, k=1, groups=gs.FP8_MAX_GROUPS + 1), dict(m=1, n=1, k=1, groups=1, ragged=5)):
        assert gs.plan_gemm_fp8(1, 0, **bad)[0] == gs.STATUS_INVALID_VALUE


class Pointer:
    """Stands for a tensor: something with a data_ptr()."""

    def __init__(self, at):
        self.at = at

    def data_ptr(self):
        return self.at


def test_native_binding_passes_arguments_through():
    """_gs_fastcall hands the library the same arguments as ctypes does: the statuses agree, whatever kind of pointer."""
    import _gs_fastcall as fast

    def call(p, m=256, lda=512, ldb=512, at=gs.R_8F_E4M3):
        return fast.gemm_fp8(None, 1, 0, m, 96, 512, 1.0, p, at, lda, p, gs.SCALE_BLK128, 4, p, gs.R_8F_E5M2, ldb, p,
                             gs.SCALE_VEC128, 96, 0, p, gs.R_16BF, 256)

    for p in (P, Pointer(P)):
        assert call(p) == OK
        assert call(p, lda=496) == BAD and call(p, at=gs.R_8I) == UNS
    assert call(None) == BAD and call(P + 8) == UNS and call(P, m=0) == OK
    assert fast.fp8_quantize(None, gs.SCALE_VEC128, 0, 256, 128, P, gs.R_16BF, 256, None, 1, 0, P, gs.R_8F_E4M3, 256, P,
                             127) == BAD
    assert fast.moe_combine(None, 8, 2, 64, P, gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64) == OK
    route = [2048, 64, 4, P, gs.R_32F, 64, None, gs.ROUTE_SIGMOID, 8, 2, True, 2.5, None, 128, P, P, P, P, P, 2**16, P, 2**20]
    assert fast.moe_route(None, *route) == OK
    for k, v, status in ((2, 65, BAD), (5, 63, BAD), (9, 9, BAD), (13, 0, BAD), (19, 8192, BAD), (21, 16, BAD), (4, gs.R_8I, UNS)):
        assert fast.moe_route(None, *route[:k], v, *route[k + 1:]) == status, k
    assert fast.moe_route_backward(None, *route, P, P, gs.R_32F, 64) == OK
    assert fast.moe_route_backward(None, *route, P, P, gs.R_32F, 63) == BAD
    assert fast.moe_combine_backward(None, 8, 2, 64, P, gs.R_16BF, 64, 16, P, P, P, P, 64, P, 63, P) == BAD
    assert fast.set_stream(None, None) == OK


def test_native_binding_refuses_what_c_cannot_hold():
    import _gs_fastcall as fast

    with pytest.raises(TypeError):
        fast.set_stream(None)
    with pytest.raises(OverflowError):
        fast.moe_combine(None, 2**31, 2, 64, P, gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)
    with pytest.raises(TypeError):
        fast.moe_combine(None, 1.5, 2, 64, P, gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)
    with pytest.raises(AttributeError):
        fast.moe_combine(None, 8, 2, 64, "y", gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)
