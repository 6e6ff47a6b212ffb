"""The Python binding without its native part (`_gs_fastcall`: built for one Python, and only where its headers are):
ctypes makes the same calls."""
import importlib.util
import sys

import pytest

import gemm_sm100 as gs

OK, BAD, UNS = gs.STATUS_NOT_INITIALIZED, gs.STATUS_INVALID_VALUE, gs.STATUS_NOT_SUPPORTED
P = 1 << 20  # a 16-byte aligned address that nothing reads


@pytest.fixture
def plain(monkeypatch):
    """The binding as it is imported where `_gs_fastcall` cannot be."""
    monkeypatch.setitem(sys.modules, "_gs_fastcall", None)
    spec = importlib.util.spec_from_file_location("gemm_sm100_plain", gs.__file__)
    module = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, spec.name, module)
    spec.loader.exec_module(module)
    return module


class Pointer:
    def data_ptr(self):
        return P


def test_same_statuses(plain):
    """What tests/test_fp8_refusals.py asks of the native binding."""
    fast = plain._fast
    assert fast.__name__ != "_gs_fastcall"

    def call(p, m=256, lda=512, at=gs.R_8F_E4M3):
        return fast.gemm_fp8(None, 1, 0, m, 96, 512, 1.0, p, at, lda, p, gs.SCALE_BLK128, 4, p, gs.R_8F_E5M2, 512, p,
                             gs.SCALE_VEC128, 96, 0, p, gs.R_16BF, 256)

    for p in (P, Pointer()):
        assert call(p) == OK
        assert call(p, lda=496) == BAD and call(p, at=gs.R_8I) == UNS
    assert call(None) == BAD and call(P + 8) == UNS and call(P, m=0) == OK
    grouped = [None, gs.GROUP_N, 1, 0, 256, 96, 512, 4, P, 1.0, P, gs.R_8F_E4M3, 512, 2**17, P, gs.SCALE_BLK128, 4, 8, P,
               gs.R_8F_E5M2, 512, P, gs.SCALE_VEC128, 96, 0.0, P, gs.R_16BF, 256, 0]
    assert fast.gemm_fp8_grouped(*grouped) == OK
    for k, v, status in ((1, 2, BAD), (7, 0, BAD), (13, 2**40 + 8, UNS), (17, -1, BAD), (28, 2**40, OK)):
        assert fast.gemm_fp8_grouped(*grouped[:k], v, *grouped[k + 1:]) == status, k
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


def test_same_refusals(plain):
    fast = plain._fast
    with pytest.raises(TypeError):
        fast.set_stream(None)
    with pytest.raises(OverflowError):
        fast.moe_combine(None, 2**31, 2, 64, P, gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)
    with pytest.raises(TypeError):
        fast.moe_combine(None, 1.5, 2, 64, P, gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)
    with pytest.raises(AttributeError):
        fast.moe_combine(None, 8, 2, 64, "y", gs.R_16BF, 64, 16, P, None, P, gs.R_16BF, 64)


@pytest.mark.gpu
def test_same_results(cuda, plain):
    """Every call once through both bindings."""
    import torch
    from routed_experts import RoutedExperts

    def outputs(binding):
        gen = torch.Generator(device="cuda").manual_seed(3)
        with binding.Handle() as h:
            layer = RoutedExperts(h, 200, 6, 2, 256, 384)
            layer.set_weights(torch.randn(6, 384, 256, generator=gen, device="cuda"))
            x, dout = (torch.randn(200, n, generator=gen, device="cuda").bfloat16() for n in (256, 384))
            logits = torch.randn(200, 6, generator=gen, device="cuda")
            out = layer.forward(x, logits).clone()
            grads = layer.backward(x, logits, dout)
            dense = torch.empty(layer.rows, 384, device="cuda")
            h.gemm_fp8(gs.OP_T, gs.OP_N, 384, layer.rows, 256, 0.5, layer.wq[1], gs.R_8F_E4M3, 256, layer.w_scale[1],
                       gs.SCALE_BLK128, 2, layer.xq, gs.R_8F_E4M3, 256, layer.x_scale, gs.SCALE_VEC128, layer.rows, 0.0, dense,
                       gs.R_32F, 384)
            torch.cuda.synchronize()
            assert h.device_error() == 0
            return [out, *grads, dense[:int(layer.offsets[-1])]]

    for a, b in zip(outputs(gs), outputs(plain)):
        assert torch.equal(a, b)
