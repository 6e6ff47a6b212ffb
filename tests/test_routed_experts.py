"""CPU tests of RoutedExperts' own part: where its buffers are, what it hands to the library and what it refuses. The
handle is a stand-in that records the calls; nothing is launched."""
import pytest
import torch

import gemm_sm100 as gs
from routed_experts import RoutedExperts


class FakeHandle:
    device = "cpu"
    stream = 0

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args, **kw: self.calls.append((name, args, kw))


def layer(handle=None, tokens=5, experts=4, top_k=2, d_in=32, d_out=48, **kw):
    return RoutedExperts(handle or FakeHandle(), tokens, experts, top_k, d_in, d_out, **kw)


def tensors(obj):
    for v in vars(obj).values():
        if isinstance(v, torch.Tensor):
            yield v
        elif isinstance(v, dict):
            yield from (t for t in v.values() if isinstance(t, torch.Tensor))


def test_buffers_are_on_the_handles_device():
    """Not on the current device, which may be another by now."""
    l = layer()
    l._gradient_buffers()
    assert {t.device for t in tensors(l)} == {torch.device("cpu")}


@pytest.mark.gpu
def test_a_handle_names_its_device(cuda):
    with gs.Handle() as h:
        assert h.device == "cuda:0"
        l = layer(h)
        assert {t.device for t in tensors(l)} == {torch.device("cuda", 0)}
