"""CPU tests of Handle.set_stream's argument, on a handle that is not one (the library answers that it is not
initialised once the argument has got through)."""
import ctypes

import pytest

import gemm_sm100 as gs


class Stream:
    def __init__(self, at):
        self.cuda_stream = at


class Tensor:
    def data_ptr(self):
        return 1 << 20


@pytest.fixture
def handle():
    h = object.__new__(gs.Handle)
    h._h = h._raw = None
    return h


@pytest.mark.parametrize("stream", [None, 0, 1 << 20, Stream(0), Stream(1 << 20), ctypes.c_void_p(), ctypes.c_void_p(1 << 20)])
def test_streams_get_through(handle, stream):
    with pytest.raises(gs.GemmError) as e:
        handle.set_stream(stream)
    assert e.value.status == gs.STATUS_NOT_INITIALIZED


@pytest.mark.parametrize("stream", [Tensor(), "stream", 1.5, Stream(Tensor())])
def test_what_is_not_a_stream_is_refused(handle, stream):
    """A tensor's address is not a stream."""
    with pytest.raises(TypeError):
        handle.set_stream(stream)
