"""Token operators: what their host code refuses before any launch, on CPU tensors that the entry points of utils/tokens.py would turn away first."""
import pytest
import torch

from multiyolov5_amd import _lib as L
from multiyolov5_amd.utils import tokens as T


@pytest.fixture(scope='module')
def calls():
    """each operator of one tensor [2, 6, 4, 16], by the argument it is"""
    from multiyolov5_amd import build
    build.build(verbose=False)
    ext = T._ext()
    pos = torch.zeros(6, 1, dtype=torch.int64)
    turns, axis = T.rope_table((8,))

    def rope(q, k):
        import ctypes as C
        return ext.rope_axes(q, k, pos, C.addressof(turns), C.addressof(axis), 8, 1, False)
    z = torch.zeros(2, 6, 4, 16)
    return {'x': lambda t: ext.layer_norm(t, None, None, 1e-5), 'rope q': lambda t: rope(t, None), 'rope k': lambda t: rope(z, t),
            'q': lambda t: ext.window_attention(t, z, z, 0, 0, False, None, None, None), 'k': lambda t: ext.window_attention(z, t, z, 0, 0, False, None, None, None),
            'v': lambda t: ext.window_attention(z, z, t, 0, 0, False, None, None, None)}


NAMES = pytest.mark.parametrize('name', ['x', 'rope q', 'rope k', 'q', 'k', 'v'])


@NAMES
def test_dual_tensors_are_refused(calls, name):
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(L.MyoloError, match='forward mode'):
            calls[name](fw.make_dual(torch.zeros(2, 6, 4, 16), torch.ones(2, 6, 4, 16)))


@NAMES
def test_traced_calls_are_refused(calls, name):
    with pytest.raises(L.MyoloError, match='traced'):
        torch.jit.trace(calls[name], torch.zeros(2, 6, 4, 16), check_trace=False)


@NAMES
def test_tensors_without_storage_are_refused(calls, name):
    with pytest.raises(L.MyoloError, match='without storage'):
        calls[name](torch._efficientzerotensor((2, 6, 4, 16)))
