"""Refusals of the routing and 8-bit floating point entry points that need no GPU."""
import ctypes as C

import numpy as np
import pytest

import llambda_b200 as LB
from llambda_b200 import _native as N
from llambda_b200 import experts as X


def _route_desc(**kw):
    d = dict(experts=16, top_k=4, score=0, groups=4, top_groups=2, group_top=2, renormalise=1,
             weight_scale=1.0)
    d.update(kw)
    return N.RouteDesc(*d.values())


@pytest.mark.parametrize("change, match", [
    (dict(experts=0), "Expert count"), (dict(experts=1025, groups=1, top_groups=1), "Expert count"),
    (dict(score=2), "score"), (dict(groups=3), "equal groups"), (dict(groups=0), "equal groups"),
    (dict(experts=66, groups=33), "equal groups"), (dict(top_groups=0), "top_groups"),
    (dict(top_groups=5), "top_groups"), (dict(group_top=3), "group_top"),
    (dict(experts=4, top_k=1), "two experts"), (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"),
    (dict(experts=64, groups=1, top_groups=1, top_k=33), "top_k"),
])
def test_route_descriptor_refusals(change, match):
    one = np.zeros(1, np.float32)
    d = _route_desc(**change)
    rc = N.lib().llambda_cuda_route_device(C.byref(d), 0, one.ctypes.data, 16, None, 1,
                                           one.ctypes.data, one.ctypes.data, None)
    assert rc == -1 and match in N.last_error()
    rc = N.lib().llambda_cuda_route(C.byref(d), one.ctypes.data, None, 1, one.ctypes.data,
                                    one.ctypes.data)
    assert rc == -1 and match in N.last_error()


def test_null_arguments_are_errors():
    L = N.lib()
    h = C.c_void_p(1)
    assert L.llambda_cuda_route_device(None, 0, None, 0, None, 1, None, None, None) == -1
    d = _route_desc()
    assert L.llambda_cuda_route_device(C.byref(d), 0, None, 16, None, 1, None, None, None) == -1
    assert L.llambda_cuda_fp8_quantize_device(0, None, 0, 1, 1, None, None, None) == -1
    assert L.llambda_cuda_fp8_session_create(None, 0, C.byref(h)) == -1 and not h.value
    assert L.llambda_cuda_fp8_session_create(None, 0, None) == -1
    h = C.c_void_p(1)
    assert L.llambda_cuda_fp8_moe_session_create(None, None, None, 0, C.byref(h)) == -1
    assert not h.value
    assert L.llambda_cuda_fp8_session_run(None, None, 1, None) == -1
    assert L.llambda_cuda_fp8_session_run_device(None, 0, None, 0, 1, 0, None, 0, None, 0, None) == -1
    assert L.llambda_cuda_fp8_session_run_quantized(None, None, None, 1, 0, None, 0, None) == -1
    assert L.llambda_cuda_fp8_moe_session_run(None, None, 1, 1, None, None, None) == -1
    assert L.llambda_cuda_fp8_moe_session_run_device(None, 0, None, 0, 1, 1, None, None, 0, None, 0,
                                                     None, 0, None) == -1
    assert L.llambda_cuda_fp8_session_workspace(None, 1) == 0
    assert L.llambda_cuda_fp8_moe_session_workspace(None, 1, 1) == 0
    assert L.llambda_cuda_fp8_session_status(None) == -1
    assert L.llambda_cuda_fp8_moe_session_status(None) == -1
    L.llambda_cuda_fp8_session_destroy(None)
    L.llambda_cuda_fp8_moe_session_destroy(None)


def test_moe_tensors_have_to_fit():
    def t(ne0, ne1, ne2, data=1):
        return N.Fp8Tensor(ne0, ne1, ne2, data, 1)

    up = t(32, 48, 4)
    for gate, down, match in ((t(16, 48, 4), t(48, 32, 4), "gate"), (t(32, 48, 3), t(48, 32, 4), "gate"),
                              (N.Fp8Tensor(0, 0, 0, None, None), t(32, 32, 4), "down"),
                              (N.Fp8Tensor(0, 0, 0, None, None), t(48, 32, 2), "down")):
        h = C.c_void_p()
        rc = N.lib().llambda_cuda_fp8_moe_session_create(C.byref(gate), C.byref(up), C.byref(down), 0,
                                                         C.byref(h))
        assert rc == -1 and match in N.last_error() and not h.value


def test_host_arguments_are_checked():
    with pytest.raises(ValueError, match="score"):
        LB.route_experts(np.zeros((2, 8), np.float32), 2, score="linear")
    with pytest.raises(ValueError, match="top_k"):
        LB.route_experts(np.zeros((2, 8), np.float32), 9)
    with pytest.raises(ValueError, match="positive token count"):
        LB.route_experts(np.zeros((0, 8), np.float32), 2)
    with pytest.raises(ValueError, match="bias"):
        LB.route_experts(np.zeros((2, 8), np.float32), 2, bias=np.zeros(7, np.float32))
    with pytest.raises(ValueError, match="scales"):
        LB.Fp8ProjectionSession.from_tensor(np.zeros((130, 64), np.uint8), np.ones((1, 1)))
    with pytest.raises(ValueError, match="e4m3 bytes"):
        LB.Fp8ProjectionSession.from_tensor(np.zeros((130, 64), np.float32), np.ones((2, 1)))
    with pytest.raises(ValueError, match="e4m3 bytes"):
        LB.Fp8MoeSession.from_tensor((np.zeros((4, 4), np.uint8), np.ones((1, 1))),
                                     (np.zeros((1, 4, 4), np.uint8), np.ones((1, 1, 1))))


def test_device_arguments_have_to_be_cuda_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        LB.route_experts(x, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        LB.fp8_quantize(x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        LB.Fp8ProjectionSession.from_device(x.to(torch.float8_e4m3fn), torch.ones(1, 1))
    with pytest.raises(ValueError, match="CUDA tensor"):
        LB.Fp8MoeSession.from_device(up=(x, x), down=(x, x))


def test_a_closed_session_refuses():
    s = X.Fp8ProjectionSession(None, 4, 4)
    with pytest.raises(ValueError, match="closed"):
        s.run(np.zeros(4, np.float32))
    s.close()
