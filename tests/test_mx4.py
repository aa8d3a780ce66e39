"""What the 4-bit operators refuse before anything reaches a GPU."""
import ctypes

import pytest
import torch

import pimaicompiler_amd as P
from pimaicompiler_amd import _lib as L


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    u = torch.zeros(2, 32, dtype=torch.uint8)
    for call in (lambda: P.mx4_quantize(x), lambda: P.mx4_quantize([1.0]), lambda: P.Mx4Tensor(u, u[:, :2], 64), lambda: P.mx4_linear(x, None),
                 lambda: P.mx4_dequantize(x), lambda: P.mx4_matmul(x, x)):
        with pytest.raises(P.NNRuntimeException):
            call()


def test_the_c_interface_needs_an_initialised_device():
    m = L.Mx4Matrix(None, None, None, 1, 32, 16)
    lib = L.load()
    for rc in (lib.pimhip_mx4_quantize(m, None, 0, 32, None), lib.pimhip_mx4_find_tops(m, None), lib.pimhip_mx4_dequantize(None, 0, 32, m, None),
               lib.pimhip_mx4_linear(None, 1, None, 32, 0, 1, m, None, 0, None), lib.pimhip_mx4_matmul(None, 1, 0, m, m, None)):
        assert rc in (L.PIMHIP_ERR_HIP, L.PIMHIP_ERR_NOT_INITIALIZED)


def test_the_struct_of_the_binding_is_the_header_s():
    assert ctypes.sizeof(L.Mx4Matrix) == 48 and [n for n, _ in L.Mx4Matrix._fields_] == ["packed", "scales", "tops", "rows", "cols", "ld_scales"]


def test_a_copy_takes_no_address_along():
    """What a matrix is read through holds the addresses of its tensors: a deep copy and one that was pickled are made anew, which needs the GPU."""
    import copy
    import pickle
    packed, scales, tops = (torch.zeros(2, n, dtype=torch.uint8) for n in (16, 16, 1))
    kept = L.Mx4Matrix(packed.data_ptr(), scales.data_ptr(), tops.data_ptr(), 2, 32, 16)
    q = P.Mx4Tensor.__new__(P.Mx4Tensor)   # as the native call leaves it: the description as bytes, and where they are
    q.packed, q.scales, q.tops, q.shape, q._keep = packed, scales, tops, torch.Size([2, 32]), bytes(kept)
    q._at, q._device_index = id(q._keep), 0
    for call in (lambda: copy.deepcopy(q), lambda: pickle.loads(pickle.dumps(q))):
        with pytest.raises(P.NNRuntimeException):
            call()


def test_a_tensor_that_carries_a_tangent_is_refused():
    import torch.autograd.forward_ad as forward
    from pimaicompiler_amd.ops import _require_no_gradient
    x = torch.zeros(2, 64)
    _require_no_gradient(x, None)
    with forward.dual_level():
        _require_no_gradient(x, None)
        dual = forward.make_dual(x, torch.ones_like(x))
        for call in (lambda: _require_no_gradient(dual), lambda: _require_no_gradient(None, x, dual)):
            with pytest.raises(P.NNRuntimeException):
                call()
            with torch.no_grad(), pytest.raises(P.NNRuntimeException):
                call()
    _require_no_gradient(x)
