"""Handles of expert layer plans: a destroyed plan's is never another's."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_the_handle_of_a_destroyed_plan_is_no_other_plan_s(ops):
    from pimaicompiler_amd import _lib as L
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    make = lambda D: ops.MoeLayerPlan((z(4, D), None), z(4, 32, D), z(4, D, 32))  # noqa: E731
    old = make(64)
    assert L.load().pimhip_moe_layer_plan_destroy(old._handle) == L.PIMHIP_OK
    new = [make(4096) for _ in range(20)]
    values = [p._handle.value for p in new]
    assert old._handle.value not in values and len(set(values)) == 20
    n = ctypes.c_uint64()
    assert L.load().pimhip_moe_layer_workspace_bytes(old._handle, 1, ctypes.byref(n)) == L.PIMHIP_ERR_INVALID_ARGUMENT
    with pytest.raises(ops.NNRuntimeException):
        old.forward(z(1, 64))
    del old                     # (what it destroys when it goes is not one of the others)
    for p in new:
        assert (p.forward(z(3, 4096))[0] == 0).all()
