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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("E,k,D,F,M", [(1, 1, 8, 1, 1), (4, 2, 40, 33, 3), (3, 3, 64, 4100, 17), (8, 2, 136, 257, 64), (60, 6, 72, 65, 13)])
def test_a_call_stays_in_its_workspace_and_outputs(ops, E, k, D, F, M, dtype):
    from pimaicompiler_amd import _lib as L
    g = torch.Generator().manual_seed(E + F)
    r = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dtype).to(DEV)  # noqa: E731
    plan = ops.MoeLayerPlan((r(E, D), None), r(E, 2 * F, D), r(E, D, F), top_k=k, gated=True)
    x = r(M, D)
    want = plan.forward(x)
    sizes = [plan.workspace_bytes(M), M * D * 2, M * k * 4, M * k * 4]
    held = [torch.full((512 + n + 512,), 171, dtype=torch.uint8, device=DEV) for n in sizes]
    at = [t.data_ptr() + 512 for t in held]
    assert L.load().pimhip_moe_layer_forward(plan._handle, x.data_ptr(), D, M, at[1], at[2], at[3], at[0], torch.cuda.current_stream().cuda_stream) == L.PIMHIP_OK
    for t, n in zip(held, sizes):
        assert (t[:512] == 171).all() and (t[512 + n:] == 171).all()
    for t, n, w in zip(held[1:], sizes[1:], want):
        assert torch.equal(t[512:512 + n].view(w.dtype), w.reshape(-1))
