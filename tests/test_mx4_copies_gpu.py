"""Copies of 4-bit matrices: in memory of their own, also when the first one is gone."""
import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)   # (a file of this test's own)


@pytest.mark.parametrize("again", [copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)), saved])
@pytest.mark.parametrize("made", ["quantized", "on a stream", "bytes"])
def test_a_copy_is_a_matrix_of_its_own(ops, again, made):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(2, 30, 600, generator=g).half().to(DEV)
    q = ops.mx4_quantize(w, stream=torch.cuda.current_stream() if made == "on a stream" else None)
    if made == "bytes":
        q = ops.Mx4Tensor(q.packed, q.scales[:, :19], 600)
    want = q.dequantize()
    c = again(q)
    assert c.shape == q.shape and torch.equal(c.packed, q.packed) and torch.equal(c.tops, q.tops)
    assert (c._c.packed, c._c.scales, c._c.tops) == (c.packed.data_ptr(), c.scales.data_ptr(), c.tops.data_ptr())
    assert c._c.packed != q._c.packed
    del q
    x = torch.randn(3, 600, generator=g).half().to(DEV)
    torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(c.dequantize(), want)
    if made == "bytes":
        assert torch.equal(ops.mx4_linear(x, c), ops.mx4_linear(x, ops.mx4_quantize(w.view(60, 600))))


def test_a_shallow_copy_shares_its_memory(ops):
    q = ops.mx4_quantize(torch.randn(8, 64, device=DEV))
    want = q.dequantize()
    c = copy.copy(q)
    del q
    assert torch.equal(c.dequantize(), want)
