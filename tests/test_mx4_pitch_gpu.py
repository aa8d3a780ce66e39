"""Through the C ABI, two matrices whose scale codes lie side by side in one buffer."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("cols,ld", [(1, 16), (100, 16), (100, 48), (1024, 64), (1030, 64), (2000, 96), (4096, 128), (4097, 1024)])
def test_quantising_leaves_the_bytes_behind_a_row_s_codes(ops, cols, ld):
    from pimaicompiler_amd import _lib as L
    rows, blocks = 5, -(-cols // 32)
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(cols)).half().to(DEV)
    want = ops.mx4_quantize(x)
    packed, tops = torch.full((rows + 1, blocks * 16), 171, dtype=torch.uint8, device=DEV), torch.full((rows + 1,), 171, dtype=torch.uint8, device=DEV)
    scales = torch.full((rows + 1, ld), 171, dtype=torch.uint8, device=DEV)
    m = L.Mx4Matrix(packed.data_ptr(), scales.data_ptr(), tops.data_ptr(), rows, cols, ld)
    assert L.load().pimhip_mx4_quantize(m, x.data_ptr(), L.PIMHIP_F16, cols, torch.cuda.current_stream().cuda_stream) == L.PIMHIP_OK
    assert torch.equal(scales[:rows, :blocks], want.scales[:, :blocks]) and torch.equal(packed[:rows], want.packed) and torch.equal(tops[:rows], want.tops)
    assert (scales[:, blocks:] == 171).all() and (scales[rows] == 171).all() and (packed[rows] == 171).all() and (tops[rows] == 171).all()
    out = torch.empty(rows, cols, device=DEV)
    assert L.load().pimhip_mx4_dequantize(out.data_ptr(), L.PIMHIP_F32, cols, m, torch.cuda.current_stream().cuda_stream) == L.PIMHIP_OK
    assert torch.equal(out, want.dequantize(torch.float32))
    y = torch.randn(3, cols, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    got = torch.empty(3, rows, dtype=torch.float16, device=DEV)
    assert L.load().pimhip_mx4_linear(got.data_ptr(), rows, y.data_ptr(), cols, L.PIMHIP_F16, 3, m, None, 0, torch.cuda.current_stream().cuda_stream) == L.PIMHIP_OK
    assert torch.equal(got, ops.mx4_linear(y, want))
