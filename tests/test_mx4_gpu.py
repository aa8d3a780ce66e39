"""Microscaled 4-bit matrices against the format's definition in 64 bits: quantisation and reading back bit for bit, products within
the bounds their roundings have."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def power(e):
    """2**e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantized(x):
    """(values in 64 bits, scale codes) of x [rows, K] on the CPU by the definition: the nearest of the sixteen values, ties to the even code."""
    rows, K = x.shape
    v = torch.zeros(rows, -(-K // 32) * 32, dtype=torch.float64)
    v[:, :K] = x.double()
    v = v.view(rows, -1, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.where((top > 0) & ~bad, torch.frexp(torch.where(bad, 1.0, top)).exponent - 3, -127).clamp(-127, 127)
    u = torch.where(bad.unsqueeze(-1), 0.0, v) * power(-e).unsqueeze(-1)
    distance = (u.abs().unsqueeze(-1) - VALUES).abs()
    near = distance.amin(-1, keepdim=True)
    is_near = distance == near                     # (one or two neighbours: every difference is exact)
    even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], dtype=torch.bool)
    code = (is_near.double() + (is_near & even).double()).argmax(-1)
    q = torch.where(u < 0, -VALUES[code], VALUES[code]) * power(e).unsqueeze(-1)
    q[bad] = float("nan")
    return q.view(rows, -1)[:, :K], torch.where(bad, 255, e + 127).to(torch.uint8)


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def weight(seed, N, K, spread=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(N, K, generator=g, dtype=torch.float64) / math.sqrt(K)
    if spread:
        w = w * torch.pow(2.0, torch.randint(-spread, spread + 1, (N, -(-K // 32)), generator=g).double()).repeat_interleave(32, 1)[:, :K]
    return w.float()


# ---- quantisation and reading back -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 480), (4, 512), (1, 1024), (7, 1025), (2, 4096), (3, 5001), (1, 16384)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantising_is_the_definition(ops, rows, K, dtype):
    g = torch.Generator().manual_seed(rows * K)
    x = (torch.randn(rows, K, generator=g) * torch.pow(2.0, torch.randint(-12, 13, (rows, K), generator=g).float())).to(dtype)
    want, codes = quantized(x)
    q = ops.mx4_quantize(x.to(DEV))
    assert tuple(q.shape) == (rows, K)
    blocks = -(-K // 32)
    assert torch.equal(q.scales[:, :blocks].cpu(), codes)
    assert torch.equal(q.tops.cpu(), codes.amax(-1))
    for out in DTYPES:
        assert same(ops.mx4_dequantize(q, out).cpu(), want.to(out))
    assert not K % 32 or not (torch.stack([q.packed & 15, q.packed >> 4], -1).flatten(1)[:, K:] & 7).any()   # zeros behind the row


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16_bit_value_and_every_tie(ops, dtype):
    """Each of the 65536 values in a block of its own kind: alone, and beside a largest value that fixes the scale."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    alone = torch.zeros(65536, 32, dtype=dtype)
    alone[:, 7] = every
    beside = torch.zeros(65536, 32, dtype=dtype)
    beside[:, 7], beside[:, 30] = every, 4.0
    for x in (alone, beside):
        want, codes = quantized(x)
        q = ops.mx4_quantize(x.to(DEV))
        assert torch.equal(q.scales[:, 0].cpu(), codes[:, 0])
        assert same(ops.mx4_dequantize(q, torch.float32).cpu(), want.float())


def test_the_ends_of_the_range(ops):
    big = torch.finfo(torch.float32).max
    x = torch.zeros(6, 64)
    x[0, :4] = torch.tensor([big, -big, big / 2, 1.0])
    x[1, :4] = torch.tensor([2.0**-149, 2.0**-130, -(2.0**-127), 2.0**-126])
    x[2, 40] = float("inf")
    x[3, 3] = float("nan")
    x[4, :] = -0.0
    x[5, :32], x[5, 32:] = float("-inf"), 3.0
    want, codes = quantized(x)
    q = ops.mx4_quantize(x.to(DEV))
    assert torch.equal(q.scales[:, :2].cpu(), codes)
    assert same(ops.mx4_dequantize(q, torch.float32).cpu(), want.float())
    assert q.tops.cpu().tolist() == [int(c[c < 255].max()) for c in codes]


def test_strides_offsets_and_leading_shapes(ops):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(9, 700, generator=g).half().to(DEV)
    for x in (wide[:, 3:133], wide[::2, 1:65], wide.t()[5:70], wide[4, 7:300], wide[:8, :640].view(2, 4, 640)[:, 1:3]):
        want, _ = quantized(x.reshape(-1, x.size(-1)).cpu())
        q = ops.mx4_quantize(x)
        assert q.shape == x.shape
        assert torch.equal(q.dequantize(torch.float32).cpu(), want.float().view(x.shape))
    q = ops.mx4_quantize(torch.empty(0, 64, dtype=torch.float16, device=DEV))
    assert tuple(q.dequantize().shape) == (0, 64)


def test_a_tensor_of_bytes_from_elsewhere(ops):
    """Any bytes: the codes' values by the definition, what a partial block holds behind its row left out."""
    g = torch.Generator().manual_seed(4)
    for rows, K in ((3, 64), (5, 45), (2, 1), (4, 1024)):
        blocks = -(-K // 32)
        packed = torch.randint(0, 256, (rows, blocks * 16), generator=g, dtype=torch.uint8)
        scales = torch.randint(100, 140, (rows, blocks), generator=g, dtype=torch.uint8)
        scales[0, 0] = 255
        codes = torch.stack([packed & 15, packed >> 4], -1).view(rows, -1)
        signed = torch.cat([VALUES, -VALUES])[codes.long()]
        want = torch.where((scales == 255).repeat_interleave(32, 1), float("nan"), signed * power(scales.int() - 127).repeat_interleave(32, 1))[:, :K]
        q = ops.Mx4Tensor(packed.to(DEV), scales.to(DEV), K)
        assert same(q.dequantize(torch.float32).cpu(), want.float())
        tops = torch.where(scales == 255, 0, scales).amax(-1)
        assert torch.equal(q.tops.cpu(), tops)


# ---- products ----------------------------------------------------------------------------------------------------------------
def check_product(got, x, w, bias, relu):
    """Against 64 bits.  fp32 sums of K products in any order are within (K + 2) 2^-24 of sum |x w| (+ |bias|: one more addition); the
    store rounds by at most half a step."""
    want = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    if relu:
        want = want.clamp(min=0)
    eps = torch.finfo(got.dtype).eps / 2
    bound = (x.size(-1) + 2) * 2.0**-24 * size
    tiny = 2.0**-25 if got.dtype == torch.float16 else 2.0**-134   # half the distance of subnormals
    bound = bound * (1 + eps) + want.abs() * eps + tiny
    # A value from max + half a step on rounds to an infinity (IEEE 754, round to nearest): by the definition of the type, not within a bound.
    info = torch.finfo(got.dtype)
    border = info.max * (1 + info.eps / 4)
    got = got.cpu().double()
    over = want.abs() - bound >= border
    assert torch.equal(got[over], torch.sign(want[over]) * math.inf)
    off = (got - want).abs()
    assert bool((off <= bound)[~over].all()), float((off / bound)[~over].max())


PRODUCTS = [(1, 1, 1), (1, 17, 31), (1, 64, 32), (2, 100, 96), (1, 1024, 1024), (3, 257, 640), (15, 31, 1025), (16, 48, 128), (17, 200, 130), (32, 65, 512), (33, 64, 4096),
            (64, 130, 777), (65, 129, 256), (100, 300, 999), (129, 257, 512), (300, 128, 64), (1, 5000, 2050), (257, 384, 1056)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear(ops, M, N, K, dtype):
    g = torch.Generator().manual_seed(M * N + K)
    x = torch.randn(M, K, generator=g).to(dtype)
    q = ops.mx4_quantize(weight(N, N, K).to(DEV))
    w = q.dequantize(torch.float32).cpu()
    bias = torch.randn(N, generator=g).to(dtype)
    check_product(ops.mx4_linear(x.to(DEV), q), x, w, None, False)
    check_product(ops.mx4_linear(x.to(DEV), q, bias.to(DEV), "aten::relu"), x, w, bias, True)


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul(ops, M, N, K, dtype):
    g = torch.Generator().manual_seed(M + N + K)
    a = ops.mx4_quantize(torch.randn(M, K, generator=g).to(DEV))
    b = ops.mx4_quantize(weight(N + 1, N, K).to(DEV))
    check_product(ops.mx4_matmul(a, b, dtype), a.dequantize(torch.float32).cpu(), b.dequantize(torch.float32).cpu(), None, False)


# Many tiles: more bands of tokens than one, steps of k that begin in the middle and go round, K that ends in every part of a step.
@pytest.mark.parametrize("M,N,K", [(1180, 1050, 96), (300, 520, 1536), (257, 129, 2080), (65, 136, 1400), (640, 127, 512), (129, 260, 250), (70, 1029, 800), (66, 100, 200), (200, 140, 1300),
                                   (600, 2100, 416),
                                   (40, 12300, 64), (3, 16400, 160), (16, 16385, 33)])
def test_products_of_many_tiles(ops, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    a, b = ops.mx4_quantize(x.to(DEV)), ops.mx4_quantize(weight(N + 2, N, K).to(DEV))
    w = b.dequantize(torch.float32).cpu()
    check_product(ops.mx4_matmul(a, b, torch.float32), a.dequantize(torch.float32).cpu(), w, None, False)
    check_product(ops.mx4_linear(x.to(DEV), b), x, w, None, False)


@pytest.mark.parametrize("M", [1, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_with_scales_far_apart_and_far_from_one(ops, M, dtype):
    """Blocks 2^-14 .. 2^14 apart inside a row, rows down to 2^-60: fp16 has no such values, its products do."""
    N, K = 50, 320
    w = weight(9, N, K, spread=14) * torch.pow(2.0, torch.linspace(-60, 8, N).round()).unsqueeze(1)
    q = ops.mx4_quantize(w.to(DEV))
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).to(dtype)
    if dtype == torch.bfloat16:
        x = x * 2.0**30
    check_product(ops.mx4_linear(x.to(DEV), q), x, q.dequantize(torch.float32).cpu(), None, False)


@pytest.mark.parametrize("M", [1, 5, 33, 130])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_nan_and_infinities_stay_in_their_rows(ops, M, dtype):
    N, K = 70, 200
    w = weight(2, N, K)
    w[13, 180], w[40, 3] = float("nan"), float("inf")
    q = ops.mx4_quantize(w.to(DEV))
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[M - 1, 199] = float("inf")
    y = ops.mx4_linear(x.to(DEV), q).cpu()
    z = ops.mx4_matmul(ops.mx4_quantize(x.to(DEV)), q, dtype).cpu()
    rows = torch.zeros(N, dtype=torch.bool)
    rows[[13, 40]] = True
    assert y[:, rows].isnan().all() and z[:, rows].isnan().all()
    assert torch.isfinite(y[:M - 1][:, ~rows]).all() and torch.isfinite(z[:M - 1][:, ~rows]).all()
    assert not torch.isfinite(y[M - 1]).any() and z[M - 1].isnan().all()


@pytest.mark.parametrize("M", [1, 3, 66])
def test_any_pitch_and_address(ops, M):
    K, N = 333, 90
    g = torch.Generator().manual_seed(11)
    wide = torch.randn(2 * M, K + 9, generator=g).half().to(DEV)
    q = ops.mx4_quantize(weight(5, N, K).to(DEV))
    w = q.dequantize(torch.float32).cpu()
    for x in (wide[:M, 1:K + 1], wide[::2, 9:], wide[:M, :K].unsqueeze(1), torch.as_strided(wide, (M, K), (K + 9, 1), 3).t().contiguous().t()):
        check_product(ops.mx4_linear(x, q).reshape(M, N), x.reshape(M, K).cpu(), w, None, False)


def test_empty_and_one_dimensional(ops):
    q = ops.mx4_quantize(weight(5, 40, 64).to(DEV))
    x = torch.randn(64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    y = ops.mx4_linear(x, q)
    assert tuple(y.shape) == (40,) and torch.equal(y, ops.mx4_linear(x.view(1, 64), q).view(40))
    assert tuple(ops.mx4_matmul(ops.mx4_quantize(x), q).shape) == (40,)
    none = x.view(1, 64)[:0]
    assert tuple(ops.mx4_linear(none, q).shape) == (0, 40) and tuple(ops.mx4_matmul(ops.mx4_quantize(none), q).shape) == (0, 40)
    no_rows = ops.mx4_quantize(none)
    assert tuple(ops.mx4_linear(x, no_rows).shape) == (0,)


def test_the_rows_around_an_output_stay_as_they_are(ops):
    """Through the C ABI with a pitch: nothing but the product's own values is written."""
    from pimaicompiler_amd import _lib as L
    for M in (1, 20, 150):
        N, K = 61, 96
        q = ops.mx4_quantize(weight(6, N, K).to(DEV))
        x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).half().to(DEV)
        for a in (x, None):
            out = torch.full((M + 2, N + 5), 7.0, dtype=torch.float16, device=DEV)
            at = out.data_ptr() + ((N + 5) + 2) * 2
            s = torch.cuda.current_stream().cuda_stream
            if a is not None:
                rc = L.load().pimhip_mx4_linear(at, N + 5, x.data_ptr(), K, L.PIMHIP_F16, M, q._c, None, 0, s)
                want = ops.mx4_linear(x, q)
            else:
                xq = ops.mx4_quantize(x)
                rc = L.load().pimhip_mx4_matmul(at, N + 5, L.PIMHIP_F16, xq._c, q._c, s)
                want = ops.mx4_matmul(xq, q)
            assert rc == 0
            assert torch.equal(out[1:M + 1, 2:2 + N], want)
            out[1:M + 1, 2:2 + N] = 7.0
            assert bool((out == 7.0).all())


def test_a_graph_replays_and_streams_keep_apart(ops):
    q = ops.mx4_quantize(weight(6, 100, 256).to(DEV))
    x = torch.randn(70, 256, generator=torch.Generator().manual_seed(1)).half().to(DEV)

    def step():
        y = ops.mx4_linear(x, q, act_type="aten::relu")
        return y, ops.mx4_matmul(ops.mx4_quantize(x), q), ops.mx4_quantize(y).dequantize()
    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    for _ in range(4):
        x.mul_(0.5).mul_(-2)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    for stream in (side, side.cuda_stream):
        side.wait_stream(torch.cuda.current_stream())
        y = ops.mx4_linear(x, q, act_type="aten::relu", stream=stream)
        side.synchronize()
        assert torch.equal(y, eager[0])


def test_equal_calls_give_equal_bits(ops):
    q = ops.mx4_quantize(weight(6, 500, 2048).to(DEV))
    for M in (1, 30, 200):
        x = torch.randn(M, 2048, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
        assert torch.equal(ops.mx4_linear(x, q), ops.mx4_linear(x, q))
        a = ops.mx4_quantize(x)
        assert torch.equal(ops.mx4_matmul(a, q), ops.mx4_matmul(a, q))


def test_refusals_on_the_gpu(ops):
    x = torch.zeros(2, 64, dtype=torch.float16, device=DEV)
    q = ops.mx4_quantize(x)
    E = ops.NNRuntimeException
    for call in (lambda: ops.mx4_linear(x[:, :32], q), lambda: ops.mx4_linear(x.float(), q), lambda: ops.mx4_linear(x, x), lambda: ops.mx4_linear(x.cpu(), q),
                 lambda: ops.mx4_linear(x, q, torch.zeros(3, dtype=torch.float16, device=DEV)), lambda: ops.mx4_linear(x, q, torch.zeros(2, device=DEV)),
                 lambda: ops.mx4_linear(x.clone().requires_grad_(), q), lambda: ops.mx4_quantize(x.int()), lambda: ops.mx4_quantize(x[:, :0]),
                 lambda: ops.mx4_quantize(x.float().requires_grad_()), lambda: ops.mx4_dequantize(x), lambda: ops.mx4_dequantize(q, torch.int8),
                 lambda: ops.mx4_matmul(q, x), lambda: ops.mx4_matmul(q, ops.mx4_quantize(x[:, :32])), lambda: ops.mx4_matmul(q, q, torch.int32),
                 lambda: ops.Mx4Tensor(q.packed, q.scales[:, :2], 65), lambda: ops.Mx4Tensor(q.packed.int(), q.scales[:, :2], 64),
                 lambda: ops.Mx4Tensor(q.packed, q.scales[:1, :2], 64), lambda: ops.Mx4Tensor(q.packed, q.scales[:, :2], 0)):
        with pytest.raises(E):
            call()
    with torch.no_grad():
        ops.mx4_linear(x.clone().requires_grad_(), q)


def test_the_c_interface_refuses_what_no_launch_can_hold(ops):
    from pimaicompiler_amd import _lib as L
    lib = L.load()
    q = ops.mx4_quantize(torch.zeros(2, 2048, dtype=torch.float16, device=DEV))
    at = (q.packed.data_ptr(), q.scales.data_ptr(), q.tops.data_ptr())
    for rows, cols, ld, want in ((1 << 34, 2048, 64, L.PIMHIP_ERR_UNSUPPORTED), (1 << 36, 32, 16, L.PIMHIP_ERR_UNSUPPORTED), (2, (1 << 26) + 1, 1 << 22, L.PIMHIP_ERR_INVALID_ARGUMENT),
                                 (2, 2048, 48, L.PIMHIP_ERR_INVALID_ARGUMENT), (2, 2048, 72, L.PIMHIP_ERR_INVALID_ARGUMENT), (2, 2048, 1 << 27, L.PIMHIP_ERR_INVALID_ARGUMENT)):
        assert lib.pimhip_mx4_quantize(L.Mx4Matrix(*at, rows, cols, ld), q.packed.data_ptr(), L.PIMHIP_F16, cols, None) == want
    big = L.Mx4Matrix(*at, 1 << 33, 2048, 64)
    assert lib.pimhip_mx4_linear(q.packed.data_ptr(), 1 << 33, q.packed.data_ptr(), 2048, L.PIMHIP_F16, 4096, big, None, 0, None) == L.PIMHIP_ERR_UNSUPPORTED
    assert lib.pimhip_mx4_matmul(q.packed.data_ptr(), 1 << 33, L.PIMHIP_F16, big, big, None) == L.PIMHIP_ERR_UNSUPPORTED
