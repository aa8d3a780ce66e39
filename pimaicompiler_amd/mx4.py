"""Weights and activations in microscaled 4-bit floating point (E2M1 values in blocks of 32 that share a power of two): quantisation,
reading back, the product of fp16 / bf16 tokens with 4-bit weights, and the product of two 4-bit operands.

The reference's weights are fp16 throughout; a product for one token is bound by its weights' bytes, and these are 17 bytes for 32
values instead of 64.  Errors are NNRuntimeException, as everywhere in this package; there is no CPU path and no backward pass.
"""
import ctypes

import torch

from . import _lib as L
from .ops import NNRuntimeException, _act_code, _check, _ensure_init, _Launch, _native, _require_no_gradient, _result

BLOCK = 32  # values that share a scale
_CODES = {torch.float16: L.PIMHIP_F16, torch.bfloat16: L.PIMHIP_BF16, torch.float32: L.PIMHIP_F32}


def _rows_of(x):
    """x [.., K] as (two-dimensional tensor whose rows are contiguous, their pitch)."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    if x2.size(0) > 1 and (x2.stride(1) != 1 or x2.stride(0) < x2.size(1)) or x2.size(0) == 1 and x2.stride(1) != 1 and x2.size(1) > 1:
        x2 = x2.contiguous()
    return x2, x2.stride(0) if x2.size(0) > 1 else x2.size(1)


def _require(name, t, dtypes):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise NNRuntimeException(f"{name} must be a tensor on the GPU (there is no CPU fallback)")
    if t.dtype not in dtypes:
        raise NNRuntimeException(f"{name} is {t.dtype}; taken are {', '.join(str(d) for d in dtypes)}")


class Mx4Tensor:
    """A matrix, or a stack of rows of any leading shape, in microscaled 4-bit floating point.

    mx4_quantize makes one of a tensor; Mx4Tensor(packed, scales, in_features) of bytes from elsewhere: packed [rows,
    ceil(K / 32) * 16] uint8 (two values a byte, the first in the low half) and scales [rows, ceil(K / 32)] uint8 (2^(code - 127); 255 makes
    a block NaN), both on the GPU.  The bytes are not copied where they can be used as they are: they are the tensor's from then on,
    and code that writes to them later has to make a new Mx4Tensor, which holds each row's largest scale besides.

    shape       the shape of the values, K last
    packed      [rows, ceil(K / 32) * 16] uint8
    scales      [rows, pitch] uint8, the pitch ceil(K / 32) rounded up to 16; what lies behind a row's codes may be anything
    tops        [rows] uint8, the largest scale code of each row
    """

    def __init__(self, packed, scales, in_features, stream=None):
        _require("packed", packed, (torch.uint8,))
        _require("scales", scales, (torch.uint8,))
        K = int(in_features)
        if packed.dim() != 2 or scales.dim() != 2 or K < 1:
            raise NNRuntimeException("packed and scales must be two-dimensional, in_features at least 1")
        rows, blocks = packed.size(0), -(-K // BLOCK)
        if tuple(packed.shape) != (rows, blocks * 16) or tuple(scales.shape) != (rows, blocks):
            raise NNRuntimeException(f"rows of {K} values are packed [rows, {blocks * 16}] and scales [rows, {blocks}]; got {tuple(packed.shape)} and "
                                     f"{tuple(scales.shape)}")
        if packed.device != scales.device:
            raise NNRuntimeException(f"packed is on {packed.device}, scales on {scales.device}")
        _ensure_init(packed)
        with _Launch(packed.device, stream, packed, scales) as handle:
            packed = packed.contiguous()
            if packed.data_ptr() % 16:
                packed = packed.clone()
            if K % BLOCK:   # zeros behind a row's end, whatever the last block held there
                packed = packed.clone()
                behind = K % BLOCK
                if behind % 2:
                    packed[:, (K // 2)] &= 15
                packed[:, (K + 1) // 2:] = 0
            pitch = -(-blocks // 16) * 16
            if pitch != blocks or not scales.is_contiguous() or scales.data_ptr() % 16:
                wide = torch.zeros((rows, pitch), dtype=torch.uint8, device=scales.device)
                wide[:, :blocks] = scales
                scales = wide
            self._hold(packed, scales, torch.empty(rows, dtype=torch.uint8, device=packed.device), (rows, K))
            _check(L.load().pimhip_mx4_find_tops(self._c, handle))

    def _hold(self, packed, scales, tops, shape):
        self.packed, self.scales, self.tops, self.shape = packed, scales, tops, torch.Size(shape)
        self._keep = L.Mx4Matrix(packed.data_ptr(), scales.data_ptr(), tops.data_ptr(), packed.size(0), self.shape[-1], scales.size(1))
        self._at = ctypes.addressof(self._keep)   # (what the native calls read the matrix through)
        self._device_index = packed.device.index

    @classmethod
    def _empty(cls, shape, device):
        rows = 1
        for n in shape[:-1]:
            rows *= n
        blocks = -(-shape[-1] // BLOCK)
        self = cls.__new__(cls)
        self._hold(torch.empty((rows, blocks * 16), dtype=torch.uint8, device=device),
                   torch.empty((rows, -(-blocks // 16) * 16), dtype=torch.uint8, device=device), torch.empty(rows, dtype=torch.uint8, device=device), shape)
        return self

    @classmethod
    def _again(cls, packed, scales, in_features, shape):
        self = cls(packed, scales, in_features)
        self.shape = torch.Size(shape)
        return self

    def __reduce__(self):
        """A deep copy, or one read from a file, is made of its own tensors: what the native calls read it through holds addresses."""
        K = self.shape[-1]
        return Mx4Tensor._again, (self.packed, self.scales[:, :-(-K // BLOCK)], K, tuple(self.shape))

    def _tensors(self):
        return self.packed, self.scales, self.tops

    @property
    def _c(self):
        return L.Mx4Matrix.from_address(self._at)

    @property
    def device(self):
        return self.packed.device

    @property
    def rows(self):
        return self.packed.size(0)

    def dequantize(self, dtype=torch.float16, stream=None):
        return mx4_dequantize(self, dtype, stream)

    def __repr__(self):
        return f"Mx4Tensor(shape={tuple(self.shape)}, device={self.device})"


def mx4_quantize(x, stream=None):
    """x [.., K] (fp16, bf16 or fp32) as an Mx4Tensor of the same shape.  A block of 32 along K gets the scale 2^(floor(log2(largest
    magnitude)) - 2), its values the nearest 4-bit one, ties to the even code, saturating at 6 scales; a block that holds an infinity or a
    NaN reads back as NaN."""
    made = _native().fast_mx4_quantize(x) if stream is None else None
    if made is not None:
        q = Mx4Tensor.__new__(Mx4Tensor)
        q.packed, q.scales, q.tops, q._keep, q._at, q._device_index = _result(made)
        q.shape = x.shape
        return q
    _require("x", x, tuple(_CODES))
    _require_no_gradient(x)
    if x.dim() < 1 or x.size(-1) < 1:
        raise NNRuntimeException("x must have at least one dimension, the last of at least one value")
    _ensure_init(x)
    with _Launch(x.device, stream, x) as handle:
        x2, ld = _rows_of(x)
        q = Mx4Tensor._empty(x.shape, x.device)
        _check(L.load().pimhip_mx4_quantize(q._c, x2.data_ptr(), _CODES[x.dtype], ld, handle))
    return q


def mx4_dequantize(q, dtype=torch.float16, stream=None):
    """The values of an Mx4Tensor in fp16, bf16 or fp32, each rounded once."""
    if not isinstance(q, Mx4Tensor):
        raise NNRuntimeException("an Mx4Tensor is read back")
    if dtype not in _CODES:
        raise NNRuntimeException(f"{dtype} is none of {', '.join(str(d) for d in _CODES)}")
    out = _native().fast_mx4_dequantize(q._at, q.shape, q._device_index, _CODES[dtype]) if stream is None else None
    if out is not None:
        return _result(out)
    _ensure_init(q.packed)
    with _Launch(q.device, stream, *q._tensors()) as handle:
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(L.load().pimhip_mx4_dequantize(out.data_ptr(), _CODES[dtype], q.shape[-1], q._c, handle))
    return out


def mx4_linear(x, weight, bias=None, act_type="none", stream=None):
    """act(x . W^T + b) for x [.., K] in fp16 or bf16, W an Mx4Tensor [N, K], b [N] of x's type or None; act_type as
    custom_aten_addmm's.  One token up to whole prompts; the result [.., N] has x's type."""
    if stream is None and isinstance(weight, Mx4Tensor) and len(weight.shape) == 2:
        out = _native().fast_mx4_linear(x, weight._at, weight._device_index, bias, act_type == "aten::relu")
        if out is not None:
            return _result(out)
    _require("x", x, (torch.float16, torch.bfloat16))
    if not isinstance(weight, Mx4Tensor) or len(weight.shape) != 2:
        raise NNRuntimeException("weight must be a two-dimensional Mx4Tensor")
    N, K = weight.shape
    if x.dim() < 1 or x.size(-1) != K:
        raise NNRuntimeException(f"x must end in {K} values, the weight's columns; it is {tuple(x.shape)}")
    if bias is not None:
        _require("bias", bias, (x.dtype,))
        if bias.numel() != N:
            raise NNRuntimeException(f"bias has {bias.numel()} elements, the product {N}")
    _require_no_gradient(x, bias)
    for t in (weight, bias):
        if t is not None and t.device != x.device:
            raise NNRuntimeException(f"x is on {x.device}, weight or bias on {t.device}")
    _ensure_init(x)
    with _Launch(x.device, stream, x, bias, *weight._tensors()) as handle:
        x2, ld = _rows_of(x)
        if bias is not None:
            bias = bias.contiguous()
        out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
        _check(L.load().pimhip_mx4_linear(out.data_ptr(), N, x2.data_ptr(), ld, _CODES[x.dtype], x2.size(0), weight._c,
                                          bias.data_ptr() if bias is not None else None, _act_code(act_type), handle))
    return out


def mx4_matmul(a, b, dtype=torch.float16, stream=None):
    """a . b^T of two Mx4Tensors, a [.., K] and b [N, K], in fp16, bf16 or fp32: [.., N].  Products are exact, sums fp32."""
    if not isinstance(a, Mx4Tensor) or not isinstance(b, Mx4Tensor) or len(b.shape) != 2:
        raise NNRuntimeException("both operands must be Mx4Tensors, the second two-dimensional")
    if dtype not in _CODES:
        raise NNRuntimeException(f"{dtype} is none of {', '.join(str(d) for d in _CODES)}")
    if a.shape[-1] != b.shape[-1]:
        raise NNRuntimeException(f"the operands disagree on the reduction width ({a.shape[-1]} vs {b.shape[-1]})")
    if a._device_index != b._device_index:
        raise NNRuntimeException(f"a is on {a.device}, b on {b.device}")
    out = _native().fast_mx4_matmul(a._at, a.shape, b._at, a._device_index, _CODES[dtype]) if stream is None else None
    if out is not None:
        return _result(out)
    _ensure_init(a.packed)
    N = b.shape[0]
    with _Launch(a.device, stream, *a._tensors(), *b._tensors()) as handle:
        out = torch.empty((*a.shape[:-1], N), dtype=dtype, device=a.device)
        _check(L.load().pimhip_mx4_matmul(out.data_ptr(), N, _CODES[dtype], a._c, b._c, handle))
    return out
